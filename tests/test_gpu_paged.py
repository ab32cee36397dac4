"""The paged cache and beam search on the GPU, against plain NumPy forms in 64 bits.

Tolerances.  Attention: the float32 bar of the other kernels, max |error| / max |reference| <= 1e-5, against
float64 of the stored (rounded) keys and values.  Rotary: two products and a sum, each rounded by at most 2^-24 of
its value, so |error| <= 2^-23 (|x cos| + |y sin|).  The cache's type rounds by at most eps / 2 of the value besides
(below the smallest normal float16, by half of 2^-24).  Scores: 2^-24 of the value for its float32, and 1e-6 for the
log of the sum (each exponential within 2^-22 of its own).  Everything whole is equal.
"""

import ctypes

import numpy as np
import pytest

from conftest import rel_err

pytestmark = pytest.mark.gpu

TOL = 1e-5
I32, I64, U8 = np.int32, np.int64, np.uint8
TYPES = ("float32", "float16", "bfloat16")


@pytest.fixture(scope="module")
def paged(gpu):
    from cv3amd import paged
    return paged


def dev(a, dtype=None):
    from cv3amd.device import to_device
    return to_device(np.ascontiguousarray(a) if dtype is None else np.ascontiguousarray(a, dtype=dtype))


def bf16_bits(x):
    """Round to nearest even; a NaN stays one."""
    b = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def stored(x, kind):
    """The cache's array of float32 values, and the values that it holds."""
    x = np.ascontiguousarray(x, np.float32)
    if kind == "float32":
        return x, x.astype(np.float64)
    if kind == "float16":
        with np.errstate(over="ignore"):
            h = x.astype(np.float16)
        return h, h.astype(np.float64)
    b = bf16_bits(x)
    return b, values(b, kind)


def values(a, kind):
    if kind == "bfloat16":
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


# ------------------------------------------------------------------------------------------------
# block tables
# ------------------------------------------------------------------------------------------------

def tables_ref(lengths, new, page, free, taken, tables, tokens):
    tables, cap = tables.copy(), tables.shape[1] * page
    total, starts, slots, positions = [], [0], [], []
    for r in range(len(lengths)):
        held = max(int(lengths[r]), 0)
        give = max(0, min(int(new[r]), cap - held, tokens - len(slots)))
        for pos in range(held, held + give):
            if pos % page == 0:
                tables[r, pos // page] = free[taken] if 0 <= taken < len(free) else -1
                taken += 1
            at = int(tables[r, pos // page])
            slots.append(at * page + pos % page if at >= 0 else -1)
            positions.append(pos)
        total.append(held + give)
        starts.append(len(slots))
    rest = [-1] * (tokens - len(slots))
    return tables, total, min(taken, 2**31 - 1), starts, slots + rest, positions + rest


def check_tables(paged, lengths, new, page, free, taken, blocks, tokens=None, seed=0):
    rng = np.random.default_rng([seed, len(lengths), page])
    tables = rng.integers(-1, 900, (len(lengths), blocks)).astype(I32)
    lengths, new, free = (np.asarray(x, I32) for x in (lengths, new, free))
    tokens = int(np.maximum(new, 0).sum()) if tokens is None else tokens
    want = tables_ref(lengths, new, page, free, taken, tables, tokens)
    td = dev(tables)
    got = paged.block_tables(lengths, new, page, free, np.array([taken], I32), td, tokens=tokens)
    assert np.array_equal(td.numpy(), want[0])
    for g, w, name in zip(got, want[1:], ("total", "taken", "starts", "slots", "positions")):
        assert np.array_equal(g, np.asarray(w).reshape(g.shape)), name


@pytest.mark.parametrize("requests,page,blocks", [(1, 16, 3), (1, 1, 40), (3, 5, 20), (64, 16, 9), (65, 64, 4),
                                                  (1023, 16, 8), (1024, 24, 6), (1025, 7, 11), (4096, 32, 3)])
def test_block_tables(paged, requests, page, blocks):
    rng = np.random.default_rng([requests, page])
    cap = page * blocks
    lengths = rng.integers(0, cap // 2 + 1, requests)
    new = rng.integers(0, cap // 2 + 1, requests)
    new[rng.random(requests) < 0.3] = 0
    free = rng.permutation(requests * blocks + 3)
    check_tables(paged, lengths, new, page, free, 2, blocks)
    check_tables(paged, lengths, np.ones(requests), page, free, 0, blocks)                  # a decode step
    check_tables(paged, lengths, new, page, free, 1, blocks, tokens=int(new.sum()) + 37)    # a padded list
    check_tables(paged, lengths, new, page, free, 0, blocks, tokens=int(new.sum()) // 2)    # a list too short
    check_tables(paged, lengths, new, page, free[:max(1, requests // 3)], 0, blocks)        # pages run out


def test_block_tables_of_reserved_pages(paged):
    """Without free pages the tables are as they are, and give every slot."""
    rng = np.random.default_rng(3)
    for requests, page, blocks in ((1, 1, 5), (70, 16, 6), (1100, 5, 9)):
        tables = rng.integers(-1, 500, (requests, blocks)).astype(I32)
        lengths, new = (rng.integers(0, page * blocks // 2 + 3, requests).astype(I32) for _ in range(2))
        tokens = int(new.sum()) + 3
        td = dev(tables)
        total, taken, starts, slots, positions = paged.block_tables(lengths, new, page, None, None, td, tokens=tokens)
        pos = [p for n, g in zip(lengths, new) for p in range(n, min(n + g, page * blocks))]
        row = [i for i, (n, g) in enumerate(zip(lengths, new)) for _ in range(n, min(n + g, page * blocks))]
        pos, row = np.array(pos, int), np.array(row, int)
        of = tables[row, pos // page].astype(I64)
        assert taken is None and np.array_equal(td.numpy(), tables)
        assert np.array_equal(total, np.maximum(lengths, np.minimum(lengths + new, page * blocks)))
        assert np.array_equal(starts, np.concatenate([[0], np.cumsum(total - lengths)]))
        assert np.array_equal(positions, np.concatenate([pos, -np.ones(tokens - len(pos), int)]))
        assert np.array_equal(slots[:len(pos)], np.where(of >= 0, of * page + pos % page, -1))
        assert np.all(slots[len(pos):] == -1)


def test_block_tables_at_the_edges(paged):
    free = np.arange(100, 140)
    check_tables(paged, [0, 0, 0], [0, 0, 0], 16, free, 0, 4)                  # no token at all
    check_tables(paged, [0, 0, 0], [0, 0, 0], 16, free, 0, 4, tokens=5)
    check_tables(paged, [0, 16, 32], [16, 16, 1], 16, free, 0, 4)              # lengths on a page's border
    check_tables(paged, [63, 64, 65, 1 << 30, 2**31 - 1], [1, 1, 1, 1, 1], 16, free, 0, 4)     # past the table
    check_tables(paged, [0, 10], [2**31 - 1, 2**31 - 1], 16, free, 0, 4, tokens=200)
    check_tables(paged, [-5, 3], [4, -7], 16, free, 0, 4, tokens=6)            # negative counts as none
    check_tables(paged, [0, 0], [20, 20], 16, free, 39, 4)                     # the last page, then none
    check_tables(paged, [0, 0], [20, 20], 16, free, 2**31 - 1, 4)
    check_tables(paged, [0, 0], [20, 20], 16, free, -1, 4)
    check_tables(paged, [3], [40], 16, np.zeros(0), 0, 4)                      # no free page
    check_tables(paged, [], [], 16, free, 0, 4, tokens=3)                      # no request
    check_tables(paged, [0], [3000], 1, np.arange(4000), 0, 4000)              # one key a page
    check_tables(paged, [40000], [60000], 65536, np.arange(4), 0, 2)           # the largest page


# ------------------------------------------------------------------------------------------------
# rotary and cache write
# ------------------------------------------------------------------------------------------------

def rotary(dim, rows, theta=1e6):
    ang = np.arange(rows)[:, None] / theta ** (np.arange(0, dim, 2) / dim)
    ang = np.concatenate([ang, ang], axis=1)
    return np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)


def turn(x, cos, sin):
    """(n, heads, d) turned, and the bound of its float32 error."""
    half = x.shape[-1] // 2
    y = np.concatenate([-x[..., half:], x[..., :half]], axis=-1)
    c, s = cos[:, None], sin[:, None]
    return x * c + y * s, 2.0 ** -23 * (np.abs(x * c) + np.abs(y * s))


def rounding(x, kind):
    if kind == "float32":
        return 0.0
    return np.maximum(np.abs(x) * (2.0 ** -11 if kind == "float16" else 2.0 ** -8), 2.0 ** -25)


APPEND = [(1, 14, 2, 64, 16), (7, 14, 2, 64, 16), (130, 16, 16, 64, 5), (33, 32, 8, 128, 32), (3, 1, 1, 8, 1),
          (19, 4, 4, 80, 24), (5, 0, 3, 96, 7), (9, 20, 4, 256, 100), (1001, 6, 2, 40, 64)]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n,heads,kv,d,page", APPEND)
def test_append(paged, n, heads, kv, d, page, kind):
    rng = np.random.default_rng([n, heads, d])
    pages = -(-2 * n // page) + 1
    rows = rng.normal(size=(n, (heads + 2 * kv) * d)).astype(np.float32)
    slots = rng.permutation(pages * page)[:n].astype(I64)
    positions = rng.integers(0, 60, n).astype(I32)
    slots[rng.random(n) < 0.1] = -1
    if n > 4:
        slots[1], slots[2] = pages * page, -(1 << 40)               # outside the cache
        positions[3], positions[4] = 60, -1                         # outside the tables
    cos, sin = rotary(d, 60)
    before = rng.normal(size=(2, pages, kv, page, d)).astype(np.float32)
    k, v = (dev(stored(b, kind)[0]) for b in before)
    held_k, held_v = (values(c.numpy(), kind) for c in (k, v))
    q = paged.append(rows, heads, positions, slots, cos, sin, k, v)
    x = rows.astype(np.float64).reshape(n, heads + 2 * kv, d)
    placed = (positions >= 0) & (positions < 60)
    at = np.where(placed, positions, 0)
    want, bound = turn(x, cos.astype(np.float64)[at], sin.astype(np.float64)[at])
    assert np.all(np.abs(q - np.where(placed[:, None, None], want[:, :heads], 0.0)) <= bound[:, :heads])
    tol_k, tol_v = np.zeros_like(held_k), np.zeros_like(held_v)
    for i in range(n):
        if placed[i] and 0 <= slots[i] < pages * page:
            p, r = divmod(int(slots[i]), page)
            held_k[p, :, r], held_v[p, :, r] = want[i, heads:heads + kv], x[i, heads + kv:]
            # a value that rounds the other way for its float32 error is off by that error more
            tol_k[p, :, r] = rounding(held_k[p, :, r], kind) * (1 + 2.0 ** -10) + bound[i, heads:heads + kv]
            tol_v[p, :, r] = rounding(held_v[p, :, r], kind)
    assert np.all(np.abs(values(k.numpy(), kind) - held_k) <= tol_k)
    assert np.all(np.abs(values(v.numpy(), kind) - held_v) <= tol_v)


@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
def test_append_of_many_rows(paged, kind):
    """A call that moves more than 256 MB: the same values at both ends and in between."""
    rng = np.random.default_rng(4)
    n, heads, kv, d, page = 32001, 14, 2, 64, 16
    pages = -(-n // page)
    rows = rng.normal(size=(n, 18 * d)).astype(np.float32)
    slots, positions = rng.permutation(pages * page)[:n].astype(I64), rng.integers(0, 500, n).astype(I32)
    cos, sin = rotary(d, 500)
    k, v = paged.new_cache(pages, kv, page, d, kind)
    q = paged.append(rows, heads, positions, slots, cos, sin, k, v)
    at = np.concatenate([np.arange(500), rng.integers(0, n, 2000), np.arange(n - 500, n)])
    x = rows[at].astype(np.float64).reshape(len(at), 18, d)
    want, bound = turn(x, cos.astype(np.float64)[positions[at]], sin.astype(np.float64)[positions[at]])
    assert np.all(np.abs(q[at] - want[:, :heads]) <= bound[:, :heads])
    got_k, got_v = (values(c.numpy(), kind).transpose(0, 2, 1, 3).reshape(-1, kv, d)[slots[at]] for c in (k, v))
    k_want = want[:, heads:heads + kv]
    assert np.all(np.abs(got_k - k_want) <= rounding(k_want, kind) * (1 + 2.0 ** -10) + bound[:, heads:heads + kv])
    assert np.all(np.abs(got_v - x[:, heads + kv:]) <= rounding(x[:, heads + kv:], kind))


def test_append_without_rotary_and_unaligned(paged):
    """No tables: q and k as they are, bit for bit.  Rows that start on any float, longer than the heads need; q in
    place of the rows'."""
    from cv3amd import _lib
    rng = np.random.default_rng(3)
    n, heads, kv, d, page, pages, ld = 11, 3, 2, 24, 4, 9, 7 * 24 + 5
    flat = rng.normal(size=1 + n * ld).astype(np.float32)
    slots = rng.permutation(pages * page)[:n].astype(I64)
    x = flat[1:].reshape(n, ld)[:, :7 * d].reshape(n, 7, d)
    k, v = paged.new_cache(pages, kv, page, d)
    fd, sd = dev(flat), dev(slots)
    _lib.call("paged_append", fd.ptr + 4, n, ld, heads, kv, d, None, sd.ptr, None, None, 0, 0, k.ptr, v.ptr, pages, page,
              None, 0, None)
    for c, rows in ((k, x[:, 3:5]), (v, x[:, 5:])):
        got = c.numpy().transpose(0, 2, 1, 3).reshape(-1, kv, d)
        assert np.array_equal(got[slots], rows)
        assert not got[np.setdiff1d(np.arange(pages * page), slots)].any()
    assert np.array_equal(paged.append(np.ascontiguousarray(x.reshape(n, -1)), heads, None, slots, None, None, k, v),
                          x[:, :heads])
    cos, sin = rotary(d, 30)
    positions = rng.integers(0, 30, n).astype(I32)
    cd, nd, pd = dev(cos), dev(sin), dev(positions)
    _lib.call("paged_append", fd.ptr + 4, n, ld, heads, kv, d, pd.ptr, sd.ptr, cd.ptr, nd.ptr, 30, 0, k.ptr, v.ptr, pages,
              page, fd.ptr + 4, ld, None)
    want, bound = turn(x.astype(np.float64), cos.astype(np.float64)[positions], sin.astype(np.float64)[positions])
    out = fd.numpy()[1:].reshape(n, ld)
    assert np.all(np.abs(out[:, :3 * d].reshape(n, 3, d) - want[:, :3]) <= bound[:, :3])
    assert np.array_equal(out[:, 3 * d:], flat[1:].reshape(n, ld)[:, 3 * d:])
    got = k.numpy().transpose(0, 2, 1, 3).reshape(-1, kv, d)[slots]
    assert np.all(np.abs(got - want[:, 3:5]) <= bound[:, 3:5])


@pytest.mark.parametrize("kind", ["float16", "bfloat16"])
def test_append_rounds_to_nearest_even_and_keeps_what_is_not_finite(paged, kind):
    eps = 2.0 ** -10 if kind == "float16" else 2.0 ** -7
    x = np.array([1 + eps / 2, 1 + 3 * eps / 2, 1 + eps / 2 + 2.0 ** -23, -(1 + eps / 2), np.inf, -np.inf, np.nan,
                  65519.9, 65520.0, 1e-8, -0.0, 3e38, 1e-40, 6e-8, 0.1, -7.3], np.float32)
    rows = np.concatenate([x, x, x])[None]
    k, v = paged.new_cache(1, 1, 1, 16, kind)
    paged.append(rows, 1, None, np.zeros(1, I64), None, None, k, v)
    want = stored(x, kind)[1]
    for c in (k, v):
        assert np.array_equal(values(c.numpy(), kind).reshape(-1), want, equal_nan=True)


# ------------------------------------------------------------------------------------------------
# attention
# ------------------------------------------------------------------------------------------------

def attention_ref(q, k, v, tables, lengths, starts, scale):
    """k, v (pages, kv heads, page, d) in float64; a key on a page outside the cache is not there."""
    b, h, d = q.shape
    pages, kv, page, _ = k.shape
    out = np.zeros((b, h, d))
    for i in range(b):
        hi = min(max(int(lengths[i]), 0), tables.shape[1] * page)
        lo = 0 if starts is None else min(max(int(starts[i]), 0), hi)
        at = np.arange(lo, hi)
        ids = tables[i, at // page]
        there = (ids >= 0) & (ids < pages)
        ids, row = ids[there], at[there] % page
        if not len(ids):
            continue
        for j in range(kv):
            qs = q[i, j * (h // kv):(j + 1) * (h // kv)].astype(np.float64)
            with np.errstate(invalid="ignore", over="ignore"):
                s = (qs @ k[ids, j, row].T) * scale
                e = np.exp(s - s.max(axis=1, keepdims=True))
                out[i, j * (h // kv):(j + 1) * (h // kv)] = e @ v[ids, j, row] / e.sum(axis=1, keepdims=True)
    return out


def batch(rng, lengths, blocks, page, extra=3):
    """Tables whose used entries are distinct pages in random order, the others -1."""
    used = [-(-max(0, min(int(n), blocks * page)) // page) for n in lengths]
    order = rng.permutation(sum(used) + extra).astype(I32)
    tables = np.full((len(lengths), blocks), -1, I32)
    at = 0
    for i, u in enumerate(used):
        tables[i, :u] = order[at:at + u]
        at += u
    return tables, sum(used) + extra


def check_attention(paged, lengths, h, kv, d, page, blocks, kind, starts=None, scale=None, sharp=1.5, seed=0):
    rng = np.random.default_rng([len(lengths), h, d, page, seed])
    lengths = np.asarray(lengths, I32)
    tables, pages = batch(rng, lengths, blocks, page)
    q = (sharp * rng.normal(size=(len(lengths), h, d))).astype(np.float32)
    ks, k64 = stored(rng.normal(size=(pages, kv, page, d)), kind)
    vs, v64 = stored(rng.normal(size=(pages, kv, page, d)), kind)
    starts = None if starts is None else np.asarray(starts, I32)
    got = paged.attention(q, dev(ks), dev(vs), tables, lengths, starts=starts, scale=scale)
    want = attention_ref(q, k64, v64, tables, lengths, starts, 1 / np.sqrt(d) if scale is None else scale)
    assert np.isfinite(got).all()
    for i in range(len(lengths)):
        if not want[i].any():
            assert not got[i].any(), f"sequence {i} sees nothing"
    tol = TOL
    if sharp > 2:       # scores off by ds change a weight p by p ds: d + 4 roundings of at most A = sum |q k| scale
        a = np.abs(q).sum(-1).max() * np.abs(k64).max() * (1 / np.sqrt(d) if scale is None else abs(scale))
        tol += 2 * (d + 4) * 2.0 ** -24 * a * np.abs(v64).max() / np.abs(want).max()
    assert rel_err(got, want) <= tol


HEADS = [(14, 2, 64), (16, 16, 64), (32, 8, 128), (20, 4, 80), (8, 1, 96), (1, 1, 8), (17, 1, 32), (40, 2, 128),
         (6, 3, 160), (4, 1, 192), (2, 2, 256), (33, 1, 256), (5, 5, 200)]
RAGGED = [0, 1, 15, 16, 17, 63, 64, 65, 200, 333]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("h,kv,d", HEADS)
def test_attention_ragged(paged, h, kv, d, kind):
    """A short table, and the same batch with a table long enough for the split form."""
    check_attention(paged, RAGGED, h, kv, d, 16, 21, kind)
    check_attention(paged, RAGGED, h, kv, d, 16, 300, kind)


@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 64, 100, 128, 1000])
@pytest.mark.parametrize("h,kv,d", [(14, 2, 64), (4, 4, 128)])
def test_attention_pages(paged, h, kv, d, page):
    check_attention(paged, [1, 77, 640, 129], h, kv, d, page, -(-700 // page), "float16")
    check_attention(paged, [1, 77, 2000, 129], h, kv, d, page, -(-4000 // page), "float32")


def test_the_largest_page(paged):
    """65536 keys a page, through all that address one: slots, the write, the attention, the move."""
    page, kv, d = 65536, 1, 16
    check_attention(paged, [70000, 5, 65536, 65537], 2, kv, d, page, 2, "float16")
    k, v = paged.new_cache(2, kv, page, d)
    own = np.array([[[0], [1]]], I32)
    total, _, _, slots, pos = paged.block_tables(np.array([60000, 65535], I32), np.array([3, 4], I32), page, None, None,
                                                 dev(own.reshape(2, 1)))
    assert list(slots) == [60000, 60001, 60002, 2 * 65536 - 1, -1, -1, -1] and list(total) == [60003, 65536]
    assert list(pos) == [60000, 60001, 60002, 65535, -1, -1, -1]
    rows = np.random.default_rng(18).normal(size=(7, 4 * d)).astype(np.float32)
    paged.append(rows, 2, None, slots, None, None, k, v)
    assert np.array_equal(k.numpy()[0, 0, 60000:60003], rows[:3, 2 * d:3 * d])
    assert np.array_equal(v.numpy()[1, 0, 65535], rows[3, 3 * d:])
    paged.beam_reorder(np.array([[0, 0]], I32), dev(own), own, np.array([65535], I32), k, v)
    assert np.array_equal(k.numpy()[1, 0, :65535], k.numpy()[0, 0, :65535]) and np.array_equal(
        v.numpy()[1, 0, 65535], rows[3, 3 * d:])


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("lengths", [[1], [64], [500], [1024], [1025], [4096], [4097], [30011], [131072],
                                     [0, 0, 0], [1] * 130, [70000, 3, 0, 900], list(range(0, 1500, 7))])
def test_attention_lengths(paged, lengths, kind):
    check_attention(paged, lengths, 14, 2, 64, 64, -(-max(lengths + [1]) // 64), kind)


@pytest.mark.parametrize("blocks", [63, 70])
def test_attention_windows(paged, blocks):
    """Keys before `starts` are not seen: windows that begin inside a page and a unit, that are empty, past the
    end, negative."""
    lengths = [500, 500, 500, 500, 64, 1000, 1000, 100, 0, 1, 900, 1008]
    starts = [0, 1, 499, 500, 63, 555, 960, 200, 0, 0, -4, 2**31 - 1]
    for kind in TYPES:
        check_attention(paged, lengths, 14, 2, 64, 16, blocks, kind, starts=starts)
    check_attention(paged, lengths, 8, 8, 128, 16, blocks, "float32", starts=starts)


@pytest.mark.parametrize("h,kv,d", [(14, 2, 64), (32, 8, 128)])
def test_attention_lengths_past_the_table(paged, h, kv, d):
    for blocks in (4, 100):
        check_attention(paged, [-1, 16 * blocks, 16 * blocks + 1, 2**31 - 1, -2**31], h, kv, d, 16, blocks, "float32")


def test_attention_scales(paged):
    for scale in (0.0, 1.0, -0.3, 0.125):
        check_attention(paged, [3, 333, 70], 14, 2, 64, 16, 30, "float32", scale=scale)
    # one key takes everything, or the scores pass the exponential's range many times over
    check_attention(paged, [3, 333, 3000], 14, 2, 64, 16, 200, "float32", sharp=300.0)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("blocks", [40, 80])
def test_attention_unseen_rows_reach_nothing(paged, kind, blocks):
    """NaN and infinities behind the last key, before the window, on pages of no sequence, and on the page that an
    absent id would clamp to; ids outside the cache are absent keys."""
    rng = np.random.default_rng(5)
    page, h, kv, d = 16, 14, 2, 64
    lengths, starts = np.array([0, 5, 37, 600, 300, 64], I32), np.array([0, 0, 20, 0, 33, 0], I32)
    tables, pages = batch(rng, lengths, blocks, page)
    tables[tables >= 0] += 1                                        # page 0 is nobody's
    pages += 1
    tables[3, 7], tables[3, 9], tables[4, 3] = -1, pages, 2**31 - 1
    tables[5, :4] = [-1, pages + 5, -2**31, -7]                     # nothing of this one is there
    seen = np.zeros((pages, page), bool)
    for i in range(len(lengths)):
        for j in range(starts[i], lengths[i]):
            if 0 <= tables[i, j // page] < pages:
                seen[tables[i, j // page], j % page] = True
    fill = rng.choice([np.nan, np.inf, -np.inf], size=(2, pages, kv, page, d))
    kvs = np.where(seen[None, :, None, :, None], rng.normal(size=(2, pages, kv, page, d)), fill)
    (ks, k64), (vs, v64) = (stored(x, kind) for x in kvs)
    q = rng.normal(size=(len(lengths), h, d)).astype(np.float32)
    got = paged.attention(q, dev(ks), dev(vs), tables, lengths, starts=starts)
    want = attention_ref(q, k64, v64, tables, lengths, starts, 0.125)
    assert not got[0].any() and not got[5].any()
    assert np.isfinite(want).all() and rel_err(got, want) <= TOL


@pytest.mark.parametrize("blocks", [10, 100])
def test_attention_seen_nan_reaches_its_heads_alone(paged, blocks):
    """A NaN among the seen keys is the outputs of its kv head's queries, one among the values its channel's; the
    other sequences and heads keep their results."""
    rng = np.random.default_rng(6)
    lengths = np.array([100, 100, 100], I32)
    tables, pages = batch(rng, lengths, blocks, 16)
    q = rng.normal(size=(3, 14, 64)).astype(np.float32)
    ks, vs = (rng.normal(size=(pages, 2, 16, 64)).astype(np.float32) for _ in range(2))
    ks[tables[1, 2], 0, 5, 7] = np.nan
    vs[tables[2, 6], 1, 3, 40] = np.nan
    got = paged.attention(q, dev(ks), dev(vs), tables, lengths)
    bad = np.zeros(got.shape, bool)
    bad[1, :7] = True
    bad[2, 7:, 40] = True
    assert np.array_equal(np.isnan(got), bad)
    ks[np.isnan(ks)], vs[np.isnan(vs)] = 0.0, 0.0
    want = attention_ref(q, ks.astype(np.float64), vs.astype(np.float64), tables, lengths, None, 0.125)
    assert rel_err(got[~bad], want[~bad]) <= TOL


def test_attention_shared_pages_and_strided_rows(paged):
    """Sequences that share pages (a common prompt), queries inside wider rows, any alignment."""
    from cv3amd import _lib
    rng = np.random.default_rng(7)
    for blocks in (20, 90):
        b, h, kv, d, page, pages = 4, 14, 2, 64, 16, 25
        tables = rng.integers(0, pages, (b, blocks)).astype(I32)
        lengths = np.array([300, 17, 320, 111], I32)
        ks, vs = (rng.normal(size=(pages, kv, page, d)).astype(np.float32) for _ in range(2))
        ldq, ldo = h * d + 2 * kv * d + 3, h * d + 7
        flat = rng.normal(size=1 + b * ldq).astype(np.float32)
        q = flat[1:].reshape(b, ldq)[:, :h * d].reshape(b, h, d)
        fd, out = dev(flat), dev(np.full(3 + b * ldo, 7.5, np.float32))
        kd, vd, td, nd = dev(ks), dev(vs), dev(tables), dev(lengths)
        _lib.call("paged_attention", fd.ptr + 4, ldq, b, h, kv, d, 0, kd.ptr, vd.ptr, pages, page, td.ptr, blocks, nd.ptr,
                  None, ctypes.c_float(0.125), out.ptr + 12, ldo, None)
        got = out.numpy()
        assert np.all(got[:3] == 7.5) and np.all(got[3:].reshape(b, ldo)[:, h * d:] == 7.5)
        want = attention_ref(q, ks.astype(np.float64), vs.astype(np.float64), tables, lengths, None, 0.125)
        assert rel_err(got[3:].reshape(b, ldo)[:, :h * d].reshape(b, h, d), want) <= TOL


def test_attention_offsets_past_32_bits(paged):
    """A cache of more than 2^31 elements, its last pages in use."""
    from cv3amd.device import DeviceArray
    rng = np.random.default_rng(8)
    kv, page, d = 2, 64, 128
    pages = (1 << 31) // (kv * page * d) + 40
    k, v = (DeviceArray((pages, kv, page, d), np.float16).zero_() for _ in range(2))
    ids = np.concatenate([rng.permutation(np.arange(pages - 30, pages))[:20], [0, 5]]).astype(I32)
    ks, vs = (rng.normal(size=(len(ids), kv, page, d)).astype(np.float16) for _ in range(2))
    for i, p in enumerate(ids):
        k.rows(int(p), int(p) + 1).copy_from(ks[i])
        v.rows(int(p), int(p) + 1).copy_from(vs[i])
    small = np.arange(22, dtype=I32)[None]
    q = rng.normal(size=(1, 8, d)).astype(np.float32)
    n = np.array([22 * 64 - 9], I32)
    want = attention_ref(q, ks.astype(np.float64), vs.astype(np.float64), small, n, None, 1 / np.sqrt(d))
    assert rel_err(paged.attention(q, k, v, ids[None], n), want) <= TOL
    # and the write and the move at such offsets
    rows = rng.normal(size=(2, (1 + 2 * kv) * d)).astype(np.float32)
    slots = np.array([(pages - 1) * page + 63, (pages - 2) * page], I64)
    paged.append(rows, 1, None, slots, None, None, k, v)
    x = rows.reshape(2, 5, d).astype(np.float16)
    assert np.array_equal(k.rows(pages - 1, pages).numpy()[0, :, 63], x[0, 1:3])
    assert np.array_equal(v.rows(pages - 2, pages - 1).numpy()[0, :, 0], x[1, 3:])
    own = np.array([[[pages - 1], [pages - 2]]], I32)
    paged.beam_reorder(np.array([[1, 1]], I32), dev(own), own, np.array([1], I32), k, v)
    assert np.array_equal(v.rows(pages - 1, pages).numpy()[0, :, 0], x[1, 3:])
    assert np.array_equal(k.rows(pages - 1, pages).numpy()[0, :, 63], x[0, 1:3])


# ------------------------------------------------------------------------------------------------
# beam selection
# ------------------------------------------------------------------------------------------------

def select_ref(logits, scores, done, stop, ban, pad):
    r, w, v = logits.shape
    out = []
    for i in range(r):
        every = []
        for b in range(w):
            s = float(scores[i, b])
            if done[i, b]:
                every.append((-np.inf if np.isnan(s) else s, -b, np.inf, 0, pad, b, True))
                continue
            x = logits[i, b].astype(np.float64)
            with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
                top = x.max()
                lse = top + np.log(np.exp(x - top).sum())
                value = s + (x - lse)
            value = np.where(np.isnan(value), -np.inf, value)
            key = np.where(np.isnan(x), -np.inf, x)
            ids = np.arange(v)
            ids = ids[~((ids >= ban[0]) & (ids < ban[1]))]
            ids = ids[np.argsort(-key[ids], kind="stable")][:w]
            every += [(value[t], -b, key[t], -t, t, b, stop[0] <= t < stop[1]) for t in ids]
        out.append(sorted(every, key=lambda c: c[:4], reverse=True)[:w])
    get = lambda n, t: np.array([[c[n] for c in row] for row in out], t)  # noqa: E731
    return get(4, I64), get(5, I32), get(0, np.float64), get(6, U8)


def check_select(paged, logits, scores, done, stop, ban=(0, 0), pad=None):
    logits, scores, done = np.asarray(logits, np.float32), np.asarray(scores, np.float32), np.asarray(done, U8)
    want = select_ref(logits, scores, done, stop, ban, stop[0] if pad is None else pad)
    got = paged.beam_select(logits, scores, done, stop, ban, pad)
    for g, w, name in zip(got, want, ("tokens", "parents", "scores", "done")):
        if name == "scores":
            with np.errstate(invalid="ignore"):
                off = np.abs(g - w)
            ok = (g == w) | (off <= 2.0 ** -23 * np.abs(w) + 1e-6)
            assert ok.all(), (g, w)
        else:
            assert np.array_equal(g, w), (name, g, w)


@pytest.mark.parametrize("requests,beams,vocab", [(1, 1, 1), (1, 1, 6761), (1, 4, 6761), (3, 2, 2), (2, 16, 16), (5, 3, 255),
                                                  (2, 8, 257), (1, 16, 8191), (1, 16, 8192), (2, 5, 8193), (24, 8, 20011),
                                                  (1, 16, 524288), (2, 16, 151936), (130, 4, 700)])
def test_select(paged, requests, beams, vocab):
    rng = np.random.default_rng([requests, beams, vocab])
    logits = (2.5 * rng.normal(size=(requests, beams, vocab))).astype(np.float32)
    scores = (rng.normal(size=(requests, beams)) * 2 - 20).astype(np.float32)
    none = np.zeros((requests, beams))
    stop = (vocab - 1, vocab)
    check_select(paged, logits, scores, none, stop)
    check_select(paged, logits, scores, rng.random((requests, beams)) < 0.4, stop)
    check_select(paged, logits, scores, none + 1, stop, pad=12345)
    if vocab >= 4 * beams:
        best = int(logits[0, 0].argmax())
        lo = max(0, min(best - beams, vocab - 2 * beams))
        check_select(paged, logits, scores, none, (best, best + 1), ban=(lo, lo + 2 * beams))
        check_select(paged, logits, scores, none, (0, vocab))                        # whatever is chosen ends
    first = np.full((requests, beams), -np.inf)                                      # the first step: one beam lives
    first[:, 0] = 0.0
    check_select(paged, logits, first, none, stop)


def test_select_ties(paged):
    """Equal values: the lower beam, then the lower token.  All of a row alike is the most that can tie."""
    rng = np.random.default_rng(1)
    for vocab in (40, 1000, 8192, 20000):
        same = np.zeros((2, 8, vocab))
        score = np.zeros((2, 8))
        check_select(paged, same, score, score, (vocab, vocab))
        check_select(paged, rng.integers(0, 3, same.shape), score, score, (vocab, vocab))
        check_select(paged, -rng.integers(0, 2, same.shape) * 0.0, score, score, (vocab, vocab))    # -0 is 0
        check_select(paged, np.sort(rng.normal(size=same.shape)), score, score, (vocab, vocab))     # all of one thread
        check_select(paged, np.sort(rng.normal(size=same.shape))[..., ::-1], score, score, (vocab, vocab))
        few = np.full(same.shape, -np.inf)
        few[:, :, ::vocab // 3] = 0.0                                                # fewer than the beams
        check_select(paged, few, score, score, (vocab, vocab))
    # far below one in size: a sum with the score tells them apart no more, the logits do
    tiny = rng.permutation(200).astype(np.float32) * np.float32(1e-30)
    check_select(paged, np.broadcast_to(tiny, (1, 4, 200)), np.zeros((1, 4)), np.zeros((1, 4)), (200, 200))


def test_select_values_that_are_no_numbers(paged):
    rng = np.random.default_rng(2)
    x = rng.normal(size=(8, 4, 3000)).astype(np.float32)
    s = rng.normal(size=(8, 4)).astype(np.float32)
    none = np.zeros((8, 4))
    x[0, 1, 77] = np.nan                # the row is out of the search
    x[1, 2] = -np.inf                   # nothing to choose
    x[2, 0, 5] = np.inf
    x[3, :, 10:] = -np.inf              # ten tokens, four beams
    x[4, 3, ::2] = np.nan
    s[5, 0], s[5, 1] = np.nan, -np.inf
    s[6] = -np.inf                      # every beam is out
    x[7] = np.finfo(np.float32).min     # a mask of the type's lowest value
    x[7, :, 42] = 0.0
    check_select(paged, x, s, none, (2999, 3000))
    check_select(paged, x, s, rng.random((8, 4)) < 0.5, (2999, 3000))
    check_select(paged, np.full((1, 3, 50), np.nan), np.zeros((1, 3)), np.zeros((1, 3)), (0, 1))
    big = rng.normal(size=(2, 4, 500)) * 1e37
    check_select(paged, big, np.zeros((2, 4)), np.zeros((2, 4)), (0, 1))


def test_select_in_place(paged):
    rng = np.random.default_rng(4)
    x, s = rng.normal(size=(3, 4, 5000)).astype(np.float32), rng.normal(size=(3, 4)).astype(np.float32)
    d = (rng.random((3, 4)) < 0.3).astype(U8)
    want = paged.beam_select(x, s, d, (9, 3000))
    sd, dd, tok, par = dev(s), dev(d), dev(np.zeros((3, 4), I64)), dev(np.zeros((3, 4), I32))
    got = paged.beam_select(dev(x), sd, dd, (9, 3000), out=(tok, par, sd, dd))
    assert got[2] is sd and got[3] is dd
    for g, w in zip(got, want):
        assert np.array_equal(g.numpy(), w)


# ------------------------------------------------------------------------------------------------
# beam reordering
# ------------------------------------------------------------------------------------------------

def reorder_ref(parents, tables, own, lengths, caches, page):
    """caches: (layers, pages, kv heads, page, d) arrays of any type."""
    tables, new = tables.copy(), [c.copy() for c in caches]
    r, w, blocks = tables.shape
    pages = caches[0].shape[1]
    old = tables.copy()
    for i in range(r):
        n = min(max(int(lengths[i]), 0), blocks * page)
        full, rest = divmod(n, page)
        for b in range(w):
            p = int(parents[i, b])
            if not 0 <= p < w:
                continue
            tables[i, b, :full], tables[i, b, full:] = old[i, p, :full], own[i, b, full:]
            if rest:
                to, fr = int(own[i, b, full]), int(own[i, p, full])
                if 0 <= to < pages and 0 <= fr < pages:
                    for c, o in zip(new, caches):
                        c[:, to, :, :rest] = o[:, fr, :, :rest]
    return tables, new


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("requests,beams,page,blocks,layers,kv,d", [
    (1, 4, 16, 6, 3, 2, 64), (3, 1, 16, 4, 1, 1, 8), (5, 16, 5, 7, 2, 3, 24), (2, 8, 64, 3, 24, 2, 64), (4, 3, 1, 9, 2, 2, 16),
    (2, 5, 100, 2, 2, 1, 256), (1, 2, 8, 700, 1, 1, 8), (33, 2, 24, 3, 1, 4, 80)])
def test_reorder(paged, requests, beams, page, blocks, layers, kv, d, kind):
    rng = np.random.default_rng([requests, beams, page])
    pages = requests * beams * blocks + 2
    own = rng.permutation(pages)[:requests * beams * blocks].reshape(requests, beams, blocks).astype(I32)
    tables = rng.integers(0, pages, own.shape).astype(I32)
    caches = [stored(rng.normal(size=(layers, pages, kv, page, d)), kind)[0] for _ in range(2)]
    k, v = dev(caches[0]), dev(caches[1])
    td = dev(tables)
    lengths = rng.integers(0, page * blocks + 1, requests).astype(I32)
    edges = [0, page, page * blocks, 1, page * blocks - 1, page * blocks + 9, -3]
    for step, parents in enumerate([rng.integers(0, beams, (requests, beams)), np.zeros((requests, beams)),
                                    np.tile(np.roll(np.arange(beams), 1), (requests, 1)),
                                    rng.integers(-2, beams + 2, (requests, beams))]):
        if step == 2:
            lengths[:len(edges)] = edges[:requests]
        parents = np.asarray(parents, I32)
        tables, caches = reorder_ref(parents, tables, own, lengths, caches, page)
        paged.beam_reorder(parents, td, own, lengths, k, v)
        assert np.array_equal(td.numpy(), tables)
        for c, w in zip((k, v), caches):
            assert np.array_equal(c.numpy().view(np.uint8), w.view(np.uint8))


def test_reorder_pages_outside_the_cache_are_not_copied(paged):
    rng = np.random.default_rng(9)
    own = np.arange(16).reshape(1, 4, 4).astype(I32)
    own[0, 1, 2], own[0, 3, 2] = -1, 16
    tables = own.copy()
    caches = [rng.normal(size=(16, 2, 8, 16)).astype(np.float32) for _ in range(2)]
    k, v, td = dev(caches[0]), dev(caches[1]), dev(tables)
    parents = np.array([[1, 0, 3, 2]], I32)
    want, new = reorder_ref(parents, tables, own, [21], [c[None] for c in caches], 8)
    paged.beam_reorder(parents, td, own, np.array([21], I32), k, v)
    assert np.array_equal(td.numpy(), want)
    assert np.array_equal(k.numpy(), new[0][0]) and np.array_equal(v.numpy(), new[1][0])


# ------------------------------------------------------------------------------------------------
# infinities among what is seen; streams, threads and graphs; the operators as one step
# ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("blocks", [13, 150])
@pytest.mark.parametrize("h,kv,d", [(14, 2, 64), (4, 2, 128)])
def test_attention_seen_infinities(paged, h, kv, d, blocks, kind):
    """An infinite key channel makes a score +inf (NaN outputs, inf - inf) or -inf (weight zero) by the query's sign;
    an infinite value is its channel's output.  Two-byte caches form such outputs in float32."""
    rng = np.random.default_rng([d, blocks])
    lengths = np.array([200, 200, 200, 200, 200], I32)
    tables, pages = batch(rng, lengths, blocks, 16)
    q = rng.normal(size=(5, h, d)).astype(np.float32)
    ks, vs = (rng.normal(size=(pages, kv, 16, d)).astype(np.float32) for _ in range(2))
    ks[tables[1, 2], 0, 5, 7] = np.inf
    ks[tables[2, 12], 1, 3, d - 1] = -np.inf
    vs[tables[3, 0], 0, 0, 1] = -np.inf
    vs[tables[3, 6], 1, 15, 9], vs[tables[3, 9], 1, 2, 9] = np.inf, -np.inf
    q[4, 1, 3] = np.inf
    (ks, k64), (vs, v64) = stored(ks, kind), stored(vs, kind)
    with np.errstate(invalid="ignore"):
        want = attention_ref(q, k64, v64, tables, lengths, None, 1 / np.sqrt(d))
    got = paged.attention(q, dev(ks), dev(vs), tables, lengths)
    assert np.isnan(want).any() and np.isinf(want).any()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[np.isinf(want)], want[np.isinf(want)])
    fine = np.isfinite(want)
    assert rel_err(got[fine], want[fine]) <= TOL


@pytest.mark.parametrize("kind", TYPES)
def test_attention_sizes_of_queries(paged, kind):
    """Queries from 2^-120 to 2^40 beside each other: each head has its own scale."""
    rng = np.random.default_rng(11)
    for blocks in (4, 90):
        lengths = np.array([50, 17], I32)
        tables, pages = batch(rng, lengths, blocks, 16)
        q = rng.normal(size=(2, 14, 64)) * 2.0 ** np.linspace(-120, 0, 14)[None, :, None]
        q[1, 3] = 0.0
        q[1, 5] *= 2.0 ** 85         # scores of 2^40 and more: one key takes all
        (ks, k64), (vs, v64) = (stored(rng.normal(size=(pages, 2, 16, 64)), kind) for _ in range(2))
        q = q.astype(np.float32)
        want = attention_ref(q, k64, v64, tables, lengths, None, 0.125)
        assert rel_err(paged.attention(q, dev(ks), dev(vs), tables, lengths), want) <= TOL


@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
@pytest.mark.parametrize("blocks", [6, 300])
@pytest.mark.parametrize("gap", [1.0, 5.0, 7.9, 30.0])
def test_attention_values_near_the_largest_float(paged, kind, blocks, gap):
    """A key whose weight is 2^gap times those before it, with values near the largest float: weights past one would
    pass it."""
    rng = np.random.default_rng(16)
    lengths = np.array([90], I32)
    tables, pages = batch(rng, lengths, blocks, 16)
    q = np.zeros((1, 2, 64), np.float32)
    q[:, :, 0] = 1.0
    ks, vs = np.zeros((2, pages, 2, 16, 64), np.float32)
    ks[tables[0, 5], :, 3, 0] = gap * np.log(2) * 8             # scale 1/8
    vs[tables[0, 5], :, 3, ::2], vs[tables[0, 5], :, 3, 1::2] = 3e38, -3e38
    for i in range(5):      # one such key more in each strip and wave, their values' sum within the float's range
        ks[tables[0, i], :, 9, 0] = gap * np.log(2) * 8
        vs[tables[0, i], :, 9] = 5e36
    (ks, k64), (vs, v64) = stored(ks, kind), stored(vs, kind)
    want = attention_ref(q, k64, v64, tables, lengths, None, 0.125)
    got = paged.attention(q, dev(ks), dev(vs), tables, lengths)
    assert np.isfinite(want).all() and rel_err(got, want) <= TOL


@pytest.mark.parametrize("vocab", [500, 6761, 30000])
def test_select_bans_whole_slices(paged, vocab):
    rng = np.random.default_rng(vocab)
    x = rng.normal(size=(2, 4, vocab))
    s, none = rng.normal(size=(2, 4)), np.zeros((2, 4))
    for ban in ((0, vocab - 4), (4, vocab), (2, vocab - 2), (-5, 10), (vocab - 10, vocab + 50), (7, 7), (9, 3),
                (0, vocab // 2)):
        check_select(paged, x, s, none, (vocab - 3, vocab), ban=ban)


def attention_inputs(rng, b, n, blocks, kind="bfloat16", h=14, kv=2, d=64, page=16):
    lengths = rng.integers(1, n + 1, b).astype(I32)
    tables, pages = batch(rng, lengths, blocks, page)
    q = rng.normal(size=(b, h, d)).astype(np.float32)
    (ks, k64), (vs, v64) = (stored(rng.normal(size=(pages, kv, page, d)), kind) for _ in range(2))
    want = attention_ref(q, k64, v64, tables, lengths, None, 1 / np.sqrt(d))
    return [dev(a) for a in (q, ks, vs, tables, lengths)], want


def test_calls_on_an_explicit_stream(gpu, paged):
    """The C entries on a stream of the caller's own, beside the thread's: scratch and results are that stream's."""
    from cv3amd import _lib, device
    rng = np.random.default_rng(12)
    (q, k, v, t, n), want = attention_inputs(rng, 9, 900, 120)
    out, st = dev(np.zeros((9, 14, 64), np.float32)), device.Stream()
    x, s = rng.normal(size=(2, 4, 9000)).astype(np.float32), rng.normal(size=(2, 4)).astype(np.float32)
    ref = select_ref(x, s, np.zeros((2, 4)), (0, 1), (0, 0), 0)
    xd, sd, dd = dev(x), dev(s), dev(np.zeros((2, 4), U8))
    tok, par, so, do = (dev(np.zeros((2, 4), t_)) for t_ in (I64, I32, np.float32, U8))
    for _ in range(3):
        _lib.call("paged_attention", q.ptr, 14 * 64, 9, 14, 2, 64, _lib.BF16, k.ptr, v.ptr, k.shape[0], 16, t.ptr, 120,
                  n.ptr, None, ctypes.c_float(0.125), out.ptr, 14 * 64, st.handle)
        _lib.call("beam_select", xd.ptr, 2, 4, 9000, sd.ptr, dd.ptr, 0, 1, 0, 0, 0, tok.ptr, par.ptr, so.ptr, do.ptr,
                  st.handle)
    _lib.call("stream_sync", st.handle)
    assert rel_err(out.numpy(), want) <= TOL
    assert np.array_equal(tok.numpy(), ref[0]) and np.array_equal(par.numpy(), ref[1])


def test_calls_from_four_threads(gpu, paged):
    import threading
    from cv3amd import device
    wrong = []

    def work(i):
        try:
            rng = np.random.default_rng([13, i])
            ins, want = attention_inputs(rng, 5 + i, 700 + 100 * i, 150)
            x = rng.normal(size=(3, 4, 7000 + i)).astype(np.float32)
            s, d = rng.normal(size=(3, 4)).astype(np.float32), np.zeros((3, 4), U8)
            ref = select_ref(x, s, d, (0, 1), (0, 0), 0)
            xd, sd, dd = dev(x), dev(s), dev(d)
            outs = [(paged.attention(*ins), paged.beam_select(xd, sd, dd, (0, 1))) for _ in range(20)]
            device.synchronize()
            for o, sel in outs:
                if rel_err(o.numpy(), want) > TOL or not np.array_equal(sel[0].numpy(), ref[0]):
                    wrong.append(i)
        except Exception as e:      # noqa: BLE001
            wrong.append(repr(e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_attention_captured_without_scratch(gpu, paged):
    """A capture takes scratch from the allocator's cache alone; where there is none, long caches run one workgroup a
    pair.  The graph replays with eager calls in between."""
    from cv3amd import _lib, device
    rng = np.random.default_rng(15)
    ins, want = attention_inputs(rng, 4, 1500, 200)
    out = dev(np.zeros((4, 14, 64), np.float32))
    device.synchronize()
    _lib.call("empty_cache")
    g = device.Graph()
    with g:
        paged.attention(*ins, out=out)
    for _ in range(3):
        out.zero_()
        g.launch()
        assert rel_err(out.numpy(), want) <= TOL
        assert rel_err(paged.attention(*ins).numpy(), want) <= TOL


def test_attention_of_empty_batches(paged):
    """Nothing to see at all, with tables long enough for the split form."""
    for lengths in ([0], [0, 0, 0], [0] * 300):
        check_attention(paged, lengths, 14, 2, 64, 16, 300, "float32")
    check_attention(paged, [500, 40, 7], 4, 2, 128, 16, 300, "bfloat16", starts=[500, 41, 2**31 - 1])
    check_attention(paged, [0, 4000, 0], 14, 2, 64, 16, 300, "float16")


def test_attention_in_place_of_its_queries(paged):
    rng = np.random.default_rng(17)
    for blocks in (60, 400):
        (q, k, v, t, n), want = attention_inputs(rng, 7, 900, blocks)
        assert paged.attention(q, k, v, t, n, out=q) is q
        assert rel_err(q.numpy(), want) <= TOL


@pytest.mark.parametrize("b", [63, 64, 65, 257, 1000, 4097, 9000])
def test_attention_large_batches(paged, b):
    """More sequences than lanes, and than lanes can hold one each: shares are found in a batch of any size."""
    rng = np.random.default_rng(b)
    lengths = np.where(rng.random(b) < 0.4, 0, rng.integers(1, 60, b))
    lengths[rng.integers(0, b, 3)] = 700
    check_attention(paged, lengths, 2, 1, 16, 16, 1700, "float16")


class Step:
    """One beam-search step over a one-layer model that is nothing but the operators: rows and logits are drawn from
    tables by token, so that every step's inputs follow from the choices before it."""

    R, W, V, H, KV, D, PAGE, BLOCKS, LAYERS = 3, 4, 300, 6, 2, 32, 4, 8, 2

    def __init__(self, paged, kind):
        self.paged, self.kind = paged, kind
        rng = np.random.default_rng(14)
        rows = self.R * self.W
        pages = rows * self.BLOCKS
        self.own = rng.permutation(pages).reshape(self.R, self.W, self.BLOCKS).astype(I32)
        self.qkv = rng.normal(size=(rows, (self.H + 2 * self.KV) * self.D)).astype(np.float32)
        self.logits = rng.normal(size=(self.R, self.W, self.V)).astype(np.float32)
        self.k0 = rng.normal(size=(2, self.LAYERS, pages, self.KV, self.PAGE, self.D)).astype(np.float32)
        self.cos, self.sin = rotary(self.D, 64)

    def state(self):
        rows = self.R * self.W
        s = dict(tables=dev(self.own), own=dev(self.own), k=dev(stored(self.k0[0], self.kind)[0]),
                 v=dev(stored(self.k0[1], self.kind)[0]), len_r=dev(np.array([0, 3, 9], I32)),
                 len_w=dev(np.repeat(np.array([0, 3, 9], I32), self.W)), one_r=dev(np.ones(self.R, I32)),
                 one_w=dev(np.ones(rows, I32)), qkv=dev(self.qkv), logits=dev(self.logits),
                 scores=dev(np.zeros((self.R, self.W), np.float32)), done=dev(np.zeros((self.R, self.W), U8)),
                 cos=dev(self.cos), sin=dev(self.sin), total_r=dev(np.zeros(self.R, I32)), total_w=dev(np.zeros(rows, I32)),
                 starts=dev(np.zeros(rows + 1, I32)), slots=dev(np.zeros(rows, I64)), pos=dev(np.zeros(rows, I32)),
                 r_starts=dev(np.zeros(self.R + 1, I32)), r_slots=dev(np.zeros(self.R, I64)),
                 r_pos=dev(np.zeros(self.R, I32)), r_tables=dev(np.zeros((self.R, self.BLOCKS), I32)),
                 q=dev(np.zeros((rows, self.H, self.D), np.float32)), out=dev(np.zeros((rows, self.H, self.D), np.float32)),
                 tokens=dev(np.zeros((self.R, self.W), I64)), parents=dev(np.zeros((self.R, self.W), I32)))
        return s

    def run(self, s):
        """Enqueues one step: the new token's slots, the cache write of both layers, attention, the choice, the
        reordering.  Every beam's pages are reserved from the start: slots come from `own`, none is taken."""
        from cv3amd import _lib
        p, rows = self.paged, self.R * self.W
        flat = s["tables"].reshape(rows, self.BLOCKS)
        p.block_tables(s["len_w"], s["one_w"], self.PAGE, None, None, s["own"].reshape(rows, self.BLOCKS),
                       out=(s["total_w"], None, s["starts"], s["slots"], s["pos"]))
        for i in range(self.LAYERS):
            k, v = (s[c].rows(i, i + 1).reshape(s[c].shape[1:]) for c in "kv")
            p.append(s["qkv"], self.H, s["pos"], s["slots"], s["cos"], s["sin"], k, v, out=s["q"])
            p.attention(s["q"], k, v, flat, s["total_w"], out=s["out"])
        p.beam_select(s["logits"], s["scores"], s["done"], (290, 300), out=(s["tokens"], s["parents"], s["scores"], s["done"]))
        _lib.call("copy_d2d", s["len_w"].ptr, s["total_w"].ptr, 4 * rows, None)
        p.block_tables(s["len_r"], s["one_r"], self.PAGE, None, None, s["r_tables"],
                       out=(s["total_r"], None, s["r_starts"], s["r_slots"], s["r_pos"]))
        _lib.call("copy_d2d", s["len_r"].ptr, s["total_r"].ptr, 4 * self.R, None)
        p.beam_reorder(s["parents"], s["tables"], s["own"], s["len_r"], s["k"], s["v"])


@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
def test_steps_captured_and_replayed(gpu, paged, kind):
    """A captured step, replayed with eager work in between, leaves what the same steps leave eagerly; two graphs of
    two states replay in turn (each has its own scratch)."""
    from cv3amd import device
    step = Step(paged, kind)

    names = ("tables", "k", "v", "len_w", "len_r", "scores", "done", "out", "tokens", "parents")
    eager = step.state()
    want = []
    for _ in range(6):
        step.run(eager)
        want.append({n: eager[n].numpy() for n in names})
    states, graphs = [step.state(), step.state()], []
    other = step.state()
    for s in states:
        step.run(other)                 # leaves scratch in the allocator's cache, which the capture then owns
        g = device.Graph()
        with g:
            step.run(s)
        graphs.append(g)
    for i in range(6):
        for s, g in zip(states, graphs):
            g.launch()
            step.run(other)             # eager calls between the replays
            if i == 3:
                device.synchronize()
            for n in names:
                got = s[n].numpy()
                assert np.array_equal(got.view(np.uint8), want[i][n].view(np.uint8)), (i, n)


@pytest.mark.parametrize("kind", TYPES)
def test_steps_against_the_reference(gpu, paged, kind):
    """The same steps followed in NumPy: slots, cache, attention outputs, choices and tables after every step."""
    step = Step(paged, kind)
    s = step.state()
    R, W, H, KV, D, PAGE = step.R, step.W, step.H, step.KV, step.D, step.PAGE
    tables, n = step.own.copy(), np.array([0, 3, 9])
    k, v = (values(stored(c, kind)[0], kind) for c in step.k0)
    scores, done = np.zeros((R, W), np.float32), np.zeros((R, W), U8)
    x = step.qkv.astype(np.float64).reshape(R * W, H + 2 * KV, D)
    for _ in range(6):
        step.run(s)
        at = np.repeat(n, W)
        turned, _ = turn(x, step.cos.astype(np.float64)[at], step.sin.astype(np.float64)[at])
        for i in range(R * W):
            p = step.own.reshape(R * W, -1)[i, at[i] // PAGE]
            k[:, p, :, at[i] % PAGE], v[:, p, :, at[i] % PAGE] = turned[i, H:H + KV], x[i, H + KV:]
        n = n + 1
        # the last layer's attention, over the tables before the reordering
        want = attention_ref(turned[:, :H], k[-1], v[-1], tables.reshape(R * W, -1), np.repeat(n, W), None, 1 / np.sqrt(D))
        # a stored key is off by half a step of its type: the scores by that share of sum |q k|, the values by theirs
        eps = {"float32": 2.0 ** -23, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}[kind]
        most = np.abs(turned[:, :H]).sum(-1).max() * np.abs(k).max() / np.sqrt(D)
        assert np.abs(s["out"].numpy() - want).max() <= (2 * eps * most + eps + TOL) * np.abs(v).max()
        tok, par, sc, done = select_ref(step.logits, scores, done, (290, 300), (0, 0), 290)
        scores = sc.astype(np.float32)
        assert np.array_equal(s["tokens"].numpy(), tok) and np.array_equal(s["parents"].numpy(), par)
        assert np.array_equal(s["done"].numpy(), done)
        assert np.abs(s["scores"].numpy() - scores).max() <= 1e-5
        scores = s["scores"].numpy()
        tables, (k, v) = reorder_ref(par, tables, step.own, n, [k, v], PAGE)
        assert np.array_equal(s["tables"].numpy(), tables)
        assert np.array_equal(s["len_r"].numpy(), n) and np.array_equal(s["len_w"].numpy(), np.repeat(n, W))
    for c, w in ((s["k"], k), (s["v"], v)):
        assert np.abs(values(c.numpy(), kind) - w).max() <= 2 * eps * np.abs(w).max()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("blocks", [4, 13, 400])
@pytest.mark.parametrize("h,kv,d", [(14, 2, 64), (4, 2, 128)])
def test_attention_of_scores_that_are_all_minus_infinity(paged, h, kv, d, blocks, kind):
    """Keys that are there and whose scores are -inf every one: the softmax is 0 / 0, NaN, and not the zeros of a
    sequence with no key to see.  One score that is a number takes it all, wherever it lies."""
    rng = np.random.default_rng([d, blocks, 2])
    n = min(16 * blocks, 3000) - 3
    lengths = np.array([n, n, n, 1, n, n, 0, n], I32)
    starts = np.array([0, 0, n - 9, 0, 0, 20, 0, 0], I32)
    tables, pages = batch(rng, lengths, blocks, 16)
    q = rng.normal(size=(8, h, d)).astype(np.float32)
    q[..., 0] = 1.0
    ks, vs = (rng.normal(size=(pages, kv, 16, d)).astype(np.float32) for _ in range(2))

    def away(i, lo, hi, heads=slice(None)):
        for j in range(lo, hi):
            ks[tables[i, j // 16], heads, j % 16, 0] = -np.inf

    away(0, 0, n)                       # every key
    away(1, 0, n, 1)                    # of one kv head
    away(2, n - 9, n)                   # every key of a window
    away(3, 0, 1)                       # the only one
    away(4, 0, n - 1)                   # all but the last, and all but the first
    away(5, 21, n)
    away(7, 0, n)                       # every key that is there: pages of the others are not
    tables[7, ::2] = -1
    (ks, k64), (vs, v64) = stored(ks, kind), stored(vs, kind)
    with np.errstate(invalid="ignore"):
        want = attention_ref(q, k64, v64, tables, lengths, starts, 1 / np.sqrt(d))
    assert list(np.isnan(want).all(axis=(1, 2))) == [True, False, True, True, False, False, False, blocks > 1]
    assert np.isnan(want[1, h // 2:]).all() and not want[6].any()
    got = paged.attention(q, dev(ks), dev(vs), tables, lengths, starts=starts)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = ~np.isnan(want)
    assert rel_err(got[fine], want[fine]) <= TOL
