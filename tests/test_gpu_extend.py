"""Attention of several new tokens per sequence over the paged cache, on the GPU, against a plain NumPy form in 64 bits.

Tolerance: the float32 bar of the other kernels, max |error| / max |reference| <= 1e-5, against float64 of the stored
(rounded) keys and values.  Operands enter the products within 2^-22, sums are float32: with |q k| of a few units a score
is off by a few 2^-21, and a weight by as much of itself.  Where scores are larger (``sharp``), one that is off by ds
changes its weight p by p ds, and ds is at most d + 4 roundings of 2^-23 of A = sum |q k| scale: added below.
"""

import ctypes

import numpy as np
import pytest

from conftest import rel_err
from test_gpu_paged import TYPES, bf16_bits, dev, stored, values

pytestmark = pytest.mark.gpu

TOL = 1e-5
I32 = np.int32


@pytest.fixture(scope="module")
def paged(gpu):
    from cv3amd import paged
    return paged


def extend_ref(q, k, v, tables, lengths, starts, window, scale, out):
    """k, v (pages, kv heads, page, d) in float64; a key on a page outside the cache is not there.  Rows of no sequence
    stay as ``out`` has them."""
    n, h, d = q.shape
    pages, kv, page, _ = k.shape
    out, g = np.array(out, np.float64), h // kv
    for b in range(len(lengths)):
        r0, r1 = int(starts[b]), int(starts[b + 1])
        total = min(max(int(lengths[b]), 0), tables.shape[1] * page)
        if r1 <= r0:
            continue
        out[r0:r1] = 0.0
        at = np.arange(total)
        ids = tables[b, at // page]
        there = (ids >= 0) & (ids < pages)
        at, ids = at[there], ids[there]
        if not len(at):
            continue
        pos = np.arange(total - (r1 - r0), total)[:, None]
        seen = (at <= pos) & ((at > pos - window) if window else True)
        some = seen.any(axis=1)
        for j in range(kv):
            kj, vj = k[ids, j, at % page], v[ids, j, at % page]
            for i in range(j * g, (j + 1) * g):
                with np.errstate(invalid="ignore", over="ignore"):
                    s = (q[r0:r1, i].astype(np.float64) @ kj.T) * scale
                    s[~seen] = -np.inf
                    e = np.exp(s - s.max(axis=1, keepdims=True))
                    e[~seen] = 0.0
                    fine = np.isfinite(vj).all()
                    o = e @ vj if fine else np.stack([(w[m, None] * vj[m]).sum(axis=0) for w, m in zip(e, seen)])
                    o = o / e.sum(axis=1, keepdims=True)
                out[r0:r1, i] = np.where(some[:, None], o, 0.0)
    return out


def make(rng, new, held, h, kv, d, page, kind, blocks=None, sharp=1.5, pad=(0, 0)):
    """Inputs of sequences that hold ``held`` keys and add ``new``: (q, k, v, tables, lengths, starts), and k, v in 64 bits."""
    new, held = np.asarray(new), np.asarray(held)
    total = new + held
    used = -(-total // page)
    blocks = max(1, int(used.max())) + 2 if blocks is None else blocks
    pages = int(used.sum()) + 3
    order, tables, at = rng.permutation(pages).astype(I32), np.full((len(new), blocks), -1, I32), 0
    for i, u in enumerate(used):
        tables[i, :u] = order[at:at + u]
        at += u
    starts = (pad[0] + np.concatenate([[0], np.cumsum(new)])).astype(I32)
    q = (sharp * rng.normal(size=(int(starts[-1]) + pad[1], h, d))).astype(np.float32)
    ks, k64 = stored(rng.normal(size=(pages, kv, page, d)), kind)
    vs, v64 = stored(rng.normal(size=(pages, kv, page, d)), kind)
    return (q, ks, vs, tables, total.astype(I32), starts), (k64, v64)


def check(paged, new, held, h, kv, d, page, kind, window=None, scale=None, sharp=1.5, blocks=None, pad=(0, 0), seed=0):
    rng = np.random.default_rng([len(new), h, d, page, seed])
    (q, ks, vs, tables, lengths, starts), (k64, v64) = make(rng, new, held, h, kv, d, page, kind, blocks, sharp, pad)
    before = rng.normal(size=q.shape).astype(np.float32)
    out = dev(before)
    got = paged.extend(dev(q), dev(ks), dev(vs), tables, lengths, starts, window=window, scale=scale, out=out).numpy()
    factor = 1 / np.sqrt(d) if scale is None else scale
    want = extend_ref(q, k64, v64, tables, lengths, starts, window, factor, before)
    assert np.isfinite(got).all()
    rows = slice(int(starts[0]), int(starts[-1]))
    assert np.array_equal(got[:rows.start], before[:rows.start]) and np.array_equal(got[rows.stop:], before[rows.stop:])
    if rows.stop == rows.start:
        return
    blind = ~want[rows].any(axis=(1, 2))
    assert not got[rows][blind].any()
    tol = TOL
    if sharp > 2:
        a = np.abs(q).sum(-1).max() * np.abs(k64).max() * abs(factor)
        tol += 2 * (d + 4) * 2.0 ** -23 * a * np.abs(v64).max() / np.abs(want[rows]).max()
    assert rel_err(got[rows], want[rows]) <= tol


HEADS = [(14, 2, 64), (16, 16, 64), (32, 8, 128), (20, 4, 80), (8, 1, 96), (1, 1, 8), (17, 1, 32), (40, 2, 128),
         (6, 3, 160), (4, 1, 192), (2, 2, 256), (33, 1, 256), (5, 5, 200), (200, 1, 24), (3, 1, 104)]
NEW = [1, 0, 5, 40, 17, 64, 3, 0, 130]
HELD = [0, 9, 63, 64, 100, 1, 700, 0, 0]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("h,kv,d", HEADS)
def test_extend_ragged(paged, h, kv, d, kind):
    check(paged, NEW, HELD, h, kv, d, 16, kind, pad=(3, 2))
    check(paged, NEW, HELD, h, kv, d, 16, kind, window=50, pad=(0, 7))


@pytest.mark.parametrize("page", [1, 3, 8, 24, 64, 100, 128, 1000])
@pytest.mark.parametrize("h,kv,d", [(14, 2, 64), (4, 4, 128)])
def test_extend_pages(paged, h, kv, d, page):
    for kind in TYPES:
        check(paged, [70, 1, 33], [40, 200, 0], h, kv, d, page, kind, seed=page)


LENGTHS = [([1], [0]), ([1], [500]), ([2], [0]), ([4], [500]), ([64], [0]), ([65], [64]), ([129], [0]), ([900], [0]),
           ([3], [30011]), ([100], [20000]), ([1] * 40, [700] * 40), ([0, 0, 0], [5, 0, 64]), ([1300, 2], [0, 3000])]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("new,held", LENGTHS, ids=lambda x: str(x)[:12])
def test_extend_lengths(paged, new, held, kind):
    check(paged, new, held, 14, 2, 64, 16, kind)


@pytest.mark.parametrize("window", [1, 2, 15, 64, 65, 300, 5000])
@pytest.mark.parametrize("kind", TYPES)
def test_extend_windows(paged, window, kind):
    check(paged, [200, 1, 40, 3], [0, 300, 1000, 9], 14, 2, 64, 16, kind, window=window)
    check(paged, [70, 30], [2000, 0], 4, 2, 128, 24, kind, window=window)


@pytest.mark.parametrize("batch", [63, 64, 65, 257, 1000, 3000])
def test_extend_large_batches(paged, batch):
    rng = np.random.default_rng(batch)
    check(paged, rng.integers(0, 5, batch), rng.integers(0, 60, batch), 4, 2, 32, 16, "bfloat16")


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("h,kv,d", [(64, 32, 8), (48, 16, 64), (32, 8, 128), (40, 10, 160)])
def test_extend_many_tiles_of_short_tables(paged, h, kv, d, kind):
    """More tiles of rows than run at once, taken by their last keys: sequences of any order and size, some of nothing,
    one with more tokens than keys, windows; and as many sequences as are ordered, and one more."""
    check(paged, [30, 0, 290, 1, 200, 290, 0, 77, 128, 3], [0, 9, 64, 400, 0, 64, 0, 20, -60, 300], h, kv, d, 16, kind, pad=(4, 5))
    check(paged, [30, 290, 200, 77, 128], [350, 64, 0, 20, 500], h, kv, d, 24, kind, window=100)
    rng = np.random.default_rng(d)
    for batch in (64, 65):
        check(paged, rng.integers(0, 30, batch), rng.integers(0, 100, batch), h, kv, d, 16, kind, seed=batch)


@pytest.mark.parametrize("kind", TYPES)
def test_extend_of_planned_sequences_in_their_order(paged, kind):
    """More items than run at once, over tables past those that go without a plan: uncut, the largest first; with one
    sequence so long that it is cut; and with windows, which leave nearly equal items."""
    new, held = [300, 0, 7, 260, 300, 130, 1, 300, 40], [4200, 5, 0, 1000, 0, 2500, 300, 3000, 64]
    check(paged, new, held, 48, 16, 64, 32, kind, pad=(2, 3))
    check(paged, [200] * 6 + [60], [0] * 6 + [20000], 64, 16, 64, 64, kind)
    check(paged, new, held, 48, 16, 64, 32, kind, window=200)
    check(paged, [250, 100, 250, 30], [2100, 0, 1500, 60], 32, 16, 64, 32, kind)            # fewer, uneven and uncut
    check(paged, [30] * 70, [50] * 69 + [4500], 32, 16, 64, 16, kind)          # more sequences than are ordered by lane


def test_extend_scales(paged):
    """Any scale: none, negative, large; scores of hundreds."""
    for kind in TYPES:
        for scale in (0.0, -0.125, 1.0, 1e-20):
            check(paged, [40, 3], [30, 200], 14, 2, 64, 16, kind, scale=scale, sharp=1.5 if abs(scale) < 1 else 2.5)
        check(paged, [40, 3], [30, 200], 14, 2, 64, 16, kind, sharp=40.0)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("h,kv,d", [(14, 2, 64), (4, 2, 128)])
def test_extend_unseen_rows_reach_nothing(paged, h, kv, d, kind):
    """NaN, infinities and the type's largest values behind the last key, on pages of no sequence, on the page that an
    absent id would clamp to, before a window; ids outside the cache are absent keys."""
    rng = np.random.default_rng(5)
    page, window = 16, 90
    new, held = [0, 5, 37, 100, 30, 12], [5, 0, 0, 500, 270, 52]
    (q, ks, vs, tables, lengths, starts), _ = make(rng, new, held, h, kv, d, page, kind)
    pages = ks.shape[0]
    free = sorted(set(range(pages)) - set(tables[tables >= 0].tolist()))
    tables[tables == 0] = free[0]                                   # page 0 is nobody's
    tables[3, 32], tables[3, 36], tables[4, 17] = -1, pages, 2**31 - 1
    tables[5, :4] = [-1, pages + 5, -2**31, -7]                     # nothing of this one is there
    for w in (None, window):
        seen = np.zeros((pages, page), bool)
        for b in range(len(new)):
            lo = 0 if w is None or new[b] == 0 else max(0, held[b] + 1 - w)
            for j in range(lo, lengths[b]):
                if 0 <= tables[b, j // page] < pages:
                    seen[tables[b, j // page], j % page] = True
        top = {"float32": 3e38, "float16": 65504.0, "bfloat16": 3e38}[kind]
        fill = rng.choice([np.nan, np.inf, -np.inf, top, -top], size=(2, pages, kv, page, d))
        kvs = np.where(seen[None, :, None, :, None], rng.normal(size=(2, pages, kv, page, d)), fill)
        (ks, k64), (vs, v64) = (stored(x, kind) for x in kvs)
        got = paged.extend(q, dev(ks), dev(vs), tables, lengths, starts, window=w)
        want = extend_ref(q, k64, v64, tables, lengths, starts, w, 1 / np.sqrt(d), np.zeros_like(q))
        assert np.isfinite(want).all() and rel_err(got, want) <= TOL
        assert not got[starts[5]:starts[6]].any()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, 6e4, 3e38, -1e30])
@pytest.mark.parametrize("where", ["k", "v"])
def test_extend_later_tokens_reach_no_earlier_query(paged, where, bad, kind):
    """What stands in a token's key or value is seen by that token's queries and later ones alone: the others keep their
    results, to the last bits that float32 gives them, also where it would spoil a tile's common scale."""
    if kind == "float16" and abs(bad) > 65504 and np.isfinite(bad):
        pytest.skip("no float16")
    rng = np.random.default_rng(6)
    h, kv, d, page, n, at = 14, 2, 64, 16, 150, 70
    (q, ks, vs, tables, lengths, starts), (k64, v64) = make(rng, [n, 20], [0, 40], h, kv, d, page, kind)
    spoilt = np.array(values(ks if where == "k" else vs, kind), np.float32)
    spoilt[tables[0, at // page], 1, at % page, 7] = bad
    new, new64 = stored(spoilt, kind)
    ks, vs, k64, v64 = (new, vs, new64, v64) if where == "k" else (ks, new, k64, new64)
    got = paged.extend(q, dev(ks), dev(vs), tables, lengths, starts)
    want = extend_ref(q, k64, v64, tables, lengths, starts, None, 0.125, np.zeros_like(q))
    reached = np.zeros(q.shape, bool)
    reached[at:n, h // 2:] = True
    assert np.isfinite(got[~reached]).all() and rel_err(got[~reached], want[~reached]) <= TOL
    with np.errstate(invalid="ignore"):
        if where == "v" and not np.isfinite(bad):       # its channel's, and no other
            channel = np.zeros(q.shape, bool)
            channel[at:n, h // 2:, 7] = True
            assert not np.isfinite(got[channel]).any() and np.isfinite(got[~channel]).all()
            assert rel_err(got[~channel], want[~channel]) <= TOL
        elif np.isnan(bad) or bad == np.inf:            # +inf times a query's sign: NaN, or a weight of 0
            assert np.array_equal(np.isnan(got), np.isnan(want))
        fine = np.isfinite(want)
        if where == "v":
            assert rel_err(got[fine], want[fine]) <= TOL


@pytest.mark.parametrize("kind,bits", [("float32", 0x7f800001), ("float32", 0xffbfffff), ("bfloat16", 0x7f81), ("bfloat16", 0xffbf),
                                       ("float16", 0x7c01)])
@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("new,held", [(40, 30), (4, 62)])
def test_extend_signalling_nan_of_later_tokens(paged, new, held, where, kind, bits):
    """Signalling NaNs in a later token's key or value, beside an earlier one far above the others: the largest number of a
    tile is still found, and queries before that token keep their results."""
    rng = np.random.default_rng(26)
    h, kv, d, page, at = 14, 2, 64, 16, 66
    for channel in (4, 5, 6, 7):
        (q, ks, vs, tables, lengths, starts), (k64, v64) = make(rng, [new], [held], h, kv, d, page, kind)
        x, x64 = (np.array(ks), k64) if where == "k" else (np.array(vs), v64)
        q[..., 4] *= 0.01                                           # a large channel of an ordinary score
        for key in (64, 65):
            big, big64 = stored(np.full(kv, 1000.0), kind)
            x[tables[0, key // page], :, key % page, 4] = big
            x64[tables[0, key // page], :, key % page, 4] = big64
        x.view({4: np.uint32, 2: np.uint16}[x.itemsize])[tables[0, at // page], :, at % page, channel] = bits
        got = paged.extend(q, dev(x if where == "k" else ks), dev(x if where == "v" else vs), tables, lengths, starts)
        n = at - held                                               # queries before that token
        x64[tables[0, at // page], :, at % page, channel] = 0.0
        want = extend_ref(q, k64, v64, tables, lengths, starts, None, 0.125, np.zeros_like(q))
        assert np.isfinite(got[:n]).all() and rel_err(got[:n], want[:n]) <= TOL
        assert np.isnan(got[n:]).any(axis=2).all()


@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
def test_extend_values_of_very_different_sizes(paged, kind):
    """A key that takes all the weight has values 2^40 times smaller than the others': the outputs are those values."""
    rng = np.random.default_rng(8)
    h, kv, d, page = 4, 2, 64, 16
    (q, ks, vs, tables, lengths, starts), (k64, v64) = make(rng, [50, 3], [100, 300], h, kv, d, page, kind)
    q[:] = 1.0
    k, v = (np.array(values(x, kind), np.float32) for x in (ks, vs))
    for b, at in ((0, 33), (1, 290)):
        k[tables[b, at // page], :, at % page] = 30.0
        v[tables[b, at // page], :, at % page] *= 2.0 ** -40
    (ks, k64), (vs, v64) = stored(k, kind), stored(v, kind)
    got = paged.extend(q, dev(ks), dev(vs), tables, lengths, starts)
    want = extend_ref(q, k64, v64, tables, lengths, starts, None, 0.125, np.zeros_like(q))
    assert np.abs(want).max() < 1e-10 and rel_err(got, want) <= 2e-5      # a score of 240: its float32 is off by 2^-17


@pytest.mark.parametrize("kind", TYPES)
def test_extend_sizes_of_queries_and_caches(paged, kind):
    """Queries, keys and values of any size, as long as their products have one."""
    rng = np.random.default_rng(9)
    for qs, ksz, vsz in ((1e-30, 1.0, 1.0), (1e-3, 1e2, 1e-4), (1e4, 1e-4, 6e3), (1e30, 1e-30 if kind != "float16" else 1e-5, 1.0),
                         (0.0, 1.0, 1.0), (1.0, 0.0, 1.0), (1.0, 1.0, 0.0)):
        if kind == "float16" and qs == 1e30:
            continue
        (q, ks, vs, tables, lengths, starts), _ = make(rng, [60, 4], [10, 200], 14, 2, 64, 16, kind)
        q = (q * np.float32(qs)).astype(np.float32)
        (ks, k64), (vs, v64) = (stored(values(x, kind) * s, kind) for x, s in ((ks, ksz), (vs, vsz)))
        got = paged.extend(q, dev(ks), dev(vs), tables, lengths, starts)
        want = extend_ref(q, k64, v64, tables, lengths, starts, None, 0.125, np.zeros_like(q))
        assert np.isfinite(got).all()
        assert np.abs(got - want).max() <= TOL * np.abs(want).max()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("h,kv,d", [(14, 2, 64), (4, 2, 128)])
def test_extend_of_scores_that_are_all_minus_infinity(paged, h, kv, d, kind):
    """Keys that are there and whose scores are -inf every one: 0 / 0, NaN, and not the zeros of a query with no key to
    see.  One score that is a number takes it all, wherever it lies."""
    rng = np.random.default_rng([d, 2])
    new, held = [30, 30, 10, 1, 40, 0, 20], [300, 300, 1200, 0, 2000, 7, 30]
    (q, ks, vs, tables, lengths, starts), _ = make(rng, new, held, h, kv, d, 16, kind)
    q[..., 0] = 1.0
    k = np.array(values(ks, kind), np.float32)

    def away(b, lo, hi, heads=slice(None)):
        for j in range(lo, hi):
            k[tables[b, j // 16], heads, j % 16, 0] = -np.inf

    away(0, 0, 330)                     # every key
    away(1, 0, 330, 1)                  # of one kv head
    away(2, 0, 1205)                    # all that the first five queries see
    away(3, 0, 1)                       # the only one
    away(4, 1, 2040)                    # all but the first
    away(6, 0, 50)
    tables[6, :4:2] = -1                # and pages that are not there
    (ks, k64), (vs, v64) = stored(k, kind), stored(values(vs, kind), kind)
    got = paged.extend(q, dev(ks), dev(vs), tables, lengths, starts)
    want = extend_ref(q, k64, v64, tables, lengths, starts, None, 1 / np.sqrt(d), np.zeros_like(q))
    assert np.isnan(want[:30]).all() and np.isnan(want[60:65]).all() and np.isfinite(want[65:70]).all()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = ~np.isnan(want)
    assert rel_err(got[fine], want[fine]) <= TOL


# (new, held) a sequence: a workgroup an item, few rows, items that a plan cuts
FORMS = {"whole": ([200, 30], [100, 0]), "few": ([5, 1, 3], [900, 20, 40]), "cut": ([130, 2, 40], [6000, 0, 1500])}


def spoil_last(rng, ins, kind, where, h=14):
    """The last token of every sequence spoilt in its key or value, which the others do not see: (k, v, k64, v64, rows that
    see none of it).  The others' tiles that hold it are formed again, their other parts are not."""
    q, ks, vs, tables, lengths, starts = ins
    page = ks.shape[2]
    k, v = (np.array(values(x, kind), np.float32) for x in (ks, vs))
    clear = np.ones(len(q), bool)
    for b in range(len(lengths)):
        at = lengths[b] - 1
        (k if where == "k" else v)[tables[b, at // page], :, at % page, 3] = np.inf if b % 2 else np.nan
        clear[starts[b + 1] - 1] = False
    (ks, k64), (vs, v64) = stored(k, kind), stored(v, kind)
    return ks, vs, k64, v64, clear


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
@pytest.mark.parametrize("spoilt", [None, "k", "v"])
def test_extend_values_near_the_largest(paged, spoilt, kind, form):
    """Means of values up to 3e38 have their size: no sum on the way there leaves float32's range, of parts that are joined
    and of rows that are formed again neither."""
    rng = np.random.default_rng(21)
    ins, _ = make(rng, *FORMS[form], 14, 2, 64, 16, kind)
    ins = list(ins)
    ins[0] *= np.float32(0.1)                               # many keys of like weight
    ins[2] = stored(3e38 * rng.uniform(0.5, 1.0, ins[2].shape), kind)[0]
    if spoilt:
        ks, vs, k64, v64, clear = spoil_last(rng, ins, kind, spoilt)
    else:
        ks, vs, clear = ins[1], ins[2], np.ones(len(ins[0]), bool)
        k64, v64 = (values(x, kind).astype(np.float64) for x in (ks, vs))
    got = paged.extend(ins[0], dev(ks), dev(vs), *ins[3:])
    want = extend_ref(ins[0], k64, v64, *ins[3:], None, 0.125, np.zeros_like(ins[0]))
    assert np.abs(want[clear]).min() > 1.4e38 and np.isfinite(got[clear]).all()
    assert rel_err(got[clear], want[clear]) <= TOL


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("h,kv,d", [(14, 2, 64), (4, 2, 128)])
@pytest.mark.parametrize("spoilt", ["k", "v"])
def test_extend_of_parts_formed_again_beside_others(paged, spoilt, h, kv, d, kind, form):
    """A row whose last keys lie in a spoilt tile, and the others in clean ones: what is formed again there and what comes
    from the matrix cores elsewhere weigh alike, since scores are small and every key counts."""
    rng = np.random.default_rng([22, d])
    ins, _ = make(rng, *FORMS[form], h, kv, d, 16, kind, sharp=0.3)
    ks, vs, k64, v64, clear = spoil_last(rng, ins, kind, spoilt)
    got = paged.extend(ins[0], dev(ks), dev(vs), *ins[3:])
    want = extend_ref(ins[0], k64, v64, *ins[3:], None, 1 / np.sqrt(d), np.zeros_like(ins[0]))
    assert np.isfinite(got[clear]).all() and rel_err(got[clear], want[clear]) <= TOL


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("lead", [0.0, 1e-5, 2.0 ** -13.9, 1.0])
def test_extend_small_weights_of_large_values(paged, lead, kind, form):
    """A key with small values that scores 24.5 above all others, whose weights are 2^-35 of its own and whose values are
    large: they count as float32 counts them, however many there are.

    A weight's exponent, 35.3 in powers of two, is rounded by 2^-19 at most and the weight by 0.7 of it, 1.4e-6."""
    rng = np.random.default_rng(23)
    for h, kv, d in ((14, 2, 64), (4, 2, 128)):
        ins, _ = make(rng, *FORMS[form], h, kv, d, 16, kind)
        q, ks, vs, tables, lengths, starts = ins
        q[:] = 0.0
        q[..., 0] = np.sqrt(d)
        k, v = np.zeros(ks.shape, np.float32), np.abs(100 + 10 * rng.normal(size=vs.shape)).astype(np.float32)
        for b in range(len(lengths)):
            k[tables[b, 0], :, 0, 0] = 24.5
            v[tables[b, 0], :, 0] *= lead
        (ks, k64), (vs, v64) = stored(k, kind), stored(v, kind)
        got = paged.extend(q, dev(ks), dev(vs), tables, lengths, starts)
        want = extend_ref(q, k64, v64, tables, lengths, starts, None, 1 / np.sqrt(d), np.zeros_like(q))
        for b in range(len(lengths)):            # a sequence's outputs have a size of their own
            r = slice(starts[b], starts[b + 1])
            assert rel_err(got[r] * 1e10, want[r] * 1e10) <= TOL, (b, d)


def apart(rng, ins, kind, big_q, big_k, low):
    """Inputs whose queries have one channel of size ``big_q``, their keys another of ``big_k``, and ``low`` where the other
    has it: their scores are as large as without."""
    q, ks, vs, tables, lengths, starts = ins
    k = np.array(values(ks, kind), np.float32)
    q[..., 9], q[..., 5] = big_q * q[..., 9], low * q[..., 5]
    k[..., 5], k[..., 9] = big_k * (1 + 0.1 * k[..., 5]), low * k[..., 9]
    ks, k64 = stored(k, kind)
    return (q, ks, vs, tables, lengths, starts), k64


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("h,kv,d", [(14, 2, 64), (4, 2, 128), (8, 1, 96)])
@pytest.mark.parametrize("big_q,big_k,low", [(70, 300, 0.01), (400, 2000, 1e-3), (1e5, 3e4, 1e-5), (1e7, 1.0, 1e-3), (1.0, 3e4, 1e-5)])
def test_extend_large_channels_that_do_not_meet(paged, big_q, big_k, low, h, kv, d, kind, form):
    """Single channels of queries and of keys far above the others, as biased projections have them, in different places:
    the scores are ordinary, and as exact as float32 makes them, whatever lies between the channels' sizes."""
    rng = np.random.default_rng([24, d])
    ins, (_, v64) = make(rng, *FORMS[form], h, kv, d, 16, kind)
    ins, k64 = apart(rng, ins, kind, big_q, big_k, low)
    got = paged.extend(ins[0], *(dev(x) for x in ins[1:3]), *ins[3:])
    want = extend_ref(ins[0], k64, v64, *ins[3:], None, 1 / np.sqrt(d), np.zeros_like(ins[0]))
    # the channel where both are large: a term that float32 rounds by 2^-24 of itself, in each of d sums
    a = max(np.abs(ins[0][..., c]).max() * np.abs(k64[..., c]).max() for c in (5, 9)) / np.sqrt(d)
    assert rel_err(got, want) <= TOL + 2 * (d + 4) * 2.0 ** -24 * a


@pytest.mark.parametrize("kind", TYPES)
def test_extend_large_channels_cost_no_more(gpu, paged, kind):
    """... and as fast: keys with a channel of 300 under queries with another of 100, five times the time of those without
    at the very most (82 times when their rows were formed again)."""
    from cv3amd import device
    rng = np.random.default_rng(25)
    times = []
    for big in (1, 0):
        ins, _ = make(rng, [300] * 6, [0] * 6, 14, 2, 64, 16, kind)
        if big:
            ins, _ = apart(rng, ins, kind, 70, 300, 0.01)
        ds, timer, out = [dev(x) for x in ins], device.Timer(), dev(np.zeros(ins[0].shape, np.float32))
        each = []
        for _ in range(5):
            timer.start()
            for _ in range(10):
                paged.extend(*ds, out=out)
            each.append(timer.stop())
        times.append(sorted(each)[2])
    assert times[0] <= 5 * times[1], times


@pytest.mark.parametrize("kind", TYPES)
def test_extend_large_values_cost_no_more(gpu, paged, kind):
    """One token's values are 2000 times the others', and rows give most of their weight to some other key: next to no weight
    counts for little there, and is not looked for by forming the rows again."""
    from cv3amd import device
    rng = np.random.default_rng(27)
    times = []
    for big in (1, 0):
        (q, ks, vs, tables, lengths, starts), (k64, v64) = make(rng, [900, 900], [0, 0], 14, 2, 64, 16, kind, sharp=6.0)
        q[..., 0], k = 40.0, np.array(values(ks, kind), np.float32)
        k[..., 0] = 0.0
        for b in range(2):
            k[tables[b, 0], :, 0, 0] = -8.0                         # 40 x 8 / 8 below the others
        v = np.array(values(vs, kind), np.float32)
        if big:
            v[tables[:, 0], :, 0] *= 2000.0
        (ks, k64), (vs, v64) = stored(k, kind), stored(v, kind)
        ds, timer, out = [dev(x) for x in (q, ks, vs, tables, lengths, starts)], device.Timer(), dev(np.zeros(q.shape, np.float32))
        each = []
        for _ in range(5):
            timer.start()
            for _ in range(10):
                paged.extend(*ds, out=out)
            each.append(timer.stop())
        times.append(sorted(each)[2])
        got, want = out.numpy(), extend_ref(q, k64, v64, tables, lengths, starts, None, 0.125, np.zeros_like(q))
        rows = np.r_[1:900, 901:1800]                               # the first tokens see that value alone
        # scores of up to 6 x 4 x 4 x 8 / 8: the sums' roundings as in ``check``
        a = np.abs(q).sum(-1).max() * np.abs(k64).max() * 0.125
        assert rel_err(got[rows], want[rows]) <= TOL + 2 * 68 * 2.0 ** -23 * a
    assert times[0] <= 5 * times[1], times


def test_extend_lengths_past_the_table(paged):
    """A length past its table counts as the table's end; more new tokens than keys: those before position 0 see nothing."""
    rng = np.random.default_rng(11)
    h, kv, d, page, blocks = 14, 2, 64, 16, 5
    tables = rng.permutation(20).astype(I32)[:15].reshape(3, 5)
    lengths, starts = np.array([1000, 4, -3], I32), np.array([0, 20, 30, 34], I32)
    q = rng.normal(size=(34, h, d)).astype(np.float32)
    for kind in TYPES:
        (ks, k64), (vs, v64) = (stored(rng.normal(size=(20, kv, page, d)), kind) for _ in range(2))
        got = paged.extend(q, dev(ks), dev(vs), tables, lengths, starts)
        want = extend_ref(q, k64, v64, tables, lengths, starts, None, 0.125, np.zeros_like(q))
        assert not want[20:26].any() and want[26:30].any() and rel_err(got, want) <= TOL
        assert not got[20:26].any() and not got[30:].any()


def test_extend_starts_outside_the_list(paged):
    """Starts are cut at the list's ends: rows past it are not read or written."""
    rng = np.random.default_rng(12)
    (q, ks, vs, tables, lengths, _), (k64, v64) = make(rng, [10, 10], [60, 0], 14, 2, 64, 16, "float32")
    lengths[:] = [70, 50]
    padded = dev(np.full((40, 14, 64), 7.5, np.float32))
    padded.rows(10, 30).copy_from(q)
    starts = np.array([-5, 10, 60], I32)
    got = paged.extend(padded.rows(10, 30), dev(ks), dev(vs), tables, lengths, starts)
    want = extend_ref(q, k64, v64, tables, lengths, np.array([0, 10, 20]), None, 0.125, np.zeros_like(q))
    assert got.shape == (20, 14, 64) and rel_err(got.numpy(), want) <= TOL


def test_extend_in_place_strided_and_unaligned(paged):
    """Queries inside wider rows at any alignment, results in place of them."""
    from cv3amd import _lib
    rng = np.random.default_rng(13)
    for kind, code in (("float32", 0), ("float16", 1), ("bfloat16", 2)):
        for new, held in (([70, 3], [20, 400]), ([5], [3000])):
            h, kv, d, page = 14, 2, 64, 16
            (q, ks, vs, tables, lengths, starts), (k64, v64) = make(rng, new, held, h, kv, d, page, kind)
            n, ld = q.shape[0], h * d + 2 * kv * d + 3
            flat = np.full(1 + n * ld, 7.5, np.float32)
            flat[1:].reshape(n, ld)[:, :h * d] = q.reshape(n, -1)
            fd, kd, vd, td, nd, sd = (dev(x) for x in (flat, ks, vs, tables, lengths, starts))
            _lib.call("paged_extend", fd.ptr + 4, ld, n, h, kv, d, code, kd.ptr, vd.ptr, ks.shape[0], page, td.ptr,
                      tables.shape[1], nd.ptr, sd.ptr, len(new), 2**63 - 1, ctypes.c_float(0.125), fd.ptr + 4, ld, None)
            got = fd.numpy()
            assert got[0] == 7.5 and np.all(got[1:].reshape(n, ld)[:, h * d:] == 7.5)
            want = extend_ref(q, k64, v64, tables, lengths, starts, None, 0.125, np.zeros_like(q))
            assert rel_err(got[1:].reshape(n, ld)[:, :h * d].reshape(q.shape), want) <= TOL


def test_extend_shared_pages(paged):
    """Sequences that share pages, as forks do."""
    rng = np.random.default_rng(14)
    (q, ks, vs, tables, lengths, starts), (k64, v64) = make(rng, [20, 20, 7], [200, 200, 100], 14, 2, 64, 16, "bfloat16")
    tables[1, :12] = tables[0, :12]
    tables[2, :6] = tables[0, :6]
    got = paged.extend(q, dev(ks), dev(vs), tables, lengths, starts)
    want = extend_ref(q, k64, v64, tables, lengths, starts, None, 0.125, np.zeros_like(q))
    assert rel_err(got, want) <= TOL


def test_extend_offsets_past_32_bits(paged):
    """A cache of more than 2^31 elements, its last pages in use."""
    from cv3amd.device import DeviceArray
    rng = np.random.default_rng(15)
    kv, page, d = 2, 64, 128
    pages = (1 << 31) // (kv * page * d) + 40
    k, v = (DeviceArray((pages, kv, page, d), np.float16).zero_() for _ in range(2))
    ids = np.concatenate([rng.permutation(np.arange(pages - 30, pages))[:6], [0, 5]]).astype(I32)
    ks, vs = (rng.normal(size=(len(ids), kv, page, d)).astype(np.float16) for _ in range(2))
    for i, p in enumerate(ids):
        k.rows(int(p), int(p) + 1).copy_from(ks[i])
        v.rows(int(p), int(p) + 1).copy_from(vs[i])
    q = rng.normal(size=(40, 8, d)).astype(np.float32)
    n, starts = np.array([8 * 64 - 9], I32), np.array([0, 40], I32)
    want = extend_ref(q, ks.astype(np.float64), vs.astype(np.float64), np.arange(8, dtype=I32)[None], n, starts, None,
                      1 / np.sqrt(d), np.zeros_like(q))
    assert rel_err(paged.extend(q, k, v, ids[None], n, starts), want) <= TOL


def test_extend_of_one_token_is_attention(paged):
    rng = np.random.default_rng(16)
    for kind in TYPES:
        (q, ks, vs, tables, lengths, starts), _ = make(rng, [1] * 30, rng.integers(0, 600, 30), 14, 2, 64, 16, kind)
        kd, vd = dev(ks), dev(vs)
        assert rel_err(paged.extend(q, kd, vd, tables, lengths, starts), paged.attention(q, kd, vd, tables, lengths)) <= TOL


def test_extend_of_nothing(paged):
    k, v = dev(np.zeros((2, 2, 16, 64), np.float32)), dev(np.zeros((2, 2, 16, 64), np.float32))
    none = paged.extend(np.zeros((0, 14, 64), np.float32), k, v, np.zeros((1, 2), I32), [5], [0, 0])
    assert none.shape == (0, 14, 64)
    rows = paged.extend(np.ones((3, 14, 64), np.float32), k, v, np.zeros((0, 2), I32), np.zeros(0, I32), np.zeros(1, I32))
    assert not rows.any()


def inputs(seed, kind="bfloat16", new=(40, 3, 0, 90), held=(500, 2000, 5, 0), h=14, kv=2, d=64):
    rng = np.random.default_rng(seed)
    ins, (k64, v64) = make(rng, new, held, h, kv, d, 16, kind)
    want = extend_ref(ins[0], k64, v64, *ins[3:], None, 1 / np.sqrt(d), np.zeros_like(ins[0]))
    return [dev(x) for x in ins], want


def test_extend_on_an_explicit_stream(gpu, paged):
    from cv3amd import _lib, device
    (q, k, v, t, n, s), want = inputs(17)
    out, st = dev(np.zeros(q.shape, np.float32)), device.Stream()
    device.synchronize()
    for _ in range(3):
        _lib.call("paged_extend", q.ptr, 14 * 64, q.shape[0], 14, 2, 64, _lib.BF16, k.ptr, v.ptr, k.shape[0], 16, t.ptr,
                  t.shape[1], n.ptr, s.ptr, 4, 2**63 - 1, ctypes.c_float(0.125), out.ptr, 14 * 64, st.handle)
    _lib.call("stream_sync", st.handle)
    assert rel_err(out.numpy(), want) <= TOL


def test_extend_from_four_threads(gpu, paged):
    import threading
    from cv3amd import device
    wrong = []

    def work(i):
        try:
            ins, want = inputs([18, i], TYPES[i % 3], new=(40 + i, 3, 0, 90))
            outs = [paged.extend(*ins) for _ in range(20)]
            device.synchronize()
            wrong.extend(i for o in outs if rel_err(o.numpy(), want) > TOL)
        except Exception as e:      # noqa: BLE001
            wrong.append(repr(e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("kind", TYPES)
def test_extend_captured_and_replayed(gpu, paged, kind):
    """A graph serves every length: the lengths, starts and tables that the device holds when it is replayed.  Eager calls
    in between; a second graph of other arrays; without scratch in the allocator's cache."""
    from cv3amd import _lib, device
    rng = np.random.default_rng(19)
    states = []
    for j in range(2):
        ins, _ = make(rng, [30, 30, 60], [500, 100, 2000], 14, 2, 64, 16, kind)
        states.append((ins, [dev(x) for x in ins], dev(np.zeros(ins[0].shape, np.float32))))
    eager = paged.extend(*states[0][1])
    device.synchronize()
    graphs = []
    for j, (_, ds, out) in enumerate(states):
        if j:
            del eager
            _lib.call("empty_cache")            # this one finds no scratch
        g = device.Graph()
        with g:
            paged.extend(*ds, out=out)
        graphs.append(g)
        eager = paged.extend(*ds)
    for new in ([30, 30, 60], [1, 0, 5], [60, 60, 0], [0, 0, 0], [3, 100, 17]):
        for (ins, ds, out), g in zip(states, graphs):
            q, ks, vs, tables, _, _ = ins
            lengths = np.minimum(np.array(new) + [500, 100, 1900], tables.shape[1] * 16).astype(I32)
            starts = np.concatenate([[0], np.cumsum(new)]).astype(I32)
            ds[4].copy_from(lengths)
            ds[5].copy_from(starts)
            out.zero_()
            g.launch()
            want = extend_ref(q, values(ks, kind), values(vs, kind), tables, lengths, starts, None, 0.125, np.zeros_like(q))
            assert np.abs(out.numpy() - want).max() <= TOL * max(np.abs(want).max(), 1.0)
            eager = paged.extend(*ds)
            assert np.abs(eager.numpy() - want).max() <= TOL * max(np.abs(want).max(), 1.0)


def test_extend_is_the_same_every_time(paged):
    """The order of the workgroups changes nothing."""
    for kind in TYPES:
        ins, _ = inputs(20, kind)
        first = paged.extend(*ins).numpy()
        for _ in range(5):
            assert np.array_equal(paged.extend(*ins).numpy(), first)
