"""Forked sequences, free pages and caches that are compacted, on the GPU, against plain NumPy.  Everything is equal:
nothing is computed but whole numbers, and rows are copied as they are."""

import numpy as np
import pytest

from test_gpu_extend import extend_ref
from test_gpu_paged import TYPES, dev, rotary, stored, values

pytestmark = pytest.mark.gpu

I32, I64 = np.int32, np.int64
SHAPES = [(3, 16, 2, 64, "float32"), (1, 1, 1, 8, "float16"), (2, 5, 3, 40, "bfloat16"), (4, 64, 1, 128, "float16"),
          (2, 100, 2, 256, "float32"), (24, 24, 2, 80, "bfloat16")]       # layers, page, kv heads, dim, type


@pytest.fixture(scope="module")
def paged(gpu):
    from cv3amd import paged
    return paged


def caches(rng, layers, pages, kv, page, d, kind):
    return [stored(rng.normal(size=(layers, pages, kv, page, d)), kind)[0] for _ in range(2)]


def held(n, blocks, page):
    return min(max(int(n), 0), blocks * page)


# ------------------------------------------------------------------------------------------------
# fork
# ------------------------------------------------------------------------------------------------

def fork_ref(parents, children, tables, lengths, free, taken, ks):
    tables, lengths, ks = tables.copy(), lengths.copy(), [k.copy() for k in ks]
    old_t, old_n, old_k = tables.copy(), lengths.copy(), [k.copy() for k in ks]
    rows, blocks = tables.shape
    page, pages = ks[0].shape[3], ks[0].shape[1]
    for i, (p, c) in enumerate(zip(parents, children)):
        if not (0 <= p < rows and 0 <= c < rows) or c in parents or list(children).count(c) > 1:
            continue
        n = held(old_n[p], blocks, page)
        full, rest = divmod(n, page)
        row = np.full(blocks, -1)
        row[:full] = old_t[p, :full]
        if rest:
            row[full] = free[taken] if 0 <= taken < len(free) else -1
            taken += 1
            src, dst = old_t[p, full], row[full]
            if 0 <= src < pages and 0 <= dst < pages:
                for new, old in zip(ks, old_k):
                    new[:, dst, :, :rest] = old[:, src, :, :rest]
        tables[c], lengths[c] = row, n
    return tables, lengths, min(taken, 2**31 - 1), ks


def check_fork(paged, parents, children, tables, lengths, free, taken, ks):
    want = fork_ref(parents, children, tables, lengths, free, taken, ks)
    td, nd, kd = dev(tables), dev(lengths), [dev(k) for k in ks]
    got = paged.fork(np.asarray(parents, I32), np.asarray(children, I32), td, nd, np.asarray(free, I32),
                     np.array([taken], I32), *kd)
    assert np.array_equal(td.numpy(), want[0]) and np.array_equal(nd.numpy(), want[1]) and got[0] == want[2]
    for k, w in zip(kd, want[3]):
        assert np.array_equal(k.numpy().view(np.uint8), w.view(np.uint8))


def sequences(rng, rows, blocks, page, extra):
    """(tables, lengths, free ids, pages): distinct pages in any order, sequences of every length."""
    lengths = rng.integers(0, blocks * page + 1, rows).astype(I32)
    lengths[0], lengths[-1] = blocks * page, max(1, blocks * page // 2)
    used = -(-lengths // page)
    pages = int(used.sum()) + extra
    order, tables, at = rng.permutation(pages).astype(I32), rng.integers(-1, pages, (rows, blocks)).astype(I32), 0
    for i, u in enumerate(used):
        tables[i, :u] = order[at:at + u]
        at += u
    return tables, lengths, order[at:], pages


@pytest.mark.parametrize("layers,page,kv,d,kind", SHAPES)
@pytest.mark.parametrize("rows,forks", [(2, 1), (9, 6), (70, 50)])
def test_fork(paged, rows, forks, layers, page, kv, d, kind):
    rng = np.random.default_rng([rows, page, d])
    blocks = 3 if page * d > 4000 else 5
    tables, lengths, free, pages = sequences(rng, rows, blocks, page, forks + 4)
    ks = caches(rng, layers, pages, kv, page, d, kind)
    place = rng.permutation(rows)
    parents = place[rng.integers(0, rows - forks, forks)]
    check_fork(paged, parents, place[rows - forks:], tables, lengths, free, 1, ks)
    check_fork(paged, parents, place[rows - forks:], tables, lengths, free[:forks // 2], 0, ks)       # pages run out


def test_fork_without_layers(paged):
    rng = np.random.default_rng(1)
    tables, lengths, free, pages = sequences(rng, 6, 4, 16, 9)
    ks = caches(rng, 1, pages, 2, 16, 64, "float32")
    want = fork_ref([0, 5], [1, 2], tables, lengths, free, 0, ks)
    td, nd, kd = dev(tables), dev(lengths), [dev(k[0]) for k in ks]
    taken = paged.fork([0, 5], [1, 2], td, nd, dev(free), dev(np.zeros(1, I32)), *kd)
    assert np.array_equal(td.numpy(), want[0]) and np.array_equal(nd.numpy(), want[1]) and taken.numpy()[0] == want[2]
    assert all(np.array_equal(k.numpy(), w[0]) for k, w in zip(kd, want[3]))


def test_fork_of_rows_that_cannot_be(paged):
    """No fork into a parent of the call, twice into one child, from or into rows that are not there; such forks take
    no page.  Tables and lengths that say nonsense are cut or count as absent."""
    rng = np.random.default_rng(2)
    rows, blocks, page = 40, 4, 16
    tables, lengths, free, pages = sequences(rng, rows, blocks, page, 30)
    ks = caches(rng, 2, pages, 2, page, 64, "float16")
    lengths[:20] = rng.integers(1, 63, 20)
    check_fork(paged, [0, 1, 2, 3, 4], [30, 0, 31, 31, 32], tables, lengths, free, 0, ks)
    check_fork(paged, [0, -1, 2, 40, 4, 5], [30, 31, -7, 33, 40, 34], tables, lengths, free, 0, ks)
    check_fork(paged, [0, 0, 0], [0, 5, 5], tables, lengths, free, 0, ks)
    check_fork(paged, [7] * 6, [20, 21, 20, 22, 20, 23], tables, lengths, free, 3, ks)
    lengths[3], lengths[4], lengths[5] = -9, 2**31 - 1, 1000
    tables[6, :4], lengths[6] = [-1, pages, 2**31 - 1, -5], 37
    check_fork(paged, [3, 4, 5, 6], [30, 31, 32, 33], tables, lengths, free, 0, ks)
    check_fork(paged, [8, 9], [30, 31], tables, lengths, free, -1, ks)
    check_fork(paged, [8, 9], [30, 31], tables, lengths, free, 2**31 - 1, ks)
    check_fork(paged, [8, 9], [30, 31], tables, lengths, np.array([pages, -3]), 0, ks)      # pages outside the cache
    check_fork(paged, [8, 9], [30, 31], tables, lengths, np.zeros(0), 0, ks)
    check_fork(paged, [], [], tables, lengths, free, 5, ks)


def test_fork_many(paged):
    """As many forks as a call takes, in tables of as many rows."""
    rng = np.random.default_rng(3)
    rows, blocks, page = 65536, 2, 4
    lengths = rng.integers(1, 9, rows).astype(I32)
    tables, pages = rng.integers(0, 5000, (rows, blocks)).astype(I32), 9200
    ks = caches(rng, 1, pages, 1, page, 8, "float32")
    place, free = rng.permutation(rows), 5000 + rng.permutation(4200)
    parents = place[rng.integers(0, 60000, 4096)]
    # in NumPy at once: children are distinct and no parents, free pages apart from the tables'
    children = place[61440:]
    n = lengths[parents]
    need = n % page > 0
    fresh = np.where(need, free[np.cumsum(need) - need], -1)
    want_t, want_n, want_k = tables.copy(), lengths.copy(), [k.copy() for k in ks]
    for b in range(blocks):
        want_t[children, b] = np.where(b < n // page, tables[parents, b], np.where(b == n // page, fresh, -1))
    want_n[children] = n
    for k, w in zip(ks, want_k):
        for rest in range(1, page):
            at = np.flatnonzero(n % page == rest)
            w[0, fresh[at], :, :rest] = k[0, tables[parents[at], n[at] // page], :, :rest]
    td, nd, kd = dev(tables), dev(lengths), [dev(k) for k in ks]
    taken = paged.fork(parents.astype(I32), children.astype(I32), td, nd, free.astype(I32), np.zeros(1, I32), *kd)
    assert np.array_equal(td.numpy(), want_t) and np.array_equal(nd.numpy(), want_n) and taken[0] == need.sum()
    assert all(np.array_equal(k.numpy(), w) for k, w in zip(kd, want_k))


def absent_last(tables, lengths, page, pages):
    """Which sequences have a part-filled last page whose id lies outside the cache."""
    n = np.array([held(x, tables.shape[1], page) for x in lengths])
    last = tables[np.arange(len(n)), np.minimum(n // page, tables.shape[1] - 1)]
    return (n % page > 0) & ((last < 0) | (last >= pages))


def test_fork_of_a_part_filled_page_that_is_absent(paged):
    """A child sees what its parent sees: of a part-filled page that is not there, nothing, whatever an ended sequence
    left in the page that would be next; such a fork takes no page, and the others' pages follow each other."""
    rng = np.random.default_rng(13)
    rows, blocks, page, kv, d, h = 12, 4, 16, 2, 64, 4
    for kind in TYPES:
        tables, lengths, free, pages = sequences(rng, rows, blocks, page, 12)
        ks = caches(rng, 1, pages, kv, page, d, kind)
        lengths[:5] = [37, 40, 20, 9, 60]
        tables[:5] = rng.permutation(np.setdiff1d(np.arange(pages), free))[:20].reshape(5, blocks)
        tables[0, 2], tables[1, 2], tables[3, 0] = -1, pages, 2**31 - 1
        assert absent_last(tables, lengths, page, pages)[:5].tolist() == [True, True, False, True, False]
        for c in ks:                                            # what ended sequences left in the free pages: NaN
            c[:, free] = stored(np.full(c[:, free].shape, np.nan), kind)[0]
        parents, children = [0, 4, 1, 2, 3, 0, 4], [5, 6, 7, 8, 9, 10, 11]
        want_t, want_n, taken = tables.copy(), lengths.copy(), 1
        for p, c in zip(parents, children):
            full = lengths[p] // page
            want_t[c], want_n[c] = -1, lengths[p]
            want_t[c, :full] = tables[p, :full]
            if p in (2, 4):
                want_t[c, full] = free[taken]
                taken += 1
        td, nd, kd = dev(tables), dev(lengths), [dev(k) for k in ks]
        got = paged.fork(np.array(parents, I32), np.array(children, I32), td, nd, free, np.array([1], I32), *kd)
        assert got[0] == taken == 4 and np.array_equal(td.numpy(), want_t) and np.array_equal(nd.numpy(), want_n)
        q = rng.normal(size=(1, h, d)).astype(np.float32).repeat(rows, 0)
        out = paged.attention(q, *(k.reshape(k.shape[1:]) for k in kd), td, nd)
        assert np.isfinite(out[children]).all() and np.array_equal(out[children], out[parents])


def test_fork_of_rows_that_cannot_be_but_for_absent_pages(paged):
    """The calls of ``test_fork_of_rows_that_cannot_be`` with sequences whose part-filled page is there."""
    rng = np.random.default_rng(2)
    rows, blocks, page = 40, 4, 16
    tables, lengths, free, pages = sequences(rng, rows, blocks, page, 30)
    ks = caches(rng, 2, pages, 2, page, 64, "float16")
    lengths[:20] = rng.integers(1, 63, 20)
    tables[:20] = rng.choice(np.setdiff1d(np.arange(pages), free), (20, blocks))

    def calls():
        assert not absent_last(tables, lengths, page, pages)[:20].any()
        check_fork(paged, [0, 1, 2, 3, 4], [30, 0, 31, 31, 32], tables, lengths, free, 0, ks)
        check_fork(paged, [0, -1, 2, 40, 4, 5], [30, 31, -7, 33, 40, 34], tables, lengths, free, 0, ks)
        check_fork(paged, [0, 0, 0], [0, 5, 5], tables, lengths, free, 0, ks)
        check_fork(paged, [7] * 6, [20, 21, 20, 22, 20, 23], tables, lengths, free, 3, ks)
        check_fork(paged, [3, 4, 5, 6], [30, 31, 32, 33], tables, lengths, free, 0, ks)
        check_fork(paged, [8, 9], [30, 31], tables, lengths, free, -1, ks)
        check_fork(paged, [8, 9], [30, 31], tables, lengths, free, 2**31 - 1, ks)
        check_fork(paged, [8, 9], [30, 31], tables, lengths, np.array([pages, -3]), 0, ks)      # pages outside the cache
        check_fork(paged, [8, 9], [30, 31], tables, lengths, np.zeros(0), 0, ks)
        check_fork(paged, [], [], tables, lengths, free, 5, ks)

    calls()
    lengths[3], lengths[4], lengths[5] = -9, 2**31 - 1, 1000
    tables[6, :2], lengths[6] = [-1, 2**31 - 1], 37                 # whole pages that are absent are shared as they stand
    calls()


# ------------------------------------------------------------------------------------------------
# free pages
# ------------------------------------------------------------------------------------------------

def held_ref(tables, lengths, page, pages):
    blocks = tables.shape[1]
    names = [tables[b, :-(-held(n, blocks, page) // page)] for b, n in enumerate(lengths)]
    names = np.concatenate(names) if names else np.zeros(0, I32)
    used = np.zeros(pages, bool)
    used[names[(names >= 0) & (names < pages)]] = True
    return used


def check_free(paged, tables, lengths, page, pages):
    tables, lengths = np.asarray(tables, I32), np.asarray(lengths, I32)
    ids, count = paged.free_pages(tables, lengths, page, pages)
    want = np.flatnonzero(~held_ref(tables, lengths, page, pages))
    assert count[0] == len(want) and np.array_equal(ids[:len(want)], want) and np.all(ids[len(want):] == -1)


@pytest.mark.parametrize("rows,blocks,page,pages", [
    (1, 1, 16, 1), (1, 3, 16, 64), (8, 57, 16, 500), (384, 119, 16, 46000), (5, 1000, 1, 4999), (3000, 2, 64, 63), (16, 64, 7, 65),
    (64, 10, 16, 131072), (64, 10, 16, 131073), (1200, 300, 8, 100001), (20, 10, 16, 1 << 24), (3, 5, 65536, 8192),
    (9000, 3, 16, 300000), (700, 400, 16, 8191)])
def test_free_pages(paged, rows, blocks, page, pages):
    rng = np.random.default_rng([rows, pages])
    tables = rng.integers(-2, pages + 2, (rows, blocks))
    lengths = rng.integers(-3, blocks * page + 20, rows)
    lengths[rng.random(rows) < 0.4] = 0
    check_free(paged, tables, lengths, page, pages)


def test_free_pages_at_the_edges(paged):
    check_free(paged, np.zeros((0, 4)), np.zeros(0), 16, 100)                               # no sequence: all of them
    check_free(paged, np.zeros((0, 4)), np.zeros(0), 16, 200000)
    check_free(paged, np.arange(100)[None], [1600], 16, 100)                                # every page held
    check_free(paged, np.arange(200000)[None], [200000], 1, 200000)
    check_free(paged, [[5, 6, 7]] * 3, [16, 17, 33], 16, 10)                                # shared, and on a page's border
    check_free(paged, [[5, 6, 7]] * 3, [-1, 2**31 - 1, 0], 16, 10)
    check_free(paged, [[2**31 - 1, -2**31, 31]], [48], 16, 32)


# ------------------------------------------------------------------------------------------------
# compact
# ------------------------------------------------------------------------------------------------

def check_compact(paged, tables, lengths, ks, pages_new, layered=True):
    tables, lengths = np.asarray(tables, I32), np.asarray(lengths, I32)
    page, pages = ks[0].shape[3], ks[0].shape[1]
    used = held_ref(tables, lengths, page, pages)
    ids = np.flatnonzero(used)
    rank = np.where(used, np.cumsum(used) - 1, -1)
    want = np.full(tables.shape, -1)
    for b, n in enumerate(lengths):
        live = -(-held(n, tables.shape[1], page) // page)
        t = tables[b, :live]
        want[b, :live] = np.where((t >= 0) & (t < pages), rank[np.clip(t, 0, pages - 1)], -1)
    want[want >= pages_new] = -1
    shape = (ks[0].shape[0], pages_new) + ks[0].shape[2:]
    new = [np.full(shape, 7, ks[0].dtype) for _ in ks]
    cut = (lambda x: x) if layered else (lambda x: x[0])
    kd, nd = [dev(cut(k)) for k in ks], [dev(cut(x)) for x in new]
    got, count = paged.compact(tables, lengths, *kd, *nd)
    assert count[0] == len(ids) and np.array_equal(got, want)
    n = min(len(ids), pages_new)
    for k, x, y in zip(ks, new, nd):
        x[:, :n] = k[:, ids[:n]]
        assert np.array_equal(y.numpy().view(np.uint8), cut(x).view(np.uint8))


@pytest.mark.parametrize("layers,page,kv,d,kind", SHAPES)
@pytest.mark.parametrize("rows", [1, 7, 60])
def test_compact(paged, rows, layers, page, kv, d, kind):
    rng = np.random.default_rng([rows, page, d])
    blocks = 4
    tables, lengths, _, pages = sequences(rng, rows, blocks, page, 5)
    lengths[rng.random(rows) < 0.3] = 0
    if rows > 2:
        tables[1, :2] = tables[0, :2]                                   # shared pages stay shared
    ks = caches(rng, layers, pages, kv, page, d, kind)
    used = int(held_ref(tables, lengths, page, pages).sum())
    for pages_new in {max(1, used), pages + 3, max(1, used // 2)}:      # just enough, a larger cache, one too small
        check_compact(paged, tables, lengths, ks, pages_new)


def test_compact_at_the_edges(paged):
    rng = np.random.default_rng(5)
    ks = caches(rng, 2, 20, 2, 16, 64, "bfloat16")
    check_compact(paged, np.zeros((0, 3)), np.zeros(0), ks, 4)
    check_compact(paged, [[1, 2, 3]] * 2, [0, -5], ks, 4)
    check_compact(paged, [[19, 25, -1], [19, 0, 2**31 - 1]], [48, 2**31 - 1], ks, 4)
    check_compact(paged, [[19, 3, 4], [19, 3, 5]], [40, 48], ks, 4, layered=False)
    ks = caches(rng, 1, 140000, 1, 1, 8, "float16")                     # more pages than one workgroup's bits
    check_compact(paged, rng.integers(0, 140000, (50, 90)), rng.integers(0, 91, 50), ks, 5000)


def test_offsets_past_32_bits(paged):
    """Caches of more than 2^31 elements."""
    from cv3amd.device import DeviceArray
    rng = np.random.default_rng(6)
    layers, kv, page, d = 2, 2, 64, 128
    pages = (1 << 30) // (kv * page * d) + 40
    k, v = (DeviceArray((layers, pages, kv, page, d), np.float16).zero_() for _ in range(2))
    k1, v1 = (DeviceArray((layers, 4, kv, page, d), np.float16).zero_() for _ in range(2))
    one = (kv, page, d)
    rows = rng.normal(size=(2, 2) + one).astype(np.float16)
    for c, i in ((k, 0), (v, 1)):
        for l in range(layers):
            c.reshape((layers * pages,) + one).rows(l * pages + pages - 1, l * pages + pages).copy_from(rows[i, l])
    tables, lengths = dev(np.array([[pages - 1], [-1]], I32)), dev(np.array([40, 0], I32))
    paged.fork([0], [1], tables, lengths, np.array([pages - 3], I32), np.zeros(1, I32), k, v)
    assert tables.numpy()[1, 0] == pages - 3 and lengths.numpy()[1] == 40
    turned, used = paged.compact(tables, lengths, k, v, k1, v1)
    assert turned.numpy().tolist() == [[1], [0]] and used.numpy()[0] == 2
    for c, i in ((k1, 0), (v1, 1)):
        got = c.numpy()
        assert np.array_equal(got[:, 1], rows[i])
        assert np.array_equal(got[:, 0, :, :40], rows[i][:, :, :40]) and not got[:, 0, :, 40:].any()


# ------------------------------------------------------------------------------------------------
# together: a scheduler's life
# ------------------------------------------------------------------------------------------------

class Cache:
    """What a scheduler keeps, and the same as plain lists of keys and values a sequence."""

    def __init__(self, paged, kind, rows=7, blocks=6, pages=36, layers=2, h=4, kv=2, d=64, page=8):
        self.paged, self.kind, self.h, self.kv, self.d, self.page, self.pages, self.layers = paged, kind, h, kv, d, page, pages, layers
        names = {"float32": "float32", "float16": "float16", "bfloat16": "bfloat16"}
        self.k, self.v = paged.new_cache(pages, kv, page, d, names[kind], layers=layers)
        self.tables, self.lengths = dev(np.full((rows, blocks), -1, I32)), dev(np.zeros(rows, I32))
        self.free, self.taken = dev(np.arange(pages, dtype=I32)), dev(np.zeros(1, I32))
        self.cos, self.sin = (dev(x) for x in rotary(d, 64))
        self.keys = [[np.zeros((2, kv, 0, d)) for _ in range(layers)] for _ in range(rows)]

    def layer(self, c, l):
        return c.rows(l, l + 1).reshape(c.shape[1:])

    def add(self, rng, new):
        """New tokens of some sequences, through every layer."""
        n = int(np.sum(new))
        total, self.taken, starts, slots, pos = self.paged.block_tables(
            self.lengths, dev(np.asarray(new, I32)), self.page, self.free, self.taken, self.tables, tokens=n + 3)
        assert self.taken.numpy()[0] <= len(self.free.numpy())
        self.lengths, at = total, starts.numpy()
        worst = 0.0
        for l in range(self.layers):
            qkv = rng.normal(size=(n + 3, (self.h + 2 * self.kv) * self.d)).astype(np.float32)
            k, v = self.layer(self.k, l), self.layer(self.v, l)
            q = self.paged.append(dev(qkv), self.h, pos, slots, self.cos, self.sin, k, v)
            got = self.paged.extend(q, k, v, self.tables, self.lengths, starts).numpy()
            qs, p = q.numpy(), pos.numpy()
            x = qkv.reshape(n + 3, -1, self.d)
            for b in range(len(new)):
                for i in range(at[b], at[b + 1]):
                    kk = x[i, self.h:self.h + self.kv].astype(np.float64)
                    half = self.d // 2
                    kk = kk * self.cos.numpy()[p[i]] + np.concatenate([-kk[:, half:], kk[:, :half]], 1) * self.sin.numpy()[p[i]]
                    row = np.stack([kk, x[i, self.h + self.kv:]])[:, :, None]
                    row = values(stored(row.astype(np.float32), self.kind)[0], self.kind)
                    self.keys[b][l] = np.concatenate([self.keys[b][l], row], axis=2)
                if at[b + 1] > at[b]:
                    kb, vb = (self.keys[b][l][j][None] for j in range(2))
                    want = extend_ref(qs[at[b]:at[b + 1]], kb, vb, np.zeros((1, 1), I32), [kb.shape[2]], [0, new[b]], None,
                                      1 / np.sqrt(self.d), np.zeros((new[b], self.h, self.d)))
                    # a key is turned here in 64 bits and there in 32: its rounding may go the other way, by a whole step
                    worst = max(worst, np.abs(got[at[b]:at[b + 1]] - want).max() / np.abs(want).max())
        step = {"float32": 2.0 ** -23, "float16": 2.0 ** -10, "bfloat16": 2.0 ** -7}[self.kind]
        assert worst <= 1e-5 + 20 * step        # scores of a few units, off by a step of one key's channels

    def fork(self, parents, children):
        self.taken = self.paged.fork(dev(np.asarray(parents, I32)), dev(np.asarray(children, I32)), self.tables,
                                     self.lengths, self.free, self.taken, self.k, self.v)
        for p, c in zip(parents, children):
            self.keys[c] = [x.copy() for x in self.keys[p]]

    def end(self, rows):
        n = self.lengths.numpy()
        for b in rows:
            n[b] = 0
            self.keys[b] = [x[:, :, :0] for x in self.keys[b]]
        self.lengths.copy_from(n)
        ids, count = self.paged.free_pages(self.tables, self.lengths, self.page, self.k.shape[1])
        self.free, self.taken = dev(ids.numpy()[:count.numpy()[0]]), dev(np.zeros(1, I32))
        held_now = {int(p) for b, m in enumerate(n) for p in self.tables.numpy()[b, :-(-int(m) // self.page)]}
        assert held_now.isdisjoint(self.free.numpy().tolist()) and len(held_now) + self.free.size == self.k.shape[1]

    def move(self, pages):
        names = {"float32": "float32", "float16": "float16", "bfloat16": "bfloat16"}
        k, v = self.paged.new_cache(pages, self.kv, self.page, self.d, names[self.kind], layers=self.layers)
        self.tables, used = self.paged.compact(self.tables, self.lengths, self.k, self.v, k, v)
        self.k, self.v = k, v
        assert used.numpy()[0] <= pages
        self.free, self.taken = dev(np.arange(used.numpy()[0], pages, dtype=I32)), dev(np.zeros(1, I32))


@pytest.mark.parametrize("kind", TYPES)
def test_a_schedulers_life(paged, kind):
    """Prompts come in slices, go on as several, end, make room, move to a smaller and a larger cache: every query sees
    exactly its own sequence's keys, whatever pages they lie on."""
    rng = np.random.default_rng(7)
    c = Cache(paged, kind)
    c.add(rng, [11, 0, 16, 5, 0, 0, 0])
    c.add(rng, [6, 0, 1, 0, 9, 0, 0])
    c.fork([0, 2, 0], [1, 5, 6])
    c.add(rng, [1, 4, 3, 8, 1, 2, 7])
    c.end([2, 0])
    c.add(rng, [20, 3, 13, 1, 0, 1, 1])
    c.move(30)
    c.fork([6], [3])
    c.add(rng, [1, 1, 1, 1, 1, 1, 1])
    c.end([0, 4, 5])
    c.move(60)
    c.add(rng, [40, 2, 2, 2, 30, 7, 2])


def test_a_step_captured_and_replayed(gpu, paged):
    """Freeing, forking, adding and attending in one graph, replayed for other lengths, with eager work in between."""
    from cv3amd import device
    rng = np.random.default_rng(8)
    rows, blocks, page, h, kv, d, pages = 5, 6, 8, 4, 2, 64, 200
    base_t = rng.permutation(pages).astype(I32)[:30].reshape(rows, blocks)
    k0, v0 = (rng.normal(size=(1, pages, kv, page, d)).astype(np.float32) for _ in range(2))
    qkv, new = rng.normal(size=(12, (h + 2 * kv) * d)).astype(np.float32), dev(np.array([2, 3, 1, 4, 2], I32))
    par, chi = dev(np.array([0, 2], I32)), dev(np.array([3, 4], I32))

    def state():
        return dict(tables=dev(base_t), n=dev(np.zeros(rows, I32)), k=dev(k0), v=dev(v0), x=dev(qkv),
                    free=dev(np.zeros(pages, I32)), count=dev(np.zeros(1, I32)), zero=dev(np.zeros(1, I32)),
                    took=dev(np.zeros(1, I32)), took2=dev(np.zeros(1, I32)), total=dev(np.zeros(rows, I32)), starts=dev(np.zeros(rows + 1, I32)),
                    slots=dev(np.zeros(12, I64)), pos=dev(np.zeros(12, I32)), q=dev(np.zeros((12, h, d), np.float32)),
                    out=dev(np.zeros((12, h, d), np.float32)))

    def step(s):
        paged.free_pages(s["tables"], s["n"], page, pages, out=(s["free"], s["count"]))
        paged.fork(par, chi, s["tables"], s["n"], s["free"], s["zero"], s["k"], s["v"], out=s["took"])
        paged.block_tables(s["n"], new, page, s["free"], s["took"], s["tables"],
                           out=(s["total"], s["took2"], s["starts"], s["slots"], s["pos"]))
        k, v = (s[c].reshape(s[c].shape[1:]) for c in "kv")
        paged.append(s["x"], h, None, s["slots"], None, None, k, v, out=s["q"])
        paged.extend(s["q"], k, v, s["tables"], s["total"], s["starts"], out=s["out"])

    lengths = [[5, 9, 16, 0, 7], [40, 1, 3, 8, 8], [0, 0, 0, 30, 2], [17, 33, 25, 1, 1]]
    names = ("tables", "n", "k", "v", "free", "count", "took", "took2", "total", "starts", "slots", "pos", "out")

    def begin(s, n):
        for name, value in (("tables", base_t), ("k", k0), ("v", v0), ("n", np.array(n, I32))):
            s[name].copy_from(value)

    eager, held_state = state(), state()
    want = []
    for n in lengths:
        begin(eager, n)
        step(eager)
        want.append({x: eager[x].numpy() for x in names})
    step(held_state)
    g = device.Graph()
    with g:
        step(held_state)
    for _ in range(2):
        for i, n in enumerate(lengths):
            begin(held_state, n)
            g.launch()
            begin(eager, n)
            step(eager)
            for x in names:
                assert np.array_equal(held_state[x].numpy(), want[i][x]), (i, x)


def test_calls_on_an_explicit_stream(gpu, paged):
    from cv3amd import _lib, device
    rng = np.random.default_rng(9)
    tables, lengths, free, pages = sequences(rng, 9, 4, 16, 12)
    ks = caches(rng, 2, pages, 2, 16, 64, "float32")
    want = fork_ref([0, 8], [1, 2], tables, lengths, free, 0, ks)
    td, nd, kd, fd = dev(tables), dev(lengths), [dev(k) for k in ks], dev(free)
    pd, cd, t0, t1 = (dev(np.array(x, I32)) for x in ([0, 8], [1, 2], [0], [9]))
    ids, count, used, turned = dev(np.zeros(pages, I32)), dev(np.zeros(1, I32)), dev(np.zeros(1, I32)), dev(np.zeros((9, 4), I32))
    new, st = [dev(np.zeros_like(k)) for k in ks], device.Stream()
    device.synchronize()
    _lib.call("paged_fork", pd.ptr, cd.ptr, 2, td.ptr, 9, 4, nd.ptr, fd.ptr, len(free), t0.ptr, t1.ptr, _lib.F32, kd[0].ptr,
              kd[1].ptr, 2, pages, 2, 16, 64, st.handle)
    _lib.call("paged_free", td.ptr, 9, 4, nd.ptr, 16, pages, ids.ptr, count.ptr, st.handle)
    _lib.call("paged_compact", td.ptr, 9, 4, nd.ptr, _lib.F32, kd[0].ptr, kd[1].ptr, 2, pages, 2, 16, 64, new[0].ptr,
              new[1].ptr, pages, turned.ptr, used.ptr, st.handle)
    _lib.call("stream_sync", st.handle)
    assert np.array_equal(td.numpy(), want[0]) and t1.numpy()[0] == want[2]
    used_ref = held_ref(want[0], want[1], 16, pages)
    assert count.numpy()[0] == (~used_ref).sum() and used.numpy()[0] == used_ref.sum()
    for k, x in zip(want[3], new):
        assert np.array_equal(x.numpy()[:, :used_ref.sum()], k[:, used_ref])


def test_two_graphs_with_scratch_of_their_own(gpu, paged):
    """A compaction and an extension that splits its keys, each captured twice, replayed in turn over other contents with
    eager calls between: no graph finds another's lists or parts."""
    from cv3amd import device
    rng = np.random.default_rng(12)
    rows, blocks, page, kv, d, pages, h, n = 3, 300, 8, 2, 64, 1000, 4, 40
    k, v = (dev(rng.normal(size=(pages, kv, page, d)).astype(np.float32)) for _ in range(2))
    tables = [dev(rng.permutation(pages).astype(I32)[:rows * blocks].reshape(rows, blocks)) for _ in range(2)]
    lengths = [dev(np.array(x, I32)) for x in ([2400, 100, 1999], [7, 2000, 0])]
    starts, q = dev(np.array([0, 20, 40, 40], I32)), [dev(rng.normal(size=(n, h, d)).astype(np.float32)) for _ in range(2)]

    def outs():
        return dict(out=dev(np.zeros((n, h, d), np.float32)), k=dev(np.zeros((400, kv, page, d), np.float32)),
                    v=dev(np.zeros((400, kv, page, d), np.float32)), t=dev(np.zeros((rows, blocks), I32)), used=dev(np.zeros(1, I32)))

    def step(i, o):
        paged.extend(q[i], k, v, tables[i], lengths[i], starts, out=o["out"])
        paged.compact(tables[i], lengths[i], k, v, o["k"], o["v"], out=(o["t"], o["used"]))

    def numbers(o):
        return {name: x.numpy() for name, x in o.items()}

    want, held, graphs = [], [outs(), outs()], []
    for i in range(2):
        o = outs()
        step(i, o)
        want.append(numbers(o))
        assert 0 < int(want[i]["used"][0]) and not np.array_equal(want[0]["t"], np.zeros((rows, blocks)))
    for i in range(2):
        step(i, held[i])                         # so that the allocator has the scratch that the capture takes
        graphs.append(device.Graph())
        with graphs[i]:
            step(i, held[i])
    for i in (0, 1, 1, 0, 0, 1):
        for name in ("out", "t", "used"):
            held[i][name].copy_from(np.zeros_like(want[i][name]))
        graphs[i].launch()
        step(1 - i, outs())
        got = numbers(held[i])
        for name, x in want[i].items():
            assert np.array_equal(got[name], x), (i, name)


def test_two_graphs_whose_contents_change(gpu, paged):
    """The same, with what the graphs read rewritten between their launches and every result cleared before: a launch
    answers for what is there, and writes all of it."""
    from cv3amd import device
    rng = np.random.default_rng(14)
    rows, blocks, page, kv, d, pages, h, n = 3, 300, 8, 2, 64, 1000, 4, 40
    k, v = (dev(rng.normal(size=(pages, kv, page, d)).astype(np.float32)) for _ in range(2))
    starts = dev(np.array([0, 20, 40, 40], I32))

    def contents():
        return dict(tables=rng.permutation(pages).astype(I32)[:rows * blocks].reshape(rows, blocks),
                    lengths=rng.integers(0, 1000, rows).astype(I32) + np.array([1400, 20, 0], I32),
                    q=rng.normal(size=(n, h, d)).astype(np.float32))

    def arrays():
        return dict(tables=dev(np.zeros((rows, blocks), I32)), lengths=dev(np.zeros(rows, I32)), q=dev(np.zeros((n, h, d), np.float32)),
                    out=dev(np.zeros((n, h, d), np.float32)), k=dev(np.zeros((500, kv, page, d), np.float32)),
                    v=dev(np.zeros((500, kv, page, d), np.float32)), t=dev(np.zeros((rows, blocks), I32)), used=dev(np.zeros(1, I32)))

    results = ("out", "k", "v", "t", "used")

    def begin(s, c):
        for name, x in c.items():
            s[name].copy_from(x)
        for name in results:
            s[name].zero_()

    def step(s):
        paged.extend(s["q"], k, v, s["tables"], s["lengths"], starts, out=s["out"])
        paged.compact(s["tables"], s["lengths"], k, v, s["k"], s["v"], out=(s["t"], s["used"]))

    eager, held, graphs = arrays(), [arrays(), arrays()], []
    for s in held:
        begin(s, contents())
        step(s)                                  # so that the allocator has the scratch that the capture takes
        graphs.append(device.Graph())
        with graphs[-1]:
            step(s)
    for i in (0, 1, 1, 0, 0, 1, 0):
        c = contents()
        begin(held[i], c)
        graphs[i].launch()
        begin(eager, c)
        step(eager)
        assert 0 < eager["used"].numpy()[0] <= 500
        for name in results:
            got = held[i][name].numpy()
            assert np.array_equal(got, eager[name].numpy()), (i, name)
        ids = np.flatnonzero(held_ref(c["tables"], c["lengths"], page, pages))
        assert np.array_equal(held[i]["k"].numpy()[:len(ids)], k.numpy()[ids]) and not held[i]["k"].numpy()[len(ids):].any()
        want = extend_ref(c["q"], k.numpy().astype(np.float64), v.numpy().astype(np.float64), c["tables"], c["lengths"],
                          starts.numpy(), None, 0.125, np.zeros_like(c["q"]))
        assert np.abs(held[i]["out"].numpy() - want).max() <= 1e-5 * np.abs(want).max()
