"""Refusals of the paged-cache and beam-search entry points: argument checks run on the host before anything is
enqueued, so they need no GPU."""

import pytest

P = 4096    # stands for a device address: never read, every call here is refused or has nothing to do


def tables(**k):
    a = dict(lengths=P, new=P, requests=3, page=16, free=P, free_count=8, taken=P, tables=P, blocks=4, tokens=5,
             total=2 * P, taken_out=2 * P, starts=P, slots=P, positions=P)
    a.update(k)
    return ("paged_tables", *a.values(), None)


def append(**k):
    a = dict(rows=P, n=3, ld=18 * 64, heads=14, kv_heads=2, d=64, positions=P, slots=P, cos=P, sin=P, rope_rows=100,
             type=0, k=P, v=P, pages=9, page=16, q=P, ldq=14 * 64)
    a.update(k)
    return ("paged_append", *a.values(), None)


def attention(**k):
    a = dict(q=P, ldq=14 * 64, batch=2, heads=14, kv_heads=2, d=64, type=0, k=P, v=P, pages=9, page=16, tables=P,
             blocks=4, lengths=P, starts=None, scale=0.125, out=P, ldo=14 * 64)
    a.update(k)
    return ("paged_attention", *a.values(), None)


def select(**k):
    a = dict(logits=P, requests=2, beams=4, vocab=100, scores=P, done=P, stop_lo=90, stop_hi=100, ban_lo=0, ban_hi=0,
             pad=90, tokens=P, parents=P, scores_out=P, done_out=P)
    a.update(k)
    return ("beam_select", *a.values(), None)


def reorder(**k):
    a = dict(parents=P, requests=2, beams=4, tables=P, own=2 * P, blocks=4, lengths=P, type=0, k=P, v=P, layers=2,
             pages=9, kv_heads=2, page=16, d=64)
    a.update(k)
    return ("beam_reorder", *a.values(), None)


REFUSED = [
    tables(requests=-1), tables(requests=4097), tables(page=0), tables(page=70000), tables(blocks=0),
    tables(blocks=1 << 40), tables(tokens=-1), tables(tokens=1 << 31), tables(free_count=-1), tables(free=None), tables(taken=None, taken_out=None),
    tables(lengths=None), tables(new=None), tables(taken=None), tables(tables=None), tables(total=None),
    tables(taken_out=None), tables(starts=None), tables(slots=None), tables(positions=None), tables(total=P),
    tables(taken_out=P),
    append(n=-1), append(d=60), append(d=0), append(d=264, ld=1 << 20, ldq=1 << 20), append(kv_heads=0),
    append(heads=-1), append(ld=18 * 64 - 1), append(ldq=14 * 64 - 1), append(cos=None), append(sin=None),
    append(positions=None), append(rope_rows=0), append(rows=None), append(slots=None), append(type=3),
    append(k=None), append(v=None), append(k=P + 8), append(pages=0), append(pages=1 << 31), append(page=0),
    append(n=1 << 40), append(n=1 << 23 | 1),
    attention(heads=15), attention(heads=0), attention(kv_heads=0), attention(d=12), attention(type=-1),
    attention(k=None), attention(v=P + 4), attention(pages=0), attention(page=0), attention(blocks=0),
    attention(blocks=1 << 30), attention(batch=-1), attention(batch=1 << 31), attention(batch=600000), attention(ldq=14 * 64 - 1),
    attention(ldo=0), attention(q=None), attention(tables=None), attention(lengths=None), attention(out=None),
    select(beams=0), select(beams=17), select(vocab=0), select(vocab=(1 << 19) + 1), select(requests=-1), select(requests=1 << 40), select(requests=1 << 22),
    select(ban_lo=2, ban_hi=99), select(vocab=3), select(logits=None), select(scores=None), select(done=None),
    select(tokens=None), select(parents=None), select(scores_out=None), select(done_out=None),
    reorder(beams=0), reorder(beams=17), reorder(type=7), reorder(page=0), reorder(pages=0), reorder(layers=0),
    reorder(kv_heads=0), reorder(d=20), reorder(blocks=0), reorder(requests=-1), reorder(parents=None),
    reorder(tables=None), reorder(own=None), reorder(own=P), reorder(lengths=None), reorder(k=None),
    reorder(v=P + 8), reorder(requests=1 << 31), reorder(requests=65536), reorder(layers=65536, kv_heads=1024),
]


@pytest.mark.parametrize("args", REFUSED, ids=lambda a: a[0])
def test_refused_before_anything_is_enqueued(args):
    from cv3amd import _lib
    with pytest.raises(ValueError):
        _lib.call(*args)
    assert _lib.lib().cv3_last_error()


def test_nothing_to_do_is_not_an_error():
    from cv3amd import _lib
    _lib.call(*append(n=0, rows=None, slots=None))
    _lib.call(*attention(batch=0, q=None, tables=None, lengths=None, out=None))
    _lib.call(*select(requests=0, logits=None))
    _lib.call(*reorder(requests=0, parents=None))


def test_python_checks_types_and_shapes():
    """The binding's own checks come before any device memory is touched."""
    import numpy as np
    from cv3amd import paged
    from cv3amd.device import DeviceArray

    class Memory:
        ptr, nbytes = P, 1 << 30

    def dev(shape, dtype=np.float32):
        return DeviceArray(shape, dtype, block=Memory())

    k, v = dev((9, 2, 16, 64)), dev((9, 2, 16, 64))
    i32, i64 = np.int32, np.int64
    with pytest.raises(TypeError):      # host caches
        paged.attention(dev((2, 14, 64)), np.zeros((9, 2, 16, 64), np.float32), v, dev((2, 4), i32), dev((2,), i32))
    with pytest.raises(TypeError):      # caches of two types
        paged.attention(dev((2, 14, 64)), k, dev((9, 2, 16, 64), np.float16), dev((2, 4), i32), dev((2,), i32))
    with pytest.raises(ValueError):     # of two shapes
        paged.attention(dev((2, 14, 64)), k, dev((8, 2, 16, 64)), dev((2, 4), i32), dev((2,), i32))
    with pytest.raises(ValueError):     # another head dim
        paged.attention(dev((2, 14, 32)), k, v, dev((2, 4), i32), dev((2,), i32))
    with pytest.raises(ValueError):     # tables of another batch
        paged.attention(dev((2, 14, 64)), k, v, dev((3, 4), i32), dev((2,), i32))
    with pytest.raises(TypeError):      # 64-bit lengths
        paged.attention(dev((2, 14, 64)), k, v, dev((2, 4), i32), dev((2,), i64))
    with pytest.raises(ValueError):     # heads that do not share evenly
        paged.attention(dev((2, 15, 64)), k, v, dev((2, 4), i32), dev((2,), i32), out=dev((2, 15, 64)))
    with pytest.raises(ValueError):     # an out of another shape
        paged.attention(dev((2, 14, 64)), k, v, dev((2, 4), i32), dev((2,), i32), out=dev((2, 64)))
    rows, at, slots, tab = dev((3, 18 * 64)), dev((3,), i32), dev((3,), i64), dev((50, 64))
    with pytest.raises(ValueError):
        paged.append(rows, 13, at, slots, tab, tab, k, v)
    with pytest.raises(ValueError):
        paged.append(rows, 14, at, slots, tab, None, k, v)
    with pytest.raises(TypeError):
        paged.append(rows, 14, at, dev((3,), i32), tab, tab, k, v)
    with pytest.raises(ValueError):
        paged.append(rows, 14, at, slots, dev((50, 32)), dev((50, 32)), k, v)
    n, t = dev((3,), i32), dev((3, 4), i32)
    with pytest.raises(TypeError):      # tables are updated in place
        paged.block_tables(n, n, 16, n, dev((1,), i32), np.zeros((3, 4), i32), tokens=5)
    with pytest.raises(ValueError):     # counts on the device: how long is the list?
        paged.block_tables(n, n, 16, n, dev((1,), i32), t)
    with pytest.raises(ValueError):
        paged.block_tables(n, dev((4,), i32), 16, n, dev((1,), i32), t, tokens=5)
    with pytest.raises(ValueError):     # total is an array of its own
        paged.block_tables(n, n, 16, n, dev((1,), i32), t, out=(n, dev((1,), i32), dev((4,), i32), dev((5,), i64),
                                                                 dev((5,), i32)))
    lg, sc, dn = dev((2, 4, 100)), dev((2, 4)), dev((2, 4), np.uint8)
    with pytest.raises(ValueError):
        paged.beam_select(lg, dev((2, 3)), dn, stop=(90, 100))
    with pytest.raises(TypeError):
        paged.beam_select(lg, sc, dev((2, 4), i32), stop=(90, 100))
    with pytest.raises(ValueError):
        paged.beam_select(lg, sc, dn, stop=(90, 100), ban=(0, 98), out=(dev((2, 4), i64), dev((2, 4), i32), sc, dn))
    with pytest.raises(ValueError):
        paged.beam_select(lg, sc, dn, stop=(90, 100), out=(dev((2, 4), i64),))
    par, bt = dev((2, 4), i32), dev((2, 4, 4), i32)
    with pytest.raises(ValueError):     # the own pages are a table of their own
        paged.beam_reorder(par, bt, bt, dev((2,), i32), k, v)
    with pytest.raises(ValueError):
        paged.beam_reorder(dev((2, 3), i32), bt, dev((2, 4, 4), i32), dev((2,), i32), k, v)
    for bad in ([1 << 31, 0, 0], [0.5, 0, 0], ["a", "b", "c"]):     # host numbers that the device's type does not hold
        with pytest.raises(ValueError):
            paged.block_tables(bad, n, 16, n, dev((1,), i32), t, tokens=5)
    with pytest.raises(ValueError):
        paged.new_cache(1, 1, 1, 8, dtype="float64")


M = 1 << 28     # apart: further than any of these calls' arrays are long


def tables_apart(**k):
    return tables(**{**dict(lengths=M, new=2 * M, free=3 * M, taken=4 * M, tables=5 * M, total=6 * M, taken_out=7 * M,
                            starts=8 * M, slots=9 * M, positions=10 * M), **k})


def append_apart(**k):
    return append(**{**dict(rows=M, positions=2 * M, slots=3 * M, cos=4 * M, sin=5 * M, k=6 * M, v=7 * M, q=8 * M), **k})


def attention_apart(**k):
    return attention(**{**dict(q=M, k=2 * M, v=3 * M, tables=4 * M, lengths=5 * M, out=6 * M), **k})


def select_apart(**k):
    return select(**{**dict(logits=M, scores=2 * M, done=3 * M, tokens=4 * M, parents=5 * M, scores_out=6 * M,
                            done_out=7 * M), **k})


def reorder_apart(**k):
    return reorder(**{**dict(parents=M, tables=2 * M, own=3 * M, lengths=4 * M, k=5 * M, v=6 * M), **k})


LD, QD, CACHE = 18 * 64 * 4, 14 * 64 * 4, 9 * 2 * 16 * 64 * 4      # bytes of a row, of its queries, of a layer's keys
OVERLAPPING = [
    # what every workgroup of the tables reads, while the first writes its results (3 requests, 4 blocks, 5 tokens)
    *(tables_apart(**{out: at * M + off}) for at, size in ((1, 12), (2, 12), (3, 32), (4, 4)) for off in (0, size - 4)
      for out in ("total", "starts", "taken_out", "positions", "tables")),
    *(tables_apart(slots=at * M - off) for at in (1, 2, 3, 4) for off in (0, 36)),
    tables_apart(total=5 * M + 44), tables_apart(starts=6 * M + 8), tables_apart(positions=9 * M + 36),
    tables_apart(taken_out=8 * M + 12),
    tables_apart(free=None, free_count=0, taken=None, taken_out=None, total=2 * M),
    append_apart(v=6 * M), append_apart(v=6 * M + CACHE - 16), append_apart(k=7 * M + CACHE - 16),
    append_apart(q=M, ldq=14 * 64), append_apart(q=M + 16), append_apart(q=M + QD, ldq=18 * 64),
    append_apart(q=M + LD - 4, ldq=18 * 64, n=2), append_apart(q=M - QD + 4, ldq=14 * 64, n=1),
    append_apart(q=M + 8 * LD, ldq=20 * 64, n=9),
    attention_apart(out=M, ldo=15 * 64), attention_apart(out=M + 4), attention_apart(out=M + QD),
    attention_apart(out=M + QD - 4, ldq=28 * 64, ldo=28 * 64), attention_apart(out=M + QD + 4, ldq=28 * 64, ldo=28 * 64),
    attention_apart(out=M - 4, batch=1),
    select_apart(scores_out=2 * M + 4), select_apart(done_out=3 * M + 7), select_apart(done_out=2 * M),
    select_apart(tokens=2 * M), select_apart(parents=3 * M - 28), select_apart(tokens=M + 8 * 100 * 4 - 8),
    select_apart(parents=4 * M + 60), select_apart(done_out=6 * M + 31),
    select_apart(scores_out=2 * M, parents=2 * M),
    reorder_apart(v=5 * M), reorder_apart(v=5 * M + 2 * CACHE - 16), reorder_apart(own=2 * M + 124),
    reorder_apart(parents=2 * M), reorder_apart(lengths=2 * M + 64), reorder_apart(own=6 * M), reorder_apart(parents=5 * M + 64),
]


@pytest.mark.parametrize("args", OVERLAPPING, ids=lambda a: a[0])
def test_results_that_overlap_are_refused(args):
    """Workgroups run in any order: a result in the place of an input that another one reads would be a race."""
    from cv3amd import _lib
    with pytest.raises(ValueError, match="overlap"):
        _lib.call(*args)


def test_results_in_place_and_beside_are_not_refused():
    """Queries in their own rows' place, results between rows of one pitch, neighbours: past the checks, to the launch
    that fails here for want of a GPU."""
    import torch
    from cv3amd import _lib
    if torch.cuda.device_count():
        pytest.skip("addresses that stand for memory")
    for args in (tables_apart(total=M + 12), tables_apart(starts=2 * M - 16), tables_apart(slots=10 * M - 40),
                 append_apart(q=M, ldq=18 * 64), append_apart(q=M + LD, n=1), append_apart(v=6 * M + CACHE),
                 append_apart(ld=32 * 64, ldq=32 * 64, q=M + LD), append_apart(ld=32 * 64, ldq=32 * 64, q=M - QD),
                 attention_apart(out=M), attention_apart(out=M, ldo=15 * 64, batch=1), attention_apart(out=M + 2 * QD),
                 attention_apart(out=M + QD, ldq=28 * 64, ldo=28 * 64), attention_apart(out=M - QD, ldq=30 * 64, ldo=30 * 64),
                 select_apart(scores_out=2 * M, done_out=3 * M), select_apart(parents=2 * M + 32),
                 reorder_apart(own=2 * M + 128), reorder_apart(v=5 * M + 2 * CACHE)):
        with pytest.raises(RuntimeError):
            _lib.call(*args)


@pytest.mark.parametrize("args", [
    attention_apart(batch=1 << 23, heads=1, kv_heads=1, ldq=64, ldo=64, out=1 << 40, k=1 << 41, v=1 << 42),
    attention_apart(batch=1 << 19, heads=16, kv_heads=16, ldq=1024, ldo=1024, out=1 << 40, k=1 << 41, v=1 << 42),
    select_apart(requests=1 << 23, beams=1, logits=1 << 40, **{x: i << 41 for i, x in enumerate(
        ("scores", "done", "tokens", "parents", "scores_out", "done_out"), 1)}),
], ids=lambda a: a[0])
def test_a_launch_of_all_its_threads_is_refused(args):
    """2^23 workgroups of 512 threads are 2^32, one more than a launch has."""
    from cv3amd import _lib
    with pytest.raises(ValueError, match="too many"):
        _lib.call(*args)


@pytest.mark.parametrize("held,beams,new,page", [([1], 1, 0, 1), ([160, 3, 32, 47], 4, 5, 16), ([16, 17, 15], 16, 0, 16),
                                                 ([5, 70000], 3, 40, 65536), ([7, 1, 900], 2, 33, 5)])
def test_reserved_pages(held, beams, new, page):
    """Every key of a prompt and of what follows has a page; a prompt's whole pages are its beams' together, and no
    other page is anybody else's."""
    import numpy as np
    from cv3amd.qwen2 import DeviceQwen2
    own, pages = DeviceQwen2._reserve(np.array(held, np.int32), beams, new, page)
    seen = []
    for n, tables in zip(held, own):
        whole, last = n // page, -(-(n + new) // page)
        assert (tables[:, :last] >= 0).all() and (tables[:, last:] == -1).all()
        assert (tables[:, :whole] == tables[0, :whole]).all()
        seen += [*tables[0, :whole], *tables[:, whole:last].reshape(-1)]
    assert sorted(seen) == list(range(pages)) and own.dtype == np.int32
