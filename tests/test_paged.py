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
