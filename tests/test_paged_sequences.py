"""Refusals of the entry points for changing sets of sequences and for scores: argument checks run on the host before
anything is enqueued, so they need no GPU."""

import numpy as np
import pytest

P = 1 << 20    # stands for a device address: never read, every call here is refused or has nothing to do
FAR = 1 << 45  # one that overlaps nothing


def extend(**k):
    a = dict(q=P, ldq=14 * 64, n=20, heads=14, kv_heads=2, d=64, type=0, k=FAR, v=FAR, pages=9, page=16, tables=2 * P,
             blocks=4, lengths=3 * P, starts=4 * P, batch=2, window=1 << 40, scale=0.125, out=P, ldo=14 * 64)
    a.update(k)
    return ("paged_extend", *a.values(), None)


def score(**k):
    a = dict(logits=P, rows=3, vocab=100, tokens=2 * P, top=4, logprobs=3 * P, entropy=4 * P, ids=5 * P, values=6 * P)
    a.update(k)
    return ("token_logprobs", *a.values(), None)


def fork(**k):
    a = dict(parents=P, children=P, forks=2, tables=2 * P, rows=5, blocks=4, lengths=3 * P, free=P, free_count=6, taken=P,
             taken_out=4 * P, type=0, k=FAR, v=2 * FAR, layers=2, pages=9, kv_heads=2, page=16, d=64)
    a.update(k)
    return ("paged_fork", *a.values(), None)


def free(**k):
    a = dict(tables=P, rows=3, blocks=4, lengths=P, page=16, pages=50, free=2 * P, count=3 * P)
    a.update(k)
    return ("paged_free", *a.values(), None)


def compact(**k):
    a = dict(tables=P, rows=3, blocks=4, lengths=P, type=0, k=FAR, v=FAR, layers=2, pages=9, kv_heads=2, page=16, d=64,
             k_new=2 * FAR, v_new=3 * FAR, pages_new=5, tables_new=2 * P, used=3 * P)
    a.update(k)
    return ("paged_compact", *a.values(), None)


REFUSED = [
    extend(heads=15), extend(heads=0), extend(kv_heads=0), extend(d=12), extend(d=0), extend(d=264), extend(type=3), extend(k=None),
    extend(v=FAR + 8), extend(pages=0), extend(pages=1 << 31), extend(page=0), extend(page=70000), extend(blocks=0),
    extend(blocks=1 << 30), extend(n=-1), extend(n=1 << 40), extend(n=600000), extend(batch=-1), extend(batch=1 << 40),
    extend(window=0), extend(window=-5), extend(ldq=14 * 64 - 1), extend(ldo=0), extend(q=None), extend(tables=None),
    extend(lengths=None), extend(starts=None), extend(out=None), extend(out=P + 4), extend(out=2 * P), extend(out=3 * P),
    extend(out=4 * P), extend(out=FAR), extend(heads=1 << 17, kv_heads=1),
    score(rows=-1), score(rows=1 << 40), score(vocab=0), score(vocab=(1 << 19) + 1), score(top=-1), score(top=33),
    score(vocab=3), score(logits=None), score(tokens=None), score(logprobs=None), score(entropy=None), score(ids=None),
    score(values=None), score(logprobs=P), score(entropy=3 * P), score(ids=2 * P), score(values=5 * P), score(entropy=P + 8),
    fork(forks=-1), fork(forks=4097), fork(rows=-1), fork(rows=65537), fork(blocks=0), fork(page=0), fork(type=9), fork(k=None),
    fork(v=FAR + 4), fork(layers=0), fork(layers=70000), fork(pages=0), fork(kv_heads=0), fork(d=20), fork(parents=None),
    fork(children=None), fork(tables=None), fork(lengths=None), fork(free=None), fork(free_count=-1), fork(taken=None),
    fork(taken_out=None), fork(taken_out=P), fork(tables=P), fork(lengths=2 * P), fork(k=2 * FAR), fork(k=P),
    free(rows=-1), free(blocks=0), free(blocks=1 << 40), free(page=0), free(pages=0), free(pages=(1 << 24) + 1), free(tables=None),
    free(lengths=None), free(free=None), free(count=None), free(free=P), free(count=2 * P + 8), free(count=P),
    compact(rows=-1), compact(blocks=0), compact(type=-1), compact(k=None), compact(v=FAR + 2), compact(layers=0),
    compact(pages=0), compact(pages=(1 << 24) + 1), compact(kv_heads=0), compact(page=0), compact(d=4), compact(k_new=None),
    compact(v_new=3 * FAR + 8), compact(pages_new=0), compact(tables=None), compact(lengths=None), compact(tables_new=None),
    compact(used=None), compact(k_new=FAR), compact(v_new=2 * FAR), compact(tables_new=P), compact(used=2 * P), compact(used=FAR),
]


@pytest.mark.parametrize("args", REFUSED, ids=lambda a: a[0])
def test_refused_before_anything_is_enqueued(args):
    from cv3amd import _lib
    with pytest.raises(ValueError):
        _lib.call(*args)
    assert _lib.lib().cv3_last_error()


def test_nothing_to_do_is_not_an_error():
    from cv3amd import _lib
    _lib.call(*extend(n=0, q=None, out=None))
    _lib.call(*extend(batch=0, tables=None, lengths=None, starts=None))
    _lib.call(*score(rows=0, logits=None, tokens=None))


def test_python_checks_types_and_shapes():
    """The binding's own checks come before any device memory is touched."""
    from cv3amd import paged
    from cv3amd.device import DeviceArray

    class Memory:
        nbytes = 1 << 30

        def __init__(self, at):
            self.ptr = at

    where = iter(range(1, 1000))

    def d(shape, dtype=np.float32):
        return DeviceArray(shape, dtype, block=Memory(next(where) << 32))

    i32, i64 = np.int32, np.int64
    k, v, q = d((9, 2, 16, 64)), d((9, 2, 16, 64)), d((20, 14, 64))
    t, n, s = d((3, 4), i32), d((3,), i32), d((4,), i32)
    refused = [
        (TypeError, lambda: paged.extend(q, np.zeros((9, 2, 16, 64), np.float32), v, t, n, s)),
        (TypeError, lambda: paged.extend(q, k, d((9, 2, 16, 64), np.float16), t, n, s)),
        (ValueError, lambda: paged.extend(q, k, d((8, 2, 16, 64)), t, n, s)),
        (ValueError, lambda: paged.extend(d((20, 14, 32)), k, v, t, n, s)),
        (ValueError, lambda: paged.extend(d((20, 14 * 64)), k, v, t, n, s)),
        (ValueError, lambda: paged.extend(q, k, v, d((12,), i32), n, s)),
        (ValueError, lambda: paged.extend(q, k, v, t, d((4,), i32), s)),
        (ValueError, lambda: paged.extend(q, k, v, t, n, d((3,), i32))),
        (TypeError, lambda: paged.extend(q, k, v, t, n, d((4,), i64))),
        (ValueError, lambda: paged.extend(q, k, v, t, n, s, window=0)),
        (ValueError, lambda: paged.extend(q, k, v, t, n, s, out=d((20, 14 * 64)))),
        (TypeError, lambda: paged.extend(q, k, v, t, n, s, out=d((20, 14, 64), np.float16))),
        (ValueError, lambda: paged.extend(d((20, 15, 64)), k, v, t, n, s, out=d((20, 15, 64)))),
        (ValueError, lambda: paged.token_logprobs(d((2, 3, 4)), d((2,), i64))),
        (ValueError, lambda: paged.token_logprobs(d((2, 50)), d((3,), i64))),
        (TypeError, lambda: paged.token_logprobs(d((2, 50)), d((2,), i32))),
        (ValueError, lambda: paged.token_logprobs(d((2, 50)), d((2,), i64), top=33)),
        (ValueError, lambda: paged.token_logprobs(d((2, 50)), d((2,), i64), out=(d((2,)),))),
        (ValueError, lambda: paged.token_logprobs(d((2, 50)), d((2,), i64), 3, out=(d((2,)), d((2,)), d((2, 2), i64), d((2, 3))))),
        (TypeError, lambda: paged.fork([0], [1], np.zeros((3, 4), i32), n, d((5,), i32), d((1,), i32), k, v)),
        (TypeError, lambda: paged.fork([0], [1], t, np.zeros(3, i32), d((5,), i32), d((1,), i32), k, v)),
        (ValueError, lambda: paged.fork(d((2,), i32), d((1,), i32), t, n, d((5,), i32), d((1,), i32), k, v)),
        (ValueError, lambda: paged.fork(d((2,), i32), d((2,), i32), t, d((4,), i32), d((5,), i32), d((1,), i32), k, v)),
        (ValueError, lambda: paged.fork(d((1, 1), i32), d((1, 1), i32), t, n, d((5,), i32), d((1,), i32), k, v)),
        (ValueError, lambda: paged.fork(d((1,), i32), d((1,), i32), t, n, d((5,), i32), d((2,), i32), k, v)),
        (ValueError, lambda: paged.free_pages(d((12,), i32), n, 16, 50)),
        (ValueError, lambda: paged.free_pages(t, d((4,), i32), 16, 50)),
        (ValueError, lambda: paged.free_pages(t, n, 16, 50, out=(d((49,), i32), d((1,), i32)))),
        (TypeError, lambda: paged.free_pages(d((3, 4)), n, 16, 50)),
        (ValueError, lambda: paged.free_pages(t, n, 16, 0)),
        (ValueError, lambda: paged.free_pages(t, n, 16, -1)),
        (ValueError, lambda: paged.compact(t, n, k, v, d((5, 2, 8, 64)), d((5, 2, 8, 64)))),
        (ValueError, lambda: paged.compact(t, n, k, v, d((1, 5, 2, 16, 64)), d((1, 5, 2, 16, 64)))),
        (ValueError, lambda: paged.compact(t, n, k, v, d((5, 2, 16, 64), np.float16), d((5, 2, 16, 64), np.float16))),
        (TypeError, lambda: paged.compact(t, n, k, v, np.zeros((5, 2, 16, 64)), v)),
        (ValueError, lambda: paged.compact(t, d((2,), i32), k, v, d((5, 2, 16, 64)), d((5, 2, 16, 64)))),
        (ValueError, lambda: paged.compact(t, n, k, v, d((5, 2, 16, 64)), d((5, 2, 16, 64)), out=(t, d((1,), i32)))),
    ]
    for error, call in refused:
        with pytest.raises(error):
            call()
