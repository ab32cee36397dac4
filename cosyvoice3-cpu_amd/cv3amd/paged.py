"""Paged key-value cache and beam search: several sequences over one set of weights.

The reference decodes one sequence into a contiguous cache (``KVCache``, cv3cpu/models/qwen2.py:74-121)
and draws one token (``_sample``, cv3cpu/models/llm.py:125-149).  These operators are the forms for many:

* ``block_tables``  pages and slots for new tokens, from the requests' lengths;
* ``append``        rotary on q and k, k and v into the cache (``apply_rope``, qwen2.py:64-71);
* ``attention``     one new token per sequence over the cache (``ops.sdpa``, cv3cpu/ops.py:267-300);
* ``beam_select``   the best continuations over beams and vocabulary (``log_softmax``, ops.py:90-93);
* ``beam_reorder``  tables and part-filled pages follow the chosen beams.

For sets of sequences that change, and texts that are scored:

* ``extend``          several new tokens per sequence over the cache, each seeing its own sequence up to itself;
* ``token_logprobs``  log probabilities of given tokens, entropy, the best alternatives;
* ``fork``            sequences that go on from others, whole pages shared;
* ``free_pages``      the pages that no sequence holds: what ``block_tables`` and ``fork`` take from;
* ``compact``         the pages that are held, into another cache.

A cache is a pair of device arrays (pages, kv heads, page, head dim): float32, float16, or bfloat16 as
uint16 bit patterns (``new_cache``).  Caches and tables live on the device and are updated in place;
everything else may be a NumPy array, uploaded for the call, and results come back as device arrays, or
as NumPy arrays where the first argument was one.  ``out`` takes the results' arrays from the caller.
Calls are enqueued on the calling thread's stream and do not synchronise; lengths, page ids and slots are
read on the device and checked there.

``attention`` and ``extend`` over long caches, ``beam_select``, ``compact``, ``token_logprobs`` of more than 8192 logits a
row, and ``free_pages`` of more than 131072 pages, 65536 table entries or 4096 tables take scratch from the allocator.  Captured into a graph they take it from the allocator's cache, and
the graph keeps it: run them once eagerly before each capture.  Where the cache has none, ``attention`` and ``extend``
run without splitting a sequence's keys over workgroups, which is slow for few long sequences; the others raise
``ScratchError``.  ``extend`` takes up to 69 to 136 MB by type and head dim from tables of more than 1024 keys on (2048 where many
sequences fill the machine), once a thread and once a graph.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple

import numpy as np

from . import _lib
from .device import DeviceArray, to_device

_ALL = 2**63 - 1             # a window of all keys
_F32, _I32, _I64, _U8 = (np.dtype(t) for t in (np.float32, np.int32, np.int64, np.uint8))
_CACHE_TYPES = {_F32: _lib.F32, np.dtype(np.float16): _lib.F16, np.dtype(np.uint16): _lib.BF16}


def new_cache(pages: int, kv_heads: int, page: int, dim: int, dtype="float32", layers: Optional[int] = None):
    """An empty (k, v) pair; ``dtype`` "float32", "float16" or "bfloat16" (held as uint16)."""
    kinds = {"float32": np.float32, "float16": np.float16, "bfloat16": np.uint16}
    if dtype not in kinds:
        raise ValueError(f"a cache is float32, float16 or bfloat16, not {dtype}")
    shape = (pages, kv_heads, page, dim) if layers is None else (layers, pages, kv_heads, page, dim)
    return DeviceArray(shape, kinds[dtype]).zero_(), DeviceArray(shape, kinds[dtype]).zero_()


def _in(x, dtype, name, shape=None) -> DeviceArray:
    """An input on the device, of the type and shape that the call takes."""
    if x.__class__ is DeviceArray and x.dtype is dtype and (shape is None or x.shape == shape):
        return x        # on every call's path
    if not isinstance(x, DeviceArray):
        a = np.asarray(x)
        if dtype.kind != "f" and a.size:
            lim = np.iinfo(dtype)
            if a.dtype.kind not in "iub" or int(a.min()) < lim.min or int(a.max()) > lim.max:
                raise ValueError(f"{name} does not hold whole numbers of {dtype}")
        x = to_device(np.ascontiguousarray(a, dtype=dtype))
    elif x.dtype != dtype:
        raise TypeError(f"{name} holds {x.dtype}, not {dtype}")
    if shape is not None and x.shape != shape:
        raise ValueError(f"{name} has the shape {x.shape}, not {shape}")
    return x


def _held(x, dtype, name, shape=None) -> DeviceArray:
    """An array that the call updates: the device's own."""
    if not isinstance(x, DeviceArray):
        raise TypeError(f"{name} is updated in place: a DeviceArray is needed")
    return _in(x, dtype, name, shape)


def _out(x, shape, dtype, name) -> DeviceArray:
    """A result's array: a new one, or the caller's."""
    if x.__class__ is DeviceArray and x.dtype is dtype and x.shape == shape:
        return x
    return DeviceArray(shape, dtype) if x is None else _held(x, dtype, name, shape)


def _outs(out, n):
    if out is None:
        return (None,) * n
    if len(out) != n or any(x is None for x in out):
        raise ValueError(f"out takes {n} arrays")
    return out


def _cache(k, v, ndim=4):
    if not isinstance(k, DeviceArray) or not isinstance(v, DeviceArray):
        raise TypeError("caches are DeviceArrays")
    if k.dtype not in _CACHE_TYPES or v.dtype != k.dtype:
        raise TypeError(f"caches are float32, float16 or uint16 (bfloat16), both alike: got {k.dtype} and {v.dtype}")
    if k.ndim != ndim or v.shape != k.shape:
        raise ValueError(f"caches are alike and of {ndim} axes: got {k.shape} and {v.shape}")
    return _CACHE_TYPES[k.dtype]


def _given(x, like):
    return x if isinstance(like, DeviceArray) else x.numpy()


def block_tables(lengths, new, page: int, free, taken, tables: DeviceArray, tokens: Optional[int] = None, out=None):
    """Pages and slots for ``new[r]`` more tokens of each request, after the ``lengths[r]`` it holds.

    ``tables`` (requests, blocks) int32 is updated: a block that begins takes the next of the page ids
    ``free``, from index ``taken[0]`` on, requests in order.  Returns (total, taken, starts, slots,
    positions): the lengths after the new tokens; the pages taken so far, more than ``len(free)`` where they
    ran out (their entries and slots are -1); each request's first token in the list (requests + 1); and the
    list of ``tokens`` slots (int64, page id * page + row) and positions, -1 behind the last token.
    ``tokens`` may be left out for a NumPy ``new``, whose sum it then is, or with ``out``.  Tokens past a
    request's table, or past ``tokens``, are not given.  ``free`` None: the tables hold every page already (a
    search's reserved pages), none is taken, and the result's ``taken`` is None.  ``out``: those five arrays,
    which share no memory with each other, ``tables`` or the inputs."""
    if not isinstance(tables, DeviceArray) or tables.ndim != 2:
        raise TypeError("tables is a DeviceArray (requests, blocks)")
    r, blocks = tables.shape
    given, out = out is not None, (None,) * 5 if out is None else out
    if len(out) != 5 or given and any(x is None for i, x in enumerate(out) if i != 1 or free is not None):
        raise ValueError("out takes five arrays: total, taken, starts, slots, positions")
    if tokens is None:
        if given:
            tokens = out[3].size
        elif isinstance(new, DeviceArray):
            raise ValueError("tokens, the length of the list, is needed with counts on the device")
        else:
            tokens = int(np.maximum(np.asarray(new, dtype=np.int64), 0).sum())
    first = lengths
    tables = _in(tables, _I32, "tables")
    lengths, new = _in(lengths, _I32, "lengths", (r,)), _in(new, _I32, "new", (r,))
    reserved = free is None
    if reserved:
        free_ptr, free_size, taken_ptr, took, took_ptr = None, 0, None, None, None
    else:
        free, taken = _in(free, _I32, "free"), _in(taken, _I32, "taken", (1,))
        took = _out(out[1], (1,), _I32, "taken")
        free_ptr, free_size, taken_ptr, took_ptr = free.ptr, free.size, taken.ptr, took.ptr
    total, starts = _out(out[0], (r,), _I32, "total"), _out(out[2], (r + 1,), _I32, "starts")
    slots, positions = _out(out[3], (tokens,), _I64, "slots"), _out(out[4], (tokens,), _I32, "positions")
    _lib.call("paged_tables", lengths.ptr, new.ptr, r, page, free_ptr, free_size, taken_ptr, tables.ptr, blocks, tokens,
              total.ptr, took_ptr, starts.ptr, slots.ptr, positions.ptr, None)
    if isinstance(first, DeviceArray):
        return total, took, starts, slots, positions
    return total.numpy(), None if reserved else took.numpy(), starts.numpy(), slots.numpy(), positions.numpy()


def append(rows, heads: int, positions, slots, cos, sin, k_cache: DeviceArray, v_cache: DeviceArray, out=None):
    """[q; k; v] rows into the cache: ``rows`` (n, (heads + 2 kv heads) * dim) float32, as the projection leaves
    them.  q and k are turned by the half-split rotary of ``positions`` (tables ``cos`` / ``sin`` (rows, dim),
    or None for none); k and v are rounded to the cache's type and written to ``slots``.  Returns the turned q
    (n, heads, dim).  A slot of -1 writes nothing; a position outside the tables writes nothing and gives
    zeros.  Slots are distinct."""
    kind = _cache(k_cache, v_cache)
    pages, kv_heads, page, d = k_cache.shape
    first = rows
    rows = _in(rows, _F32, "rows")
    if rows.ndim != 2 or rows.shape[1] != (heads + 2 * kv_heads) * d:
        raise ValueError(f"rows of {heads} + 2 x {kv_heads} heads of {d} are needed, got {rows.shape}")
    n = rows.shape[0]
    slots = _in(slots, _I64, "slots", (n,))
    if (cos is None) != (sin is None):
        raise ValueError("the rotary needs both tables")
    turn = cos is not None
    if turn:
        positions = _in(positions, _I32, "positions", (n,))
        cos = _in(cos, _F32, "cos")
        if cos.ndim != 2 or cos.shape[1] != d:
            raise ValueError(f"rotary tables are (rows, {d}), got {cos.shape}")
        sin = _in(sin, _F32, "sin", cos.shape)
    q = _out(out, (n, heads, d), _F32, "out")
    _lib.call("paged_append", rows.ptr, n, rows.shape[1], heads, kv_heads, d, positions.ptr if turn else None,
              slots.ptr, cos.ptr if turn else None, sin.ptr if turn else None, cos.shape[0] if turn else 0, kind,
              k_cache.ptr, v_cache.ptr, pages, page, q.ptr, heads * d, None)
    return _given(q, first)


def attention(q, k_cache: DeviceArray, v_cache: DeviceArray, tables, lengths, starts=None,
              scale: Optional[float] = None, out=None):
    """One new token per sequence: softmax(scale q . k) v of ``q`` (batch, heads, dim) over the ``lengths[b]`` keys
    that ``tables[b]`` (batch, blocks) lists, from key ``starts[b]`` on (a window; default 0).  Query heads
    share kv heads in groups.  A sequence with no key to see, such as a padding row, gives zeros, one whose
    scores are all -inf NaN (0 / 0); what lies in rows that are not seen reaches nothing.  Weights (at most one)
    times values are summed in float32 and then divided: a sum past the largest float is infinite."""
    kind = _cache(k_cache, v_cache)
    pages, kv_heads, page, d = k_cache.shape
    first = q
    q = _in(q, _F32, "q")
    if q.ndim != 3 or q.shape[2] != d:
        raise ValueError(f"queries are (batch, heads, {d}), got {q.shape}")
    b, h, _ = q.shape
    tables = _in(tables, _I32, "tables")
    if tables.ndim != 2 or tables.shape[0] != b:
        raise ValueError(f"tables are ({b}, blocks), got {tables.shape}")
    lengths = _in(lengths, _I32, "lengths", (b,))
    if starts is not None:
        starts = _in(starts, _I32, "starts", (b,))
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    o = _out(out, q.shape, _F32, "out")
    _lib.call("paged_attention", q.ptr, h * d, b, h, kv_heads, d, kind, k_cache.ptr, v_cache.ptr, pages, page,
              tables.ptr, tables.shape[1], lengths.ptr, starts.ptr if starts is not None else None, float(scale),
              o.ptr, h * d, None)
    return _given(o, first)


def beam_select(logits, scores, done, stop: Tuple[int, int], ban: Tuple[int, int] = (0, 0),
                pad: Optional[int] = None, out=None):
    """The best continuations of each request's beams: ``logits`` (requests, beams, vocab), ``scores`` and
    ``done`` (requests, beams) float32 and uint8. Beam b with token t is worth scores[b] +
    log_softmax(logits[b])[t], formed in float64 but for the exponentials of the softmax's sum, which are float32
    (its log within 1e-6: candidates of two beams that lie closer may change places, those of one beam never); an
    ended beam goes on with ``pad`` (default the first stop id) at its own score. Tokens of [ban[0], ban[1]) are
    not chosen (below a minimal length, the stop ids). Returns (tokens int64, parents int32, scores, done), best
    first; equal values: the lower beam, in one beam the larger logit, then the lower token. ``done`` of the
    result: the parent's, or a token of [stop[0], stop[1]). ``out``: those four arrays; scores and done may be the
    call's own."""
    first = logits
    logits = _in(logits, _F32, "logits")
    if logits.ndim != 3:
        raise ValueError(f"logits are (requests, beams, vocab), got {logits.shape}")
    r, w, v = logits.shape
    scores, done = _in(scores, _F32, "scores", (r, w)), _in(done, _U8, "done", (r, w))
    shape, out = (r, w), _outs(out, 4)
    tokens, parents = _out(out[0], shape, _I64, "tokens"), _out(out[1], shape, _I32, "parents")
    scored, ended = _out(out[2], shape, _F32, "scores"), _out(out[3], shape, _U8, "done")
    _lib.call("beam_select", logits.ptr, r, w, v, scores.ptr, done.ptr, stop[0], stop[1], ban[0], ban[1],
              stop[0] if pad is None else pad, tokens.ptr, parents.ptr, scored.ptr, ended.ptr, None)
    return tuple(_given(x, first) for x in (tokens, parents, scored, ended))


def beam_reorder(parents, tables: DeviceArray, own, lengths, k_cache: DeviceArray, v_cache: DeviceArray):
    """Beams follow their ``parents`` (requests, beams) int32, in place.  Beam w of request r writes the pages
    ``own[r, w]`` (requests, beams, blocks); of the ``lengths[r]`` keys that the request's beams hold, whole
    pages may lie with any beam (``tables``, shaped as ``own``), the part-filled last one is its own.  A
    beam's table becomes its parent's up to there and its own pages behind; the part-filled page's rows are
    copied from the parent's page, in every layer of the caches (layers, pages, kv heads, page, dim), or
    (pages, kv heads, page, dim).  Nothing is copied for a whole prompt or page."""
    kind = _cache(k_cache, v_cache, k_cache.ndim if getattr(k_cache, "ndim", 0) == 5 else 4)
    layers = k_cache.shape[0] if k_cache.ndim == 5 else 1
    pages, kv_heads, page, d = k_cache.shape[-4:]
    if not isinstance(tables, DeviceArray) or tables.ndim != 3:
        raise TypeError("tables is a DeviceArray (requests, beams, blocks)")
    r, w, blocks = tables.shape
    _held(tables, _I32, "tables")
    own, parents = _in(own, _I32, "own", tables.shape), _in(parents, _I32, "parents", (r, w))
    lengths = _in(lengths, _I32, "lengths", (r,))
    _lib.call("beam_reorder", parents.ptr, r, w, tables.ptr, own.ptr, blocks, lengths.ptr, kind, k_cache.ptr,
              v_cache.ptr, layers, pages, kv_heads, page, d, None)


def extend(q, k_cache: DeviceArray, v_cache: DeviceArray, tables, lengths, starts, window: Optional[int] = None,
           scale: Optional[float] = None, out=None):
    """New tokens of several sequences over the cache: softmax(scale q . k) v of the ragged list ``q`` (rows, heads,
    dim).  Rows ``starts[b]`` to ``starts[b + 1]`` (batch + 1, rising, as ``block_tables`` gives them) are sequence b's
    last tokens, whose keys are in the cache already (``append``): the last of them is at position ``lengths[b]`` - 1.
    A query at position p sees the keys up to p that ``tables[b]`` (batch, blocks) lists, the last ``window`` of them
    alone if that is given.  Query heads share kv heads in groups.  Rows outside [starts[0], starts[-1]) are left as
    they are (zeros in an array that the call makes).  A query with no key to see gives zeros, one whose scores are
    all -inf NaN (0 / 0); what lies in rows that are not seen reaches nothing.  Queries and weights enter the products
    with 22 bits of the largest in their row or tile, float32 keys and values too, and sums are float32: the error is
    that of float32 arithmetic.  Rows where that would lose more (outputs far smaller than the largest value, small
    numbers that count under far larger ones, results that are not finite) are formed again in float32, one after the
    other, at 90 to 180 times the price.  ``out`` may be ``q``."""
    kind = _cache(k_cache, v_cache)
    pages, kv_heads, page, d = k_cache.shape
    first = q
    q = _in(q, _F32, "q")
    if q.ndim != 3 or q.shape[2] != d:
        raise ValueError(f"queries are (rows, heads, {d}), got {q.shape}")
    n, h, _ = q.shape
    tables = _in(tables, _I32, "tables")
    if tables.ndim != 2:
        raise ValueError(f"tables are (batch, blocks), got {tables.shape}")
    b, blocks = tables.shape
    lengths, starts = _in(lengths, _I32, "lengths", (b,)), _in(starts, _I32, "starts", (b + 1,))
    if window is not None and window < 1:
        raise ValueError(f"a window of {window} keys")
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    o = DeviceArray(q.shape, _F32).zero_() if out is None else _out(out, q.shape, _F32, "out")
    _lib.call("paged_extend", q.ptr, h * d, n, h, kv_heads, d, kind, k_cache.ptr, v_cache.ptr, pages, page, tables.ptr,
              blocks, lengths.ptr, starts.ptr, b, _ALL if window is None else window, float(scale), o.ptr, h * d, None)
    return _given(o, first)


def token_logprobs(logits, tokens, top: int = 0, out=None):
    """What given tokens are worth: of each row of ``logits`` (rows, vocab) the log probability of ``tokens`` (rows,)
    int64 (0 for a token outside the vocabulary, such as a padding row's -1), the entropy of the distribution in nats,
    and its ``top`` (0 to 32) best tokens with their log probabilities, best first, equal logits by the lower token.
    Returns (logprobs, entropy, ids (rows, top) int64, values (rows, top)).  Formed in float64 but for the exponentials
    of the sums, which are float32.  A row with a NaN or +inf, or of -inf alone, gives NaN (and ids, for which NaN counts
    as -inf).  ``out``: those four arrays."""
    first = logits
    logits = _in(logits, _F32, "logits")
    if logits.ndim != 2:
        raise ValueError(f"logits are (rows, vocab), got {logits.shape}")
    n, v = logits.shape
    tokens = _in(tokens, _I64, "tokens", (n,))
    out = _outs(out, 4)
    if not 0 <= top <= min(32, v):
        raise ValueError(f"0 to 32 alternatives out of {v} tokens, not {top}")
    lp, entropy = _out(out[0], (n,), _F32, "logprobs"), _out(out[1], (n,), _F32, "entropy")
    ids, values = _out(out[2], (n, top), _I64, "ids"), _out(out[3], (n, top), _F32, "values")
    _lib.call("token_logprobs", logits.ptr, n, v, tokens.ptr, top, lp.ptr, entropy.ptr, ids.ptr, values.ptr, None)
    return tuple(_given(x, first) for x in (lp, entropy, ids, values))


def _layered(k, v):
    """(type, layers, pages, kv heads, page, dim) of caches with or without an axis of layers."""
    kind = _cache(k, v, k.ndim if getattr(k, "ndim", 0) == 5 else 4)
    return (kind, k.shape[0] if k.ndim == 5 else 1, *k.shape[-4:])


def fork(parents, children, tables: DeviceArray, lengths: DeviceArray, free, taken, k_cache: DeviceArray,
         v_cache: DeviceArray, out=None):
    """Sequences that go on from others, in place: row ``children[i]`` of ``tables`` (sequences, blocks) and ``lengths``
    becomes row ``parents[i]``.  Whole pages are shared; the rows of a part-filled last page are copied into a page of
    the child's own, the next of the page ids ``free`` from index ``taken[0]`` on, forks in order, in every layer of the
    caches (layers, pages, kv heads, page, dim), or (pages, kv heads, page, dim).  Returns the pages taken so far, more
    than ``len(free)`` where they ran out (the child's entry is then -1).  A part-filled page that the parent lists as
    absent is absent (-1) for the child too, and takes no page.  Children are distinct and no parents of the call; a fork
    whose child is, or whose rows do not exist, is not made."""
    kind, layers, pages, kv_heads, page, d = _layered(k_cache, v_cache)
    if not isinstance(tables, DeviceArray) or tables.ndim != 2:
        raise TypeError("tables is a DeviceArray (sequences, blocks)")
    rows, blocks = tables.shape
    _held(tables, _I32, "tables")
    _held(lengths, _I32, "lengths", (rows,))
    first = taken
    parents = _in(parents, _I32, "parents")
    children = _in(children, _I32, "children", parents.shape)
    if parents.ndim != 1:
        raise ValueError(f"parents are a list, got {parents.shape}")
    free, taken = _in(free, _I32, "free"), _in(taken, _I32, "taken", (1,))
    took = _out(out, (1,), _I32, "out")
    _lib.call("paged_fork", parents.ptr, children.ptr, parents.size, tables.ptr, rows, blocks, lengths.ptr, free.ptr,
              free.size, taken.ptr, took.ptr, kind, k_cache.ptr, v_cache.ptr, layers, pages, kv_heads, page, d, None)
    return _given(took, first)


def free_pages(tables, lengths, page: int, pages: int, out=None):
    """The page ids of [0, ``pages``) that no sequence holds, ascending: (ids (pages,) int32 with -1 behind the last,
    their number (1,) int32).  Sequence b holds the first ceil(``lengths[b]`` / ``page``) entries of its row of ``tables``
    (sequences, blocks), so one that has ended is given up by setting its length to 0.  The ids are ``free`` for
    ``block_tables`` and ``fork``, with ``taken`` set to 0."""
    first = tables
    tables = _in(tables, _I32, "tables")
    if tables.ndim != 2:
        raise ValueError(f"tables are (sequences, blocks), got {tables.shape}")
    rows, blocks = tables.shape
    if pages < 1:
        raise ValueError(f"a cache of {pages} pages")
    lengths, out = _in(lengths, _I32, "lengths", (rows,)), _outs(out, 2)
    free, count = _out(out[0], (pages,), _I32, "free"), _out(out[1], (1,), _I32, "count")
    _lib.call("paged_free", tables.ptr, rows, blocks, lengths.ptr, page, pages, free.ptr, count.ptr, None)
    return _given(free, first), _given(count, first)


def compact(tables, lengths, k_cache: DeviceArray, v_cache: DeviceArray, k_new: DeviceArray, v_new: DeviceArray,
            out=None):
    """What is held of a cache, moved into another one of any number of pages (a smaller one for what is left, a larger
    one to go on): every page that a sequence holds (as in ``free_pages``) is copied once, in the order of their ids, to
    the pages 0, 1, .. of ``k_new`` and ``v_new``, in every layer.  Returns (tables (sequences, blocks) for the new cache,
    -1 behind a sequence's last block, and the number of pages held (1,), more than the new cache has where it was
    too small: what did not fit is -1).  Pages that sequences share stay shared.  The least of both caches' pages and the
    tables' entries, times the layers, is below 2^24."""
    kind, layers, pages, kv_heads, page, d = _layered(k_cache, v_cache)
    if _layered(k_new, v_new) != (kind, layers, k_new.shape[-4], kv_heads, page, d) or k_new.ndim != k_cache.ndim:
        raise ValueError(f"the new caches are {k_new.shape}, those in use {k_cache.shape}")
    first = tables
    tables = _in(tables, _I32, "tables")
    if tables.ndim != 2:
        raise ValueError(f"tables are (sequences, blocks), got {tables.shape}")
    rows, blocks = tables.shape
    lengths, out = _in(lengths, _I32, "lengths", (rows,)), _outs(out, 2)
    turned, used = _out(out[0], tables.shape, _I32, "tables"), _out(out[1], (1,), _I32, "used")
    _lib.call("paged_compact", tables.ptr, rows, blocks, lengths.ptr, kind, k_cache.ptr, v_cache.ptr, layers, pages,
              kv_heads, page, d, k_new.ptr, v_new.ptr, k_new.shape[-4], turned.ptr, used.ptr, None)
    return _given(turned, first), _given(used, first)
