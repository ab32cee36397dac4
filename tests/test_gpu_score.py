"""Log probabilities of given tokens, entropy and best alternatives on the GPU, against NumPy in 64 bits.

Tolerance.  Each exponential is float32, within 2^-22 of its own size (its argument x - max, at most 2^7 where it counts,
is rounded to 2^-24 of itself, and so is the product with log2 e: 2^-17 of an exponential of e^-88, 2^-21 of those that
count); sums are float64 but for groups of four.  So the log of the sum is within 1e-6, as is the entropy relative to
1 + its size, and a result has its own 2^-24 besides.
"""

import numpy as np
import pytest

from test_gpu_paged import dev

pytestmark = pytest.mark.gpu

I64 = np.int64


@pytest.fixture(scope="module")
def paged(gpu):
    from cv3amd import paged
    return paged


def score_ref(x, tokens, top):
    x64 = x.astype(np.float64)
    n, v = x.shape
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        mx = x64.max(axis=1, keepdims=True)
        e = np.exp(x64 - mx)
        s = e.sum(axis=1, keepdims=True)
        lse = mx + np.log(s)
        y = np.where(x64 == -np.inf, 0.0, x64 - mx)
        entropy = (np.log(s) - (e * y).sum(axis=1, keepdims=True) / s)[:, 0]
        entropy[~np.isfinite(lse[:, 0])] = np.nan
        given = (tokens >= 0) & (tokens < v)
        lp = np.where(given, x64[np.arange(n), np.where(given, tokens, 0)] - lse[:, 0], 0.0)
        order = np.where(np.isnan(x), -np.inf, x)
        ids = np.argsort(-order, axis=1, kind="stable")[:, :top]
        values = np.take_along_axis(np.where(np.isnan(x64), -np.inf, x64), ids, axis=1) - lse
        # results are float32: -3e38 beside a maximum of 3e38 is worth -6e38, past its largest (3.4e38)
        most = np.finfo(np.float32).max
        lp, values = (np.where(np.abs(a) > most, np.sign(a) * np.inf, a) for a in (lp, values))
    return lp, entropy, ids, values


def close(got, want, slack=1e-6):
    bad = ~np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[bad & ~np.isnan(want)], want[bad & ~np.isnan(want)])
    assert np.all(np.abs(got - want)[~bad] <= slack + 2.0 ** -24 * np.abs(want[~bad]))


def check(paged, x, tokens, top):
    x, tokens = np.ascontiguousarray(x, np.float32), np.asarray(tokens, I64)
    lp, entropy, ids, values = paged.token_logprobs(x, tokens, top=top)
    want = score_ref(x, tokens, top)
    assert np.array_equal(ids, want[2])
    close(lp, want[0])
    fine = np.isfinite(want[1])
    assert np.array_equal(np.isnan(entropy), np.isnan(want[1]))
    assert np.all(np.abs(entropy - want[1])[fine] <= 1e-6 * (1 + want[1][fine]))
    close(values, want[3])


SIZES = [(1, 1, 1), (1, 6761, 5), (6, 6761, 0), (70, 6761, 32), (3, 2, 2), (5, 255, 16), (4, 256, 8), (7, 257, 9), (2, 32, 32),
         (3, 1023, 1), (2, 8191, 8), (2, 8192, 8), (2, 8193, 8), (3, 16385, 32), (5, 128000, 5), (1, 151936, 20),
         (2, 1 << 19, 32), (2, (1 << 19) - 1, 0), (2000, 300, 3), (300, 20001, 2),
         (4, 2047, 5), (3, 2048, 32), (3, 2049, 32), (2, 4095, 0), (2, 4096, 8), (2, 4097, 9)]


@pytest.mark.parametrize("rows,vocab,top", SIZES)
def test_scores(paged, rows, vocab, top):
    rng = np.random.default_rng([rows, vocab])
    x = 2.5 * rng.normal(size=(rows, vocab))
    tokens = rng.integers(0, vocab, rows)
    check(paged, x, tokens, top)
    tokens[rng.random(rows) < 0.3] = -1                 # padded rows, and ids outside the vocabulary
    tokens[0] = vocab
    check(paged, 10.0 * x, tokens, top)


@pytest.mark.parametrize("vocab", [40, 2048, 4000, 6761, 20000])
def test_scores_of_equal_logits(paged, vocab):
    """Ties go to the lower token, wherever their slices lie; more equal logits than the list of a slice holds."""
    rng = np.random.default_rng(vocab)
    x = np.stack([np.zeros(vocab), rng.integers(-2, 3, vocab), np.where(np.arange(vocab) % 3 == 0, 1.0, -0.0),
                  np.where(np.arange(vocab) == vocab - 1, 5.0, 0.0), -np.arange(vocab, dtype=float), np.arange(vocab) / 7.0])
    for top in (1, 5, 8, 9, 32):
        check(paged, x, [0, vocab - 1, vocab // 2, 1, vocab - 1, 0], top)


@pytest.mark.parametrize("vocab", [64, 2047, 4095, 6761, 20000])
def test_scores_that_are_no_numbers(paged, vocab):
    """-inf (a banned token) adds nothing; a NaN, +inf, or -inf alone makes its own row NaN."""
    rng = np.random.default_rng(vocab + 1)
    x = rng.normal(size=(9, vocab)).astype(np.float32)
    x[1, ::2] = -np.inf
    x[2, :] = -np.inf
    x[2, vocab - 3] = 4.0                               # one token left
    x[3, :] = -np.inf
    x[4, vocab // 2] = np.nan
    x[5, 7] = np.inf
    x[6, vocab - 1] = np.nan
    x[6, :vocab - 1] = -np.inf
    x[7] = 3e38 * np.sign(x[7])
    tokens = [0, 2, vocab - 3, 5, 6, 7, 8, int(np.argmin(x[7])), -1]
    for top in (0, 5, 32):
        check(paged, x, tokens, top)
    x[4] = np.nan
    check(paged, x, [-1] * 9, 3)


def test_scores_of_nothing(paged):
    lp, entropy, ids, values = paged.token_logprobs(np.zeros((0, 50), np.float32), np.zeros(0, I64), top=4)
    assert lp.shape == entropy.shape == (0,) and ids.shape == values.shape == (0, 4)


def test_scores_of_an_unaligned_view(paged):
    """Rows of an odd number of logits, from any 4-byte boundary."""
    from cv3amd import _lib
    rng = np.random.default_rng(3)
    x, t = rng.normal(size=(5, 9001)).astype(np.float32), rng.integers(0, 9001, 5)
    flat, tokens = dev(np.concatenate([[7.0], x.reshape(-1)]).astype(np.float32)), dev(t.astype(I64))
    lp, en, ids, va = dev(np.zeros(5, np.float32)), dev(np.zeros(5, np.float32)), dev(np.zeros((5, 6), I64)), dev(np.zeros((5, 6), np.float32))
    _lib.call("token_logprobs", flat.ptr + 4, 5, 9001, tokens.ptr, 6, lp.ptr, en.ptr, ids.ptr, va.ptr, None)
    want = score_ref(x, t, 6)
    close(lp.numpy(), want[0])
    close(en.numpy(), want[1], 1e-5)
    assert np.array_equal(ids.numpy(), want[2])
    close(va.numpy(), want[3])


def test_scores_on_an_explicit_stream_and_captured(gpu, paged):
    from cv3amd import _lib, device
    rng = np.random.default_rng(4)
    for vocab in (6761, 30000):
        x = [rng.normal(size=(20, vocab)).astype(np.float32) for _ in range(2)]
        t = rng.integers(0, vocab, 20)
        want = [score_ref(y, t, 5) for y in x]
        xd, td, st = dev(x[0]), dev(t.astype(I64)), device.Stream()
        out = (dev(np.zeros(20, np.float32)), dev(np.zeros(20, np.float32)), dev(np.zeros((20, 5), I64)), dev(np.zeros((20, 5), np.float32)))
        device.synchronize()
        _lib.call("token_logprobs", xd.ptr, 20, vocab, td.ptr, 5, *(o.ptr for o in out), st.handle)
        _lib.call("stream_sync", st.handle)
        assert np.array_equal(out[2].numpy(), want[0][2])
        close(out[0].numpy(), want[0][0])
        paged.token_logprobs(xd, td, 5)         # leaves its scratch in the allocator's cache
        g = device.Graph()
        with g:
            paged.token_logprobs(xd, td, 5, out=out)
        for i in (0, 1, 0, 1):
            xd.copy_from(x[i])
            g.launch()
            got = [o.numpy() for o in out]
            eager = [o.numpy() for o in paged.token_logprobs(xd, td, 5)]
            assert all(np.array_equal(a, b) for a, b in zip(got, eager))
            assert np.array_equal(got[2], want[i][2])
            close(got[0], want[i][0])


def test_scores_captured_without_scratch_are_refused(gpu, paged):
    from cv3amd import _lib, device
    x, t = dev(np.zeros((4, 20000), np.float32)), dev(np.zeros(4, I64))
    out = paged.token_logprobs(x, t, 3)
    device.synchronize()
    _lib.call("empty_cache")
    g = device.Graph()
    with g:
        with pytest.raises(_lib.ScratchError):
            paged.token_logprobs(x, t, 3, out=out)
