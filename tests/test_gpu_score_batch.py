"""DeviceQwen2.score_batch: given continuations of several prompts over the paged cache, against the oracle's LM run over
one sequence at a time (Qwen2-0.5B's geometry, two layers, synthetic weights)."""

import numpy as np
import pytest

from test_gpu_batch import logp, prompts, setup

pytestmark = pytest.mark.gpu

# logits are within 1e-5 of the oracle's (as in generate_batch's tests, at magnitudes of about 1): a log probability, a
# logit less the logarithm of a sum of exponentials, within twice that
NEAR = 2e-5


def wanted(lm, prompt, tokens):
    """Log probabilities (float64, whole rows) before each token of a continuation."""
    x = prompt if len(tokens) < 2 else np.concatenate([prompt, lm.speech_emb(tokens[:-1])])
    z = lm.head(lm.body.forward(x, lm.body.new_cache())[len(prompt) - 1:]).astype(np.float64)
    z -= z.max(axis=1, keepdims=True)
    return z - np.log(np.exp(z).sum(axis=1, keepdims=True))


def check(lm, xs, texts, got, top, near=NEAR):
    assert [len(g) for g in got] == [len(t) for t in texts]
    for x, cs, gs in zip(xs, texts, got):
        for c, (lp, entropy, ids, values) in zip(cs, gs):
            n = len(c)
            assert lp.shape == entropy.shape == (n,) and ids.shape == values.shape == (n, top) and ids.dtype == np.int64
            if not n:
                continue
            p = wanted(lm, x, [int(t) for t in c])
            assert np.abs(lp - p[np.arange(n), c]).max() <= near
            # -sum p log p: each log probability off by up to near, its weight by that share of itself
            assert np.abs(entropy + (np.exp(p) * p).sum(axis=1)).max() <= near * (2 + np.abs(p).max())
            best = -np.sort(-p, axis=1)[:, :top]
            assert np.abs(values - best).max(initial=0) <= near
            assert np.abs(values - np.take_along_axis(p, ids, axis=1)).max(initial=0) <= near


def tokens(rng, *counts):
    return [rng.integers(0, 6761, n).tolist() for n in counts]


@pytest.mark.parametrize("profile,page,top", [("per_channel", 16, 4), ("balanced", 5, 0), ("tiny", 64, 32)])
def test_scores_are_the_oracles(gpu, profile, page, top):
    from cv3amd.qwen2 import DeviceQwen2
    lm, store = setup(profile)
    d = DeviceQwen2(store, cap=64)
    rng = np.random.default_rng(21)
    xs = prompts(rng, (37, 1, 16, 50))
    texts = [tokens(rng, 3, 17, 1), tokens(rng, 2), [], tokens(rng, 0, 8, 1, 30, 2)]
    check(lm, xs, texts, d.score_batch(xs, texts, top, page=page), top)


def test_one_token_each_and_nothing_to_score(gpu):
    from cv3amd.qwen2 import DeviceQwen2
    lm, store = setup("per_channel")
    d = DeviceQwen2(store, cap=64)
    rng = np.random.default_rng(22)
    xs = prompts(rng, (16, 3))
    texts = [tokens(rng, 1, 1), tokens(rng, 1)]
    check(lm, xs, texts, d.score_batch(xs, texts, 2), 2)
    assert d.score_batch([], []) == [] and d.score_batch(xs, [[], []]) == [[], []]
    for part in d.score_batch(xs, [[[]], [[], np.zeros(0, np.int64)]], 3):
        assert all(g[0].size == 0 and g[2].shape == (0, 3) for g in part)
    same, = d.score_batch(xs[:1], [[texts[0][0]] * 3])           # the same continuation three times
    assert len({float(g[0][0]) for g in same}) == 1


def test_scores_of_a_search_are_its_sum(gpu):
    """What beam search and the greedy steps found is worth what they said."""
    from cv3amd.qwen2 import DeviceQwen2
    _, store = setup("per_channel")
    d = DeviceQwen2(store, cap=64)
    xs = prompts(np.random.default_rng(23), (19, 33, 4))
    for beams in (1, 3):
        found = d.generate_batch(xs, 7, min_len=7, beams=beams)
        scored = d.score_batch(xs, [[t] for t, _ in found], 1)
        for (t, total), ((lp, _, ids, _),) in zip(found, scored):
            assert len(t) == 7 and abs(lp.sum(dtype=np.float64) - total) <= 7 * NEAR
            if beams == 1:      # the likeliest of all but the stop ids, so of all where none of those is likelier
                assert all(i == a or i >= 6561 for i, a in zip(ids[:, 0], t))


def test_scores_in_parts(gpu, monkeypatch):
    """The limits of a call made small: four sequences and twenty rows at a time, cuts inside prompts and continuations,
    and more continuations of one prompt than one pass takes."""
    from cv3amd import qwen2
    lm, store = setup("per_channel")
    d = qwen2.DeviceQwen2(store, cap=64)
    rng = np.random.default_rng(24)
    xs = prompts(rng, (30, 1, 9, 45))
    texts = [tokens(rng, 5, 26, 2, 1, 44, 3, 7), tokens(rng, 4), tokens(rng, 1, 1, 1, 1), tokens(rng, 0, 9)]
    monkeypatch.setattr(qwen2, "_TABLE_ROWS", 4)
    monkeypatch.setattr(qwen2, "_PROMPT_ROWS", 20)
    check(lm, xs, texts, d.score_batch(xs, texts, 3, page=7), 3)


def test_scores_in_parts_of_so_many_keys(gpu, monkeypatch):
    """The keys of a pass bounded by small numbers: no cache is larger, but for a prompt with one continuation alone."""
    from cv3amd import paged, qwen2
    lm, store = setup("per_channel")
    d = qwen2.DeviceQwen2(store, cap=64)
    rng = np.random.default_rng(29)
    xs = prompts(rng, (30, 1, 9, 45))
    texts = [tokens(rng, 5, 26, 2, 1, 44, 3, 7), tokens(rng, 4), tokens(rng, 1, 1, 1, 1), tokens(rng, 0, 9)]
    made, new_cache = [], paged.new_cache
    monkeypatch.setattr(paged, "new_cache", lambda pages, *a, **k: made.append(pages) or new_cache(pages, *a, **k))
    for most in (1, 90, 140):
        monkeypatch.setattr(qwen2, "_SCORE_KEYS", most)
        check(lm, xs, texts, d.score_batch(xs, texts, 3, page=7), 3)
        alone = [-(-n // 7) + -(-(n + len(c) - 1) // 7) - n // 7 for n, cs in zip((30, 1, 9, 45), texts) for c in cs if c]
        assert max(made) * 7 <= max(most, 7 * max(alone)) and (most > 1 or sorted(made) == sorted(alone))
        made.clear()


@pytest.mark.parametrize("cache,eps", [("float16", 2.0 ** -11), ("bfloat16", 2.0 ** -8)])
def test_two_byte_caches(gpu, cache, eps):
    """Keys and values rounded once: half a step of their type each.  Two layers' outputs move by that share of values of
    at most about 1 each way, twice (a key's rounding through its weight, and a value's), and a log probability by twice
    what a logit does."""
    from cv3amd.qwen2 import DeviceQwen2
    lm, store = setup("per_channel")
    d = DeviceQwen2(store, cap=64)
    rng = np.random.default_rng(25)
    xs = prompts(rng, (37, 16))
    texts = [tokens(rng, 6, 12), tokens(rng, 20)]
    check(lm, xs, texts, d.score_batch(xs, texts, 2, cache=cache), 2, NEAR + 8 * eps)


def test_refusals(gpu):
    from cv3amd.qwen2 import DeviceQwen2
    _, store = setup("per_channel")
    d = DeviceQwen2(store, cap=64)
    x = prompts(np.random.default_rng(26), (3,))
    for bad in (dict(prompts=[np.zeros((3, 10))], continuations=[[[1]]]), dict(prompts=[np.zeros((0, 896))], continuations=[[[1]]]),
                dict(prompts=x, continuations=[]), dict(prompts=x, continuations=[[[1]], [[1]]]),
                dict(prompts=x, continuations=[[[-1]]]), dict(prompts=x, continuations=[[[6761]]]),
                dict(prompts=x, continuations=[[[0.5]]]), dict(prompts=x, continuations=[[[[1]]]]), dict(prompts=x, continuations=[[3]]),
                dict(prompts=x, continuations=[[[1]]], top=33), dict(prompts=x, continuations=[[[1]]], top=-1),
                dict(prompts=x, continuations=[[[1]]], page=0), dict(prompts=x, continuations=[[[1]]], page=65537),
                dict(prompts=x, continuations=[[[1]]], cache="int8")):
        with pytest.raises(ValueError):
            d.score_batch(**bad)


def test_the_objects_own_cache_is_left(gpu):
    from cv3amd.qwen2 import DeviceQwen2
    lm, store = setup("per_channel")
    d = DeviceQwen2(store, cap=64)
    rng = np.random.default_rng(27)
    xs = prompts(rng, (20, 7))
    d.prefill(xs[0], 0)
    d.score_batch(xs, [tokens(rng, 5), tokens(rng, 3, 3)], 1)
    assert d.generate_after_prefill(1, graph=False)[0] == int(logp(lm, xs[0], []).argmax())


def test_two_calls_at_once(gpu):
    """Two threads, each with its own stream, answer as a call alone."""
    import threading
    from cv3amd.qwen2 import DeviceQwen2
    _, store = setup("per_channel")
    d = DeviceQwen2(store, cap=64)
    rng = np.random.default_rng(28)
    xs = prompts(rng, (21, 8, 30))
    texts = [tokens(rng, 9, 2), tokens(rng, 17), tokens(rng, 1, 30)]
    got = [None, None]

    def one(i):
        got[i] = d.score_batch(xs, texts, 4)

    threads = [threading.Thread(target=one, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for want, a, b in zip(d.score_batch(xs, texts, 4), *got):
        for w, x, y in zip(want, a, b):
            assert all(np.array_equal(i, j) and np.array_equal(i, k) for i, j, k in zip(w, x, y))
