"""DeviceQwen2.generate_batch: several prompts from one set of weights, greedy and by beam search, over the paged cache,
against the oracle's LM run one sequence at a time (Qwen2-0.5B's geometry, two layers, synthetic weights)."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

SIZE = 6561     # ids from here on stop


def setup(profile):
    import oracle.quant
    import cv3amd.quant
    from cv3amd import synth
    from cv3amd.weights import WeightStore
    from oracle.llm import CosyVoice3LM
    t = synth.quantize_store(synth.qwen2_tensors(layers=2), profile, oracle.quant.quantize_q8, oracle.quant.quantize_q4)
    meta = synth.qwen2_meta(layers=2)
    return (CosyVoice3LM(WeightStore(t, meta, oracle.quant.QTensor), "llm."),
            WeightStore(t, meta, cv3amd.quant.QTensor))


def prompts(rng, lengths):
    return [(rng.standard_normal((n, 896)) * 0.02).astype(np.float32) for n in lengths]


def logp(lm, prompt, tokens):
    """Log probabilities (float64) of the next token after a prompt and its tokens."""
    x = prompt if not tokens else np.concatenate([prompt, lm.speech_emb(tokens)])
    z = lm.head(lm.body.forward(x, lm.body.new_cache())[-1:])[0].astype(np.float64)
    return z - z.max() - np.log(np.exp(z - z.max()).sum())


def search(lm, prompt, beams, max_len, min_len, size):
    """Plain beam search: (score, tokens, ended) hypotheses, best first; ties are not met."""
    live = [(0.0, [], False)]
    for i in range(max_len):
        every = []
        for score, tokens, ended in live:
            if ended:
                every.append((score, tokens, True))
                continue
            p = logp(lm, prompt, tokens)
            if i < min_len:
                p[size:size + 200] = -np.inf
            for t in np.argsort(-p, kind="stable")[:beams]:
                every.append((score + p[t], tokens + [int(t)], size <= t < size + 200))
        live = sorted(every, key=lambda c: -c[0])[:beams]
        if all(e for _, _, e in live):
            break
    score, tokens, _ = live[0]
    return [t for t in tokens if not size <= t < size + 200], score


@pytest.mark.parametrize("profile,page", [("per_channel", 16), ("balanced", 5), ("tiny", 64)])
def test_greedy_batch_is_the_oracles_sequences(gpu, profile, page):
    from cv3amd.qwen2 import DeviceQwen2
    lm, store = setup(profile)
    d = DeviceQwen2(store, cap=64)
    xs = prompts(np.random.default_rng(1), (37, 1, 16, 50, 5, 64))
    got = d.generate_batch(xs, 8, min_len=8, page=page)
    for x, (tokens, score) in zip(xs, got):
        seen, total = [], 0.0
        for _ in range(8):
            p = logp(lm, x, seen)
            total += p[:SIZE].max()
            seen.append(int(p[:SIZE].argmax()))
        assert tokens == seen
        assert abs(score - total) <= 1e-4     # eight log probabilities from logits within 1e-5 of about 1
    # the same object's own cache and the single-sequence path are as before
    d.prefill(xs[0], 0)
    assert d.generate_after_prefill(1, graph=False)[0] == int(logp(lm, xs[0], []).argmax())


def test_prompts_longer_than_the_single_sequences_cache(gpu):
    from cv3amd.device import to_device
    from cv3amd.qwen2 import DeviceQwen2
    lm, store = setup("per_channel")
    d = DeviceQwen2(store, cap=64, prompt_planes=False)
    xs = prompts(np.random.default_rng(6), (1100, 3))
    for x, (tokens, _) in zip(xs, d.generate_batch([to_device(xs[0]), xs[1].astype(np.float64)], 2, min_len=2, page=64)):
        first = int(logp(lm, x, [])[:SIZE].argmax())
        assert tokens == [first, int(logp(lm, x, [first])[:SIZE].argmax())]


def test_beam_search_is_the_plain_one(gpu):
    from cv3amd.qwen2 import DeviceQwen2
    lm, store = setup("per_channel")
    d = DeviceQwen2(store, cap=64)
    xs = prompts(np.random.default_rng(2), (19, 33, 4))
    for beams, page in ((3, 16), (5, 4)):
        for x, (tokens, score) in zip(xs, d.generate_batch(xs, 6, min_len=2, beams=beams, page=page)):
            want, total = search(lm, x, beams, 6, 2, SIZE)
            assert tokens == want
            assert abs(score - total) <= 1e-4


def test_beams_end_at_their_stop(gpu):
    """A wide range of stop ids, so that hypotheses end at different lengths while others go on."""
    from cv3amd.qwen2 import DeviceQwen2
    lm, store = setup("per_channel")
    d = DeviceQwen2(store, cap=64)
    xs = prompts(np.random.default_rng(3), (12, 7))
    first = [int(logp(lm, x, []).argmax()) for x in xs]
    size = max(1, min(first) - 100)           # the likeliest first token of one prompt lies among the stop ids
    for min_len in (0, 1, 3):
        for x, (tokens, score) in zip(xs, d.generate_batch(xs, 5, min_len=min_len, speech_token_size=size, beams=4)):
            want, total = search(lm, x, 4, 5, min_len, size)
            assert tokens == want
            assert abs(score - total) <= 1e-4


@pytest.mark.parametrize("cache", ["float16", "bfloat16"])
def test_two_byte_caches(gpu, cache):
    """Scores of the tokens that were chosen: keys and values off by half a step of their type (2^-11, 2^-8) move a
    score q.k by that share of sum |q k|, and through two layers the log probabilities by less than ten such shares."""
    from cv3amd.qwen2 import DeviceQwen2
    lm, store = setup("per_channel")
    d = DeviceQwen2(store, cap=64)
    xs = prompts(np.random.default_rng(4), (40, 9))
    for x, (tokens, score) in zip(xs, d.generate_batch(xs, 5, min_len=5, beams=2, cache=cache)):
        total = sum(logp(lm, x, tokens[:i])[t] for i, t in enumerate(tokens))
        assert len(tokens) == 5 and abs(score - total) <= 5 * 10 * (2.0 ** -11 if cache == "float16" else 2.0 ** -8)


def test_two_calls_at_once(gpu, monkeypatch):
    """Two threads, each with its own stream: the weights' layout that the first call makes is whole before the other
    reads it, and both answer as a call alone."""
    import threading
    from cv3amd import qwen2
    _, store = setup("per_channel")
    d = qwen2.DeviceQwen2(store, cap=64)
    xs = prompts(np.random.default_rng(7), (21, 8, 30))
    order, wait, pack = [], qwen2.synchronize, qwen2._Stacked.planes

    def packing(self, *args):
        order.append(("pack", d._batch is None))
        return pack(self, *args)

    def waiting():
        order.append(("wait", d._batch is None))
        wait()

    monkeypatch.setattr(qwen2._Stacked, "planes", packing)
    monkeypatch.setattr(qwen2, "synchronize", waiting)
    got = [None, None]

    def one(i):
        got[i] = d.generate_batch(xs, 6, min_len=6, beams=2)

    threads = [threading.Thread(target=one, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    # packed once, waited for, and seen by nobody before
    assert [n for n, _ in order] == ["pack"] * (len(order) - 1) + ["wait"] and all(unseen for _, unseen in order)
    assert got[0] == got[1] == d.generate_batch(xs, 6, min_len=6, beams=2)


def test_refusals(gpu):
    from cv3amd.qwen2 import DeviceQwen2
    _, store = setup("per_channel")
    d = DeviceQwen2(store, cap=64)
    x = prompts(np.random.default_rng(5), (3,))
    assert d.generate_batch([], 5) == []
    for bad in (dict(prompts=[np.zeros((3, 10))], max_len=2), dict(prompts=[np.zeros((0, 896))], max_len=2),
                dict(prompts=x, max_len=0), dict(prompts=x, max_len=2, beams=17), dict(prompts=x, max_len=2, beams=0),
                dict(prompts=x, max_len=2, cache="int8"), dict(prompts=x, max_len=2, page=0),
                dict(prompts=x, max_len=2, speech_token_size=7000)):
        with pytest.raises(ValueError):
            d.generate_batch(**bad)


def greedy(lm, x, steps):
    seen = []
    for _ in range(steps):
        seen.append(int(logp(lm, x, seen)[:SIZE].argmax()))
    return seen


def test_more_prompts_than_one_call_of_the_tables(gpu):
    """4100 sequences: each step's slots are listed 4096 requests at a time."""
    from cv3amd.qwen2 import DeviceQwen2
    lm, store = setup("per_channel")
    d = DeviceQwen2(store, cap=64)
    few = prompts(np.random.default_rng(10), (1, 3, 2, 1))
    xs = [few[0]] * 4095 + few + [few[0]]
    got = d.generate_batch(xs, 3, min_len=3, page=2)
    for at in (0, 4094, 4095, 4096, 4097, 4098, 4099):
        assert got[at][0] == greedy(lm, xs[at], 3)
    got = d.generate_batch([few[1]] * 300, 3, min_len=3, beams=14)      # 4200 sequences of 300 prompts
    want, total = search(lm, few[1], 14, 3, 3, SIZE)
    for tokens, score in (got[0], got[292], got[293], got[299]):
        assert tokens == want and abs(score - total) <= 1e-4


def test_batches_in_parts(gpu, monkeypatch):
    """The limits of a call made small: slots of four requests and prompts of twenty tokens at a time, cuts inside a
    prompt and between two."""
    from cv3amd import qwen2
    _, store = setup("per_channel")
    d = qwen2.DeviceQwen2(store, cap=64)
    xs = prompts(np.random.default_rng(11), (30, 1, 9, 20, 45, 2))
    want = [d.generate_batch(xs, 5, min_len=5, beams=b, page=7) for b in (1, 3)]
    monkeypatch.setattr(qwen2, "_TABLE_ROWS", 4)
    monkeypatch.setattr(qwen2, "_PROMPT_ROWS", 20)
    for b, w in zip((1, 3), want):
        for (tokens, score), (expected, total) in zip(d.generate_batch(xs, 5, min_len=5, beams=b, page=7), w):
            assert tokens == expected and abs(score - total) <= 1e-4


def test_refused_before_any_work(gpu, monkeypatch):
    """What a step would refuse is refused before memory is taken and a prompt is run."""
    from cv3amd import paged
    from cv3amd.qwen2 import DeviceQwen2
    _, store = setup("per_channel")
    d = DeviceQwen2(store, cap=64)
    monkeypatch.setattr(paged, "new_cache", None)       # reached: TypeError
    x, = prompts(np.random.default_rng(14), (2,))
    for bad in (dict(prompts=[x], max_len=2, page=65537), dict(prompts=[x] * 600000, max_len=2),
                dict(prompts=[x] * 40000, max_len=2, beams=16)):
        with pytest.raises(ValueError):
            d.generate_batch(**bad)
    monkeypatch.setattr(d, "vocab", 205)                # ids 10 .. 204 stop: ten to choose from while they are banned
    with pytest.raises(ValueError, match="fewer tokens"):
        d.generate_batch([x], 2, min_len=1, beams=11, speech_token_size=10)
    monkeypatch.setattr(d, "vocab", 10)
    with pytest.raises(ValueError, match="fewer tokens"):
        d.generate_batch([x], 2, beams=11, speech_token_size=9)


def test_pages_that_are_reserved(gpu, monkeypatch):
    """A prompt's whole pages once for its beams, and each beam's own from there to its last token: no more."""
    from cv3amd import paged
    from cv3amd.qwen2 import DeviceQwen2
    _, store = setup("per_channel")
    d = DeviceQwen2(store, cap=64)
    made, new_cache = [], paged.new_cache
    monkeypatch.setattr(paged, "new_cache", lambda pages, *a, **k: made.append(pages) or new_cache(pages, *a, **k))
    lengths = (160, 3, 32, 47)
    for beams, max_len in ((1, 6), (4, 6), (4, 1)):
        d.generate_batch(prompts(np.random.default_rng(12), lengths), max_len, min_len=max_len, beams=beams, page=16)
        assert made.pop() == sum(n // 16 + beams * (-(-(n + max_len - 1) // 16) - n // 16) for n in lengths)


def test_weights_that_fail_to_be_packed(gpu, monkeypatch):
    """Without memory the decode's weights serve; any other failure is the caller's to see, and the next call packs."""
    from cv3amd import _lib, qwen2
    from cv3amd.device import DeviceArray
    _, store = setup("per_channel")
    d = qwen2.DeviceQwen2(store, cap=64, prompt_planes=False)
    xs = prompts(np.random.default_rng(13), (5, 8))
    real = _lib.call

    def call(name, *args):
        if name == "pack_code_planes":
            raise _lib.HIPError("kernel launch failed")
        return real(name, *args)

    with monkeypatch.context() as m:
        m.setattr(_lib, "call", call)
        with pytest.raises(_lib.HIPError, match="launch failed"):
            d.generate_batch(xs, 4, min_len=4)
    want = d.generate_batch(xs, 4, min_len=4)
    codes = 1152 * 896 + 896 * 896 + 9728 * 896 + 896 * 4864
    assert d._batch and d.batch_nbytes == 2 * (2 * codes + 4 * (1152 + 896 + 9728 + 896))     # two layers
    full = qwen2.DeviceQwen2(store, cap=64)
    held = full.prompt_nbytes
    assert full.batch_nbytes == 0
    full.generate_batch(xs, 2)
    assert full.prompt_nbytes == held        # o and down are the prompt's
    assert full.batch_nbytes == 2 * (2 * (1152 + 9728) * 896 + 4 * (1152 + 9728))

    class NoMemory(DeviceArray):
        def __init__(self, shape, dtype=np.float32, *a, **k):
            if np.dtype(dtype) == np.uint16:
                raise _lib.HIPError("hipMalloc failed")
            super().__init__(shape, dtype, *a, **k)

    bare = qwen2.DeviceQwen2(store, cap=64, prompt_planes=False)
    with monkeypatch.context() as m:
        m.setattr(qwen2, "DeviceArray", NoMemory)
        got = bare.generate_batch(xs, 4, min_len=4)
    assert bare._batch == {} and bare.batch_nbytes == 0
    assert [t for t, _ in got] == [t for t, _ in want] == [t for t, _ in bare.generate_batch(xs, 4, min_len=4)]


@pytest.mark.parametrize("profile", ["per_channel", "balanced", "tiny"])
def test_one_prompt_alone(gpu, profile):
    """One greedy prompt: a row a step, on the decode's own weights; also one of a single token."""
    from cv3amd.qwen2 import DeviceQwen2
    lm, store = setup(profile)
    d = DeviceQwen2(store, cap=64)
    for x in prompts(np.random.default_rng(8), (23, 1)):
        (tokens, _), = d.generate_batch([x], 6, min_len=6)
        assert tokens == greedy(lm, x, 6)
    assert d.generate_batch([x], 1, min_len=1)[0][0] == greedy(lm, x, 1)


@pytest.mark.parametrize("profile", ["per_channel", "balanced", "tiny"])
def test_without_the_code_planes(gpu, profile):
    """Several prompts on the decode's own weights, as where the planes find no memory: the planes' tokens."""
    from cv3amd.qwen2 import DeviceQwen2
    lm, store = setup(profile)
    d = DeviceQwen2(store, cap=64)
    xs = prompts(np.random.default_rng(9), (30, 1, 9))
    want = [d.generate_batch(xs, 6, min_len=6, beams=b) for b in (1, 3)]
    assert d._batch
    bare = DeviceQwen2(store, cap=64, prompt_planes=False)
    bare._batch = {}
    for b, w in zip((1, 3), want):
        for (tokens, score), (expected, total) in zip(bare.generate_batch(xs, 6, min_len=6, beams=b), w):
            assert tokens == expected and abs(score - total) <= 1e-4
    assert [t for t, _ in want[0]] == [greedy(lm, x, 6) for x in xs]
