"""Performance cases of the paged-cache and beam-search operators (``cv3amd.paged``).

Five operators, as a program that serves several sequences from one set of weights calls them:

* ``tables``   ``paged.block_tables``: pages and slots for the new tokens of a batch of requests;
* ``append``   ``paged.append``: rotary on q and k, k and v into the paged cache;
* ``attend``   ``paged.attention``: one new token a sequence over the paged cache;
* ``select``   ``paged.beam_select``: the best continuations over beams and vocabulary;
* ``reorder``  ``paged.beam_reorder``: tables and part-filled pages follow the chosen beams.

Where ``own`` is false, ``run`` computes the same from elementary torch operations.
"""

import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cosyvoice3-cpu_amd")
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)

LAYERS = 24                                             # of the LM whose cache the beams share
GEOMETRIES = ((14, 2, 64), (16, 16, 64), (32, 8, 128), (20, 4, 80), (8, 1, 96))   # query heads, kv heads, head dim
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SPEECH_VOCAB, SPEECH_TOKENS = 6761, 6561                # the LM head's rows; ids from 6561 on stop a sentence


def listed():
    return [
        # one decode step of eight sentences: the smallest call, all latency
        dict(name="tables 8 steps", kind="tables", requests=8, new=1, held=900, page=16),
        # the prompts of a full serving batch at once, some with a cached beginning
        dict(name="tables 384 prompts", kind="tables", requests=384, new=1200, held=700, page=64),
        # one decode step of eight sentences through the LM's rotary and cache write
        dict(name="append 8 steps f32", kind="append", tokens=8, heads=14, kv_heads=2, dim=64, page=16, type="f32"),
        # several prompts side by side at a wide grouped geometry, bfloat16 cache
        dict(name="append 6001 tokens bf16", kind="append", tokens=6001, heads=32, kv_heads=8, dim=128, page=32,
             type="bf16"),
        # one sentence with its voice prompt: the LM's own decode attention
        dict(name="attend 1 x 500 f32", kind="attend", batch=1, length=500, ragged=False, window=0, heads=14,
             kv_heads=2, dim=64, page=16, type="f32"),
        # a serving batch of sentences at every stage, one row of it padding
        dict(name="attend 24 ragged f32", kind="attend", batch=24, length=1000, ragged=True, window=0, heads=14,
             kv_heads=2, dim=64, page=16, type="f32"),
        # three very long contexts: the work of few rows split over the cache's length
        dict(name="attend 3 x 100001 f16", kind="attend", batch=3, length=100001, ragged=False, window=0, heads=14,
             kv_heads=2, dim=64, page=64, type="f16"),
        # a large ragged batch at a wide grouped geometry, bfloat16 cache: the largest
        dict(name="attend 96 ragged bf16", kind="attend", batch=96, length=6000, ragged=True, window=0, heads=32,
             kv_heads=8, dim=128, page=32, type="bf16"),
        # one sentence searched with four beams over the speech vocabulary
        dict(name="select 1 x 4 of 6761", kind="select", requests=1, beams=4, vocab=SPEECH_VOCAB),
        # a batch of searches over a text-sized vocabulary
        dict(name="select 24 x 8 of 128000", kind="select", requests=24, beams=8, vocab=128000),
        # the four beams of one sentence, float32 cache of the whole LM
        dict(name="reorder 1 x 4 f32", kind="reorder", requests=1, beams=4, length=400, kv_heads=2, dim=64, page=16,
             type="f32"),
        # a batch of searches with larger pages
        dict(name="reorder 16 x 8 bf16", kind="reorder", requests=16, beams=8, length=500, kv_heads=2, dim=64,
             page=64, type="bf16"),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["tables", "append", "attend", "attend", "attend", "select", "reorder"])
    page = rng.choice([8, 16, 24, 32, 64, 100, 128])
    heads, kv_heads, dim = rng.choice(GEOMETRIES)
    type_ = rng.choice(list(TYPES))
    if kind == "tables":
        return dict(kind=kind, requests=log_int(1, 384), new=rng.choice([1, log_int(2, 1200)]),
                    held=log_int(1, 2000), page=page)
    if kind == "append":
        return dict(kind=kind, tokens=log_int(1, 6000), heads=heads, kv_heads=kv_heads, dim=dim, page=page, type=type_)
    if kind == "attend":
        batch = log_int(1, 128)
        room = 1.5e8 / (batch * kv_heads * dim)         # elements of the keys: no more than the largest listed case
        length = log_int(1, int(min(120000, max(2, room))))
        return dict(kind=kind, batch=batch, length=length, ragged=rng.random() < 0.6,
                    window=rng.choice([0, 0, 0, max(1, length // 3)]), heads=heads, kv_heads=kv_heads, dim=dim,
                    page=page, type=type_)
    if kind == "select":
        return dict(kind=kind, requests=log_int(1, 24), beams=rng.choice([2, 3, 4, 5, 8]), vocab=log_int(600, 128000))
    return dict(kind=kind, requests=log_int(1, 16), beams=rng.choice([2, 3, 4, 5, 8]), length=log_int(2, 500),
                kv_heads=rng.choice([1, 2, 4]), dim=rng.choice([64, 80]), page=rng.choice([8, 16, 24, 32, 64]),
                type=type_)


# ----------------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------------

class _Held:
    """A tensor of the program, and (``array``) the same memory as the framework's device array."""

    def __init__(self, tensor):
        self.tensor, self._array = tensor, None
        self.ptr, self.nbytes = tensor.data_ptr(), tensor.numel() * tensor.element_size()

    @property
    def array(self):
        if self._array is None:
            import numpy as np
            from cv3amd.device import DeviceArray
            kinds = {torch.float32: np.float32, torch.float16: np.float16, torch.bfloat16: np.uint16,
                     torch.int32: np.int32, torch.int64: np.int64, torch.uint8: np.uint8}
            self._array = DeviceArray(tuple(self.tensor.shape), kinds[self.tensor.dtype], block=self)
        return self._array


class _Inputs:
    """Seeded tensors on the GPU."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(int(seed))

    def normal(self, *shape, dtype=torch.float32, scale=1.0):
        # two-byte types are drawn by slices: a cache need not fit twice in float32
        if dtype == torch.float32:
            return torch.randn(shape, generator=self.gen, device="cuda") * scale
        out = torch.empty(shape, dtype=dtype, device="cuda")
        flat, step = out.reshape(-1), 1 << 26
        for i in range(0, flat.numel(), step):
            n = min(step, flat.numel() - i)
            flat[i:i + n] = torch.randn(n, generator=self.gen, device="cuda") * scale
        return out

    def ints(self, lo, hi, *shape, dtype=torch.int32):
        """Whole numbers of [lo, hi]."""
        return torch.randint(lo, hi + 1, shape, generator=self.gen, device="cuda").to(dtype)

    def order(self, n):
        return torch.randperm(n, generator=self.gen, device="cuda").to(torch.int32)


def _ceil(a, b):
    return -(-a // b)


def _lengths(case, draw):
    """Tokens of each sequence: up to ``length``; where a batch is ragged, every stage of it and one padding row."""
    b, top = case["batch"], case["length"]
    n = draw.ints(1, top, b) if case["ragged"] else draw.ints(max(1, top - 15), top, b)
    n[0] = top
    if case["ragged"] and b >= 8:
        n[b // 2] = 0
    return n


def _rotary(dim, positions):
    inv = 1.0 / (1e6 ** (torch.arange(0, dim, 2, dtype=torch.float64, device="cuda") / dim))
    ang = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * inv
    ang = torch.cat([ang, ang], dim=1)
    return ang.cos().float(), ang.sin().float()


def prepare(case, seed):
    draw, kind = _Inputs(seed), case["kind"]
    t = {}
    if kind == "tables":
        r, page = case["requests"], case["page"]
        held = draw.ints(0, case["held"], r)
        new = draw.ints(1, case["new"], r)
        blocks = _ceil(case["held"] + case["new"], page)
        pool = draw.order(2 * r * blocks)
        have = (held + page - 1) // page
        table = pool[:r * blocks].reshape(r, blocks).clone()
        table[torch.arange(blocks, device="cuda")[None] >= have[:, None]] = -1
        tokens = r * case["new"]
        t = dict(lengths=held, new=new, free=pool[r * blocks:].clone(), tables=table,
                 taken=torch.full((1,), 3, dtype=torch.int32, device="cuda"),
                 total=torch.empty_like(held), taken_out=torch.empty(1, dtype=torch.int32, device="cuda"),
                 starts=torch.empty(r + 1, dtype=torch.int32, device="cuda"),
                 slots=torch.empty(tokens, dtype=torch.int64, device="cuda"),
                 positions=torch.empty(tokens, dtype=torch.int32, device="cuda"))
    elif kind == "append":
        n, h, hk, d, page = (case[k] for k in ("tokens", "heads", "kv_heads", "dim", "page"))
        pages = 2 * _ceil(n, page)
        cos, sin = _rotary(d, 1024)
        t = dict(rows=draw.normal(n, (h + 2 * hk) * d), positions=draw.ints(0, 1023, n),
                 slots=draw.order(pages * page)[:n].to(torch.int64), cos=cos, sin=sin,
                 k=draw.normal(pages, hk, page, d, dtype=TYPES[case["type"]]),
                 v=draw.normal(pages, hk, page, d, dtype=TYPES[case["type"]]),
                 q=torch.empty(n, h, d, device="cuda"))
    elif kind == "attend":
        b, h, hk, d, page = (case[k] for k in ("batch", "heads", "kv_heads", "dim", "page"))
        n = _lengths(case, draw)
        blocks = _ceil(case["length"], page)
        used = (n + page - 1) // page
        first = torch.cumsum(used, 0) - used
        pages = int(used.sum())
        at = torch.arange(blocks, device="cuda")[None]
        table = torch.where(at < used[:, None], draw.order(pages)[(first[:, None] + at).clamp(max=pages - 1)],
                            torch.full((), -1, dtype=torch.int32, device="cuda"))
        t = dict(q=draw.normal(b, h, d, scale=1.5), k=draw.normal(pages, hk, page, d, dtype=TYPES[case["type"]]),
                 v=draw.normal(pages, hk, page, d, dtype=TYPES[case["type"]]), tables=table.contiguous(), lengths=n,
                 out=torch.empty(b, h, d, device="cuda"))
        if case["window"]:
            t["starts"] = (n - case["window"]).clamp(min=0)
    elif kind == "select":
        r, w, v = case["requests"], case["beams"], case["vocab"]
        scores = draw.normal(r, w, scale=2.0) - 20.0
        done = draw.ints(0, 9, r, w, dtype=torch.uint8) == 0        # a tenth of the beams have ended
        t = dict(logits=draw.normal(r, w, v, scale=2.5), scores=scores, done=done.to(torch.uint8),
                 tokens=torch.empty(r, w, dtype=torch.int64, device="cuda"),
                 parents=torch.empty(r, w, dtype=torch.int32, device="cuda"), scores_out=torch.empty_like(scores),
                 done_out=torch.empty(r, w, dtype=torch.uint8, device="cuda"))
    else:
        r, w, hk, d, page, top = (case[k] for k in ("requests", "beams", "kv_heads", "dim", "page", "length"))
        n = draw.ints(max(1, top - page + 1), top, r)
        blocks = _ceil(top, page)
        pages = r * w * blocks
        pages_of = draw.order(pages).reshape(r, w, blocks)
        full = (n // page)[:, None, None]
        back = draw.ints(0, w - 1, r, w, blocks, dtype=torch.int64)             # whole blocks lie with any beam
        table = torch.where(torch.arange(blocks, device="cuda") < full, pages_of.gather(1, back), pages_of)
        t = dict(parents=draw.ints(0, w - 1, r, w), tables=table.contiguous(), pages=pages_of, lengths=n,
                 k=draw.normal(LAYERS, pages, hk, page, d, dtype=TYPES[case["type"]]),
                 v=draw.normal(LAYERS, pages, hk, page, d, dtype=TYPES[case["type"]]))
    return {"case": case, **{k: _Held(v) for k, v in t.items()}}


# ----------------------------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------------------------

def _stop(case):
    """(first, end) of the ids that end a hypothesis."""
    return (SPEECH_TOKENS, SPEECH_VOCAB) if case["vocab"] == SPEECH_VOCAB else (2, 3)


def _calls(s):
    from cv3amd import paged
    case, kind = s["case"], s["case"]["kind"]
    a = {k: v.array for k, v in s.items() if k != "case"}
    if kind == "tables":
        paged.block_tables(a["lengths"], a["new"], case["page"], a["free"], a["taken"], a["tables"],
                           out=(a["total"], a["taken_out"], a["starts"], a["slots"], a["positions"]))
        return [s[k].tensor for k in ("tables", "total", "taken_out", "starts", "slots", "positions")]
    if kind == "append":
        paged.append(a["rows"], case["heads"], a["positions"], a["slots"], a["cos"], a["sin"], a["k"], a["v"],
                     out=a["q"])
        return [s[k].tensor for k in ("q", "k", "v")]
    if kind == "attend":
        paged.attention(a["q"], a["k"], a["v"], a["tables"], a["lengths"], starts=a.get("starts"), out=a["out"])
        return s["out"].tensor
    if kind == "select":
        paged.beam_select(a["logits"], a["scores"], a["done"], stop=_stop(case),
                          out=(a["tokens"], a["parents"], a["scores_out"], a["done_out"]))
        return [s[k].tensor for k in ("tokens", "parents", "scores_out", "done_out")]
    paged.beam_reorder(a["parents"], a["tables"], a["pages"], a["lengths"], a["k"], a["v"])
    return [s[k].tensor for k in ("tables", "k", "v")]


def _plain_tables(t, page):
    held, table = t["lengths"].long(), t["tables"]
    r, blocks = table.shape
    tokens, at = t["slots"].shape[0], torch.arange(blocks, device=table.device)
    want = torch.minimum(t["new"].long(), blocks * page - held).clamp(min=0)
    ends = torch.cumsum(want, 0).clamp(max=tokens)
    starts = torch.cat([ends.new_zeros(1), ends])
    total = held + (ends - starts[:-1])
    have = (held + page - 1) // page
    need = (total + page - 1) // page - have
    first = t["taken"].long() + torch.cumsum(need, 0) - need
    index = first[:, None] + at - have[:, None]
    fresh = (at >= have[:, None]) & (at < (have + need)[:, None])
    ids = torch.where(index < t["free"].shape[0], t["free"][index.clamp(0, t["free"].shape[0] - 1)], -1)
    table.copy_(torch.where(fresh, ids, table))
    i = torch.arange(tokens, device=table.device)
    row = torch.searchsorted(ends, i, right=True).clamp(max=r - 1)
    pos = held[row] + i - starts[row]
    given = i < ends[-1]
    of = table[row, (pos // page).clamp(0, blocks - 1)].long()
    slots = torch.where(given & (of >= 0), of * page + pos % page, -1)
    taken = (t["taken"].long() + need.sum()).int()
    return [table, total.int(), taken, starts.int(), slots, torch.where(given, pos, -1).int()]


def _turn(x, cos, sin):
    half = x.shape[-1] // 2
    return x * cos + torch.cat([-x[..., half:], x[..., :half]], dim=-1) * sin


def _plain_append(t, heads):
    kc, vc = t["k"], t["v"]
    _, hk, page, d = kc.shape
    rows = t["rows"].reshape(t["rows"].shape[0], heads + 2 * hk, d)
    cos, sin = (t[k][t["positions"]][:, None] for k in ("cos", "sin"))
    at, off = t["slots"] // page, t["slots"] % page
    kc[at, :, off] = _turn(rows[:, heads:heads + hk], cos, sin).to(kc.dtype)
    vc[at, :, off] = rows[:, heads + hk:].to(vc.dtype)
    return [_turn(rows[:, :heads], cos, sin), kc, vc]


def _plain_attention(t):
    q, table, n = t["q"], t["tables"].clamp(min=0), t["lengths"]
    b, h, d = q.shape
    _, hk, page, _ = t["k"].shape
    keys = table.shape[1] * page
    k, v = (t[x][table].float().transpose(1, 2).reshape(b, hk, keys, d) for x in "kv")
    at = torch.arange(keys, device=q.device)
    seen = at < n[:, None]
    if "starts" in t:
        seen = seen & (at >= t["starts"][:, None])
    s = torch.matmul(q.reshape(b, hk, h // hk, d) / math.sqrt(d), k.transpose(2, 3).contiguous())
    s = torch.where(seen[:, None, None], s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top > -math.inf, top, 0.0))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    return o.reshape(b, h, d)


def _plain_select(t, stop):
    """In 64 bits: neighbouring candidates may lie closer than 32 bits tell apart."""
    x, scores, done = t["logits"], t["scores"].double(), t["done"].bool()
    r, w, v = x.shape
    bits = x.view(torch.int32).long()
    order = torch.where(bits < 0, -(bits & 0x7fffffff), bits)               # rises with the logit; -0.0 as 0.0
    best = (order * (1 << 20) + (v - 1 - torch.arange(v, device=x.device))).topk(w, dim=-1).values
    token = v - 1 - (best & ((1 << 20) - 1))
    x64 = x.double()
    top = x64.amax(-1, keepdim=True)
    lse = top + torch.exp(x64 - top).sum(-1, keepdim=True).log()
    value = scores[..., None] + (x64.gather(2, token) - lse)
    rank = torch.arange(w, device=x.device)
    value = torch.where(done[..., None], torch.where(rank == 0, scores[..., None], -math.inf), value)
    token = torch.where(done[..., None], stop[0], token)
    value, at = torch.sort(value.reshape(r, w * w), dim=1, descending=True, stable=True)
    at = at[:, :w]
    token, parent = token.reshape(r, w * w).gather(1, at), at // w
    ended = done.gather(1, parent) | ((token >= stop[0]) & (token < stop[1]))
    return [token, parent.int(), value[:, :w].float(), ended.to(torch.uint8)]


def _plain_reorder(t):
    kc, vc, table, pages, n = t["k"], t["v"], t["tables"], t["pages"], t["lengths"].long()
    r, w, blocks = table.shape
    page = kc.shape[3]
    parent = t["parents"].long()
    full, rest = n // page, n % page
    up = parent[..., None].expand(r, w, blocks)
    table.copy_(torch.where(torch.arange(blocks, device=table.device) < full[:, None, None], table.gather(1, up),
                            pages))
    own_page = pages.gather(2, full.clamp(max=blocks - 1)[:, None, None].expand(r, w, 1))[..., 0].long()
    source = own_page.gather(1, parent).reshape(-1)
    own_page = own_page.reshape(-1)
    moved = torch.arange(page, device=table.device)[None] < rest.repeat_interleave(w)[:, None]
    moved = moved[None, :, None, :, None]
    for c in (kc, vc):
        c[:, own_page] = torch.where(moved, c[:, source], c[:, own_page])
    return [table, kc, vc]


def run(s):
    if own:
        return _calls(s)
    case, kind = s["case"], s["case"]["kind"]
    t = {k: v.tensor for k, v in s.items() if k != "case"}
    if kind == "tables":
        return _plain_tables(t, case["page"])
    if kind == "append":
        return _plain_append(t, case["heads"])
    if kind == "attend":
        return _plain_attention(t)
    if kind == "select":
        return _plain_select(t, _stop(case))
    return _plain_reorder(t)


# ----------------------------------------------------------------------------------------------
# what a pass cannot do without
# ----------------------------------------------------------------------------------------------

def work(case):
    """Where sizes come from the seed, their mean."""
    kind = case["kind"]
    size = {"f32": 4, "f16": 2, "bf16": 2}.get(case.get("type"), 4)
    if kind == "tables":
        r, new = case["requests"], (case["new"] + 1) / 2
        pages = r * max(1.0 / case["page"], new / case["page"])
        # lengths, counts, a page in use; ids out and in; starts and totals; slots and positions (all of them listed)
        return {"bytes": r * 12 + pages * 8 + r * 8 + r * case["new"] * 12, "flops": 0}
    if kind == "append":
        n, h, hk, d = (case[k] for k in ("tokens", "heads", "kv_heads", "dim"))
        return {"bytes": n * ((2 * h + 2 * hk) * d * 4 + 2 * hk * d * size + 12) + min(n, 1024) * d * 8,
                "flops": 3.0 * n * (h + hk) * d}
    if kind == "attend":
        b, h, hk, d, top = (case[k] for k in ("batch", "heads", "kv_heads", "dim", "length"))
        mean = (top + 1) / 2 if case["ragged"] else top - min(15, top - 1) / 2
        if case["window"]:
            w = min(case["window"], top)
            mean = (w * (w + 1) / 2 + (top - w) * w) / top if case["ragged"] else w
        rows = b - 1 if case["ragged"] and b >= 8 else b
        keys = top if b == 1 and not case["window"] else rows * mean
        return {"bytes": keys * 2 * hk * d * size + keys / case["page"] * 4 + 8.0 * b * h * d + 4.0 * b,
                "flops": 4.0 * keys * h * d}
    if kind == "select":
        rows = case["requests"] * case["beams"]
        return {"bytes": rows * (4.0 * case["vocab"] + 4 + 1 + 8 + 4 + 4 + 1), "flops": 3.0 * rows * case["vocab"]}
    r, w, page = case["requests"], case["beams"], case["page"]
    moved = r * (w - 1) * (min(page, case["length"]) - 1) / 2           # rows of beams that follow another one
    return {"bytes": moved * 2 * 2 * LAYERS * case["kv_heads"] * case["dim"] * size
            + 8.0 * r * w * _ceil(case["length"], page) + 4.0 * r * (w + 1), "flops": 0}


# ----------------------------------------------------------------------------------------------
# the same results in 64 bits, from the definitions
# ----------------------------------------------------------------------------------------------

def _exact_append(case, t):
    h, hk, d, page = (case[k] for k in ("heads", "kv_heads", "dim", "page"))
    n, half = case["tokens"], d // 2
    rows = t["rows"].double().view(n, h + 2 * hk, d)
    turned = rows.clone()
    for lo, a, b, sign in ((0, 0, half, -1.0), (half, half, 0, 1.0)):
        c, s = (t[x].double()[t["positions"].long(), lo:lo + half].unsqueeze(1) for x in ("cos", "sin"))
        turned[:, :, lo:lo + half] = rows[:, :, a:a + half] * c + sign * rows[:, :, b:b + half] * s
    k, v = (t[x].double().transpose(1, 2).contiguous().view(-1, hk, d) for x in "kv")     # a row a slot
    k[t["slots"]] = turned[:, h:h + hk]
    v[t["slots"]] = rows[:, h + hk:]
    return [turned[:, :h]] + [x.view(-1, page, hk, d).transpose(1, 2).contiguous() for x in (k, v)]


def _exact_attention(case, t):
    h, hk, d = (case[k] for k in ("heads", "kv_heads", "dim"))
    out = torch.zeros(case["batch"], h, d, dtype=torch.float64, device="cuda")
    lengths = t["lengths"].tolist()
    starts = t["starts"].tolist() if "starts" in t else [0] * len(lengths)
    for b, (lo, hi) in enumerate(zip(starts, lengths)):
        if hi <= lo:
            continue
        ids = t["tables"][b, :_ceil(hi, case["page"])].long()
        for j in range(hk):
            k, v = (t[x][ids, j].double().reshape(-1, d)[lo:hi] for x in "kv")
            for i in range(j * (h // hk), (j + 1) * (h // hk)):
                s = (k * t["q"][b, i].double()).sum(1) / math.sqrt(d)
                e = torch.exp(s - s.max())
                out[b, i] = (e[:, None] * v).sum(0) / e.sum()
    return out


def _exact_select(case, t):
    """The chosen scores alone: what is whole has no nearer value."""
    stop, r, w = _stop(case), case["requests"], case["beams"]
    got = torch.empty(r, w, dtype=torch.float64, device="cuda")
    for i in range(r):
        every = []
        for b in range(w):
            score = t["scores"][i, b].double()
            if int(t["done"][i, b]):
                every.append(score.reshape(1))
            else:
                x = t["logits"][i, b].double()
                every.append(score + torch.log_softmax(x, 0).sort(descending=True).values[:w])
        got[i] = torch.cat(every).sort(descending=True).values[:w]
    return [None, None, got, None]


def _exact_reorder(case, t):
    n, page, w = t["lengths"].tolist(), case["page"], case["beams"]
    parents, pages = t["parents"].tolist(), t["pages"].tolist()
    done = []
    for c in (t["k"], t["v"]):
        new = c.clone()
        for i, length in enumerate(n):
            at, rest = divmod(length, page)
            if rest:
                for j in range(w):
                    new[:, pages[i][j][at], :, :rest] = c[:, pages[i][parents[i][j]][at], :, :rest]
        done.append(new)        # moved, not computed: the values of the cache's own type are exact
    return [None] + done


def exact(case, seed):
    kind = case["kind"]
    if kind == "tables":
        return None
    t = {k: v.tensor for k, v in prepare(case, seed).items() if k != "case"}
    if kind == "append":
        return _exact_append(case, t)
    if kind == "attend":
        return _exact_attention(case, t)
    return _exact_select(case, t) if kind == "select" else _exact_reorder(case, t)
