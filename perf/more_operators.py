"""Performance cases of the operators that serve and score changing sets of sequences (``cv3amd.paged``).

Five operators, as a scheduler over the paged cache calls them:

* ``extend``   ``paged.extend``: attention of a chunk of new tokens a sequence over the paged cache;
* ``score``    ``paged.token_logprobs``: log probabilities of given tokens, entropy, best alternatives;
* ``fork``     ``paged.fork``: sequences that go on from others, whole pages shared;
* ``free``     ``paged.free_pages``: the pages that no sequence holds any more;
* ``compact``  ``paged.compact``: the pages that are held, into another cache.

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

LAYERS = 24                                             # of the LM whose cache is forked and compacted
GEOMETRIES = ((14, 2, 64), (16, 16, 64), (32, 8, 128), (20, 4, 80), (8, 1, 96))   # query heads, kv heads, head dim
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SPEECH_VOCAB = 6761                                     # the LM head's rows


def listed():
    return [
        # four drafted tokens of one sentence, checked in one pass: the smallest attention, all latency
        dict(name="extend 1 x 4 over 500 f32", kind="extend", batch=1, chunk=4, held=500, ragged=False, window=0,
             heads=14, kv_heads=2, dim=64, page=16, type="f32"),
        # the prompts of a batch of sentences: voice prompt and text, nothing cached before
        dict(name="extend 12 prompts f32", kind="extend", batch=12, chunk=900, held=0, ragged=True, window=0,
             heads=14, kv_heads=2, dim=64, page=16, type="f32"),
        # a slice of a very long prompt: few rows over a long cache
        dict(name="extend 1 x 500 over 60001 f16", kind="extend", batch=1, chunk=500, held=60001, ragged=False,
             window=0, heads=14, kv_heads=2, dim=64, page=64, type="f16"),
        # prompts in slices at a wide grouped geometry, every stage of them, bfloat16 cache: the largest
        dict(name="extend 12 ragged bf16", kind="extend", batch=12, chunk=800, held=5000, ragged=True, window=0,
             heads=32, kv_heads=8, dim=128, page=32, type="bf16"),
        # the next tokens of a few sentences with their alternatives
        dict(name="score 6 of 6761", kind="score", rows=6, vocab=SPEECH_VOCAB, top=5),
        # whole texts scored over a text-sized vocabulary
        dict(name="score 500 of 128000", kind="score", rows=500, vocab=128000, top=8),
        # three more candidates for one sentence, float32 cache of the whole LM
        dict(name="fork 1 by 3 f32", kind="fork", parents=1, each=3, length=400, kv_heads=2, dim=64, page=16,
             type="f32"),
        # candidates for a batch of sentences with larger pages
        dict(name="fork 16 by 7 bf16", kind="fork", parents=16, each=7, length=500, kv_heads=2, dim=64, page=64,
             type="bf16"),
        # a few sentences, one of which has ended
        dict(name="free of 8", kind="free", batch=8, length=900, page=16),
        # a full serving batch, a part of it ended, beginnings shared
        dict(name="free of 384", kind="free", batch=384, length=1900, page=16),
        # what is left of a small cache
        dict(name="compact 4 f32", kind="compact", batch=4, length=300, kv_heads=2, dim=64, page=16, type="f32"),
        # what is left of a serving batch, into a cache of its size
        dict(name="compact 48 bf16", kind="compact", batch=48, length=900, kv_heads=2, dim=64, page=32, type="bf16"),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["extend", "extend", "extend", "score", "score", "fork", "free", "compact"])
    page = rng.choice([8, 16, 24, 32, 64, 100, 128])
    heads, kv_heads, dim = rng.choice(GEOMETRIES)
    type_ = rng.choice(list(TYPES))
    if kind == "extend":
        batch, chunk = log_int(1, 24), log_int(1, 1500)
        # scores of a padded batch, and products: no more than the largest listed case has
        keys = min(5e8 / (batch * chunk * heads), 4e10 / (batch * chunk * heads * dim), 1e8 / (batch * kv_heads * dim), 60000)
        chunk = int(min(chunk, max(1, math.sqrt(keys * chunk))))
        held = rng.choice([0, log_int(1, int(max(1, keys - chunk)))]) if keys > chunk + 1 else 0
        return dict(kind=kind, batch=batch, chunk=chunk, held=held, ragged=rng.random() < 0.6,
                    window=rng.choice([0, 0, 0, max(1, (chunk + held) // 3)]), heads=heads, kv_heads=kv_heads, dim=dim,
                    page=page, type=type_)
    if kind == "score":
        vocab = log_int(300, 128000)
        return dict(kind=kind, rows=log_int(1, int(min(8000, 6.4e7 / vocab))), vocab=vocab,
                    top=rng.choice([0, 1, 5, 8, 16]))
    if kind == "fork":
        return dict(kind=kind, parents=log_int(1, 12), each=rng.choice([1, 2, 3, 4, 7]), length=log_int(2, 500),
                    kv_heads=rng.choice([1, 2]), dim=rng.choice([64, 80]), page=rng.choice([8, 16, 24, 32]), type=type_)
    if kind == "free":
        return dict(kind=kind, batch=log_int(1, 384), length=log_int(1, 1900), page=page)
    batch = log_int(1, 48)
    return dict(kind=kind, batch=batch, length=log_int(2, int(min(900, 20000 / batch))), kv_heads=rng.choice([1, 2]),
                dim=rng.choice([64, 80]), page=rng.choice([8, 16, 24, 32, 64]), type=type_)


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
                     torch.int32: np.int32, torch.int64: np.int64}
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

    def stages(self, hi, n):
        """Whole numbers spread evenly over [0, hi], in any order but for the first, which is hi: their sum is the same
        for every seed."""
        at = torch.arange(n, device="cuda") * hi // n
        at = at[torch.randperm(n - 1, generator=self.gen, device="cuda") + 1] if n > 1 else at[:0]
        return torch.cat([torch.full((1,), hi, device="cuda"), at]).to(torch.int32)

    def order(self, n):
        return torch.randperm(n, generator=self.gen, device="cuda").to(torch.int32)


def _ceil(a, b):
    return -(-a // b)


def _zeros(*shape, dtype=torch.int32):
    return torch.zeros(shape, dtype=dtype, device="cuda")


def _tables(n, blocks, page, ids):
    """A page of ``ids`` for every block that n tokens of a sequence begin, -1 behind."""
    used = (n + page - 1) // page
    first = torch.cumsum(used, 0) - used
    at = torch.arange(blocks, device="cuda")[None]
    return torch.where(at < used[:, None], ids[(first[:, None] + at).clamp(max=ids.shape[0] - 1)],
                       torch.full((), -1, dtype=torch.int32, device="cuda")).contiguous()


def _sequences(case, draw):
    """Lengths and tables of a serving batch: of every three sequences one goes on from the one before it, its first
    half of whole pages shared; a quarter has ended, its table left as it was.  Also the cache's pages."""
    b, top, page = case["batch"], case["length"], case["page"]
    n = draw.stages(top - 1, b) + 1
    blocks = _ceil(top, page)
    pages = b * blocks + 3
    table = _tables(n, blocks, page, draw.order(pages))
    row = torch.arange(b, device="cuda")
    before = (row - 1).clamp(min=0)
    shared = torch.where(row % 3 == 1, torch.minimum(n, n[before]) // page // 2, 0)
    table = torch.where(torch.arange(blocks, device="cuda") < shared[:, None], table[before], table).contiguous()
    ended = draw.ints(0, 3, b) == 0
    ended[0] = False
    return torch.where(ended, 0, n).to(torch.int32), table, pages


def prepare(case, seed):
    draw, kind = _Inputs(seed), case["kind"]
    if kind == "extend":
        b, h, hk, d, page = (case[k] for k in ("batch", "heads", "kv_heads", "dim", "page"))
        if case["ragged"]:
            new, held = draw.stages(case["chunk"], b), draw.stages(case["held"], b)
            new[1:] = torch.where(new[1:] * 8 < case["chunk"], 0, new[1:])      # an eighth has nothing to add
        else:
            new = torch.full((b,), case["chunk"], dtype=torch.int32, device="cuda")
            held = torch.full((b,), case["held"], dtype=torch.int32, device="cuda")
        n = held + new
        starts = torch.cat([new.new_zeros(1), torch.cumsum(new, 0).to(torch.int32)])
        rows = int(starts[-1]) + (5 if case["ragged"] else 0)   # a padded list: rows behind the last sequence
        pages = int(((n + page - 1) // page).sum())
        blocks = _ceil(case["chunk"] + case["held"], page)
        t = dict(q=draw.normal(rows, h, d, scale=1.5), k=draw.normal(pages, hk, page, d, dtype=TYPES[case["type"]]),
                 v=draw.normal(pages, hk, page, d, dtype=TYPES[case["type"]]),
                 tables=_tables(n, blocks, page, draw.order(pages)), lengths=n.to(torch.int32), starts=starts,
                 out=torch.zeros(rows, h, d, device="cuda"))
    elif kind == "score":
        n, v, top = case["rows"], case["vocab"], case["top"]
        tokens = draw.ints(0, v - 1, n, dtype=torch.int64)
        if n > 4:
            tokens[n // 2] = -1                                 # a padded row
        t = dict(logits=draw.normal(n, v, scale=2.5), tokens=tokens, logprobs=torch.empty(n, device="cuda"),
                 entropy=torch.empty(n, device="cuda"), ids=_zeros(n, top, dtype=torch.int64),
                 values=torch.empty(n, top, device="cuda"))
    elif kind == "fork":
        p, e, hk, d, page, top = (case[k] for k in ("parents", "each", "kv_heads", "dim", "page", "length"))
        blocks, total = _ceil(top, page), p * (e + 1)
        place = draw.order(total)                               # parents and children lie in any rows
        n = draw.ints(max(1, top - page + 1), top, p)
        pages = p * (blocks + e) + 5
        ids = draw.order(pages)
        lengths, tables = _zeros(total), torch.full((total, blocks), -1, dtype=torch.int32, device="cuda")
        lengths[place[:p].long()] = n
        tables[place[:p].long()] = _tables(n, blocks, page, ids)
        t = dict(parents=place[:p].repeat_interleave(e).contiguous(), children=place[p:].contiguous(), tables=tables,
                 lengths=lengths, free=ids[p * blocks:].contiguous(), taken=torch.full_like(_zeros(1), 2),
                 taken_out=_zeros(1), k=draw.normal(LAYERS, pages, hk, page, d, dtype=TYPES[case["type"]]),
                 v=draw.normal(LAYERS, pages, hk, page, d, dtype=TYPES[case["type"]]))
    elif kind == "free":
        n, table, pages = _sequences(case, draw)
        t = dict(lengths=n, tables=table, free=_zeros(pages), count=_zeros(1))
    else:
        n, table, pages = _sequences(case, draw)
        room = case["batch"] * (table.shape[1] + 3) // 2 + table.shape[1]        # for all that can be held, and more
        shape = (case["kv_heads"], case["page"], case["dim"])
        kt = TYPES[case["type"]]
        t = dict(lengths=n, tables=table, k=draw.normal(LAYERS, pages, *shape, dtype=kt),
                 v=draw.normal(LAYERS, pages, *shape, dtype=kt), k_new=_zeros(LAYERS, room, *shape, dtype=kt),
                 v_new=_zeros(LAYERS, room, *shape, dtype=kt), tables_new=_zeros(*table.shape), used=_zeros(1))
    return {"case": case, **{k: _Held(v) for k, v in t.items()}}


# ----------------------------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------------------------

def _calls(s):
    from cv3amd import paged
    case, kind = s["case"], s["case"]["kind"]
    a = {k: v.array for k, v in s.items() if k != "case"}
    if kind == "extend":
        paged.extend(a["q"], a["k"], a["v"], a["tables"], a["lengths"], a["starts"], window=case["window"] or None,
                     out=a["out"])
        return s["out"].tensor
    if kind == "score":
        out = (a["logprobs"], a["entropy"], a["ids"], a["values"])
        paged.token_logprobs(a["logits"], a["tokens"], top=case["top"], out=out)
        return [s[k].tensor for k in ("logprobs", "entropy", "ids", "values")]
    if kind == "fork":
        paged.fork(a["parents"], a["children"], a["tables"], a["lengths"], a["free"], a["taken"], a["k"], a["v"],
                   out=a["taken_out"])
        return [s[k].tensor for k in ("tables", "lengths", "taken_out", "k", "v")]
    if kind == "free":
        paged.free_pages(a["tables"], a["lengths"], case["page"], s["free"].tensor.shape[0],
                         out=(a["free"], a["count"]))
        return [s["free"].tensor, s["count"].tensor]
    paged.compact(a["tables"], a["lengths"], a["k"], a["v"], a["k_new"], a["v_new"], out=(a["tables_new"], a["used"]))
    return [s[k].tensor for k in ("tables_new", "used", "k_new", "v_new")]


def _plain_extend(t, case):
    """The batch padded to its longest chunk and its longest cache."""
    q, table, n, starts = t["q"], t["tables"].clamp(min=0), t["lengths"].long(), t["starts"].long()
    rows, h, d = q.shape
    _, hk, page, _ = t["k"].shape
    b, keys, chunk = n.shape[0], table.shape[1] * page, case["chunk"]
    k, v = (t[x][table].float().transpose(1, 2).reshape(b, hk, keys, d) for x in "kv")
    i, at = torch.arange(chunk, device=q.device), torch.arange(keys, device=q.device)
    new = starts[1:] - starts[:-1]
    x = q[(starts[:-1, None] + i).clamp(max=rows - 1)].reshape(b, chunk, hk, h // hk, d).permute(0, 2, 3, 1, 4)
    s = torch.matmul(x.reshape(b, hk, -1, d) / math.sqrt(d), k.transpose(2, 3).contiguous())
    pos = (n - new)[:, None] + i
    seen = (at <= pos[..., None]) & (i < new[:, None])[..., None]
    if case["window"]:
        seen = seen & (at > pos[..., None] - case["window"])
    s = torch.where(seen[:, None, None], s.view(b, hk, h // hk, chunk, keys), -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top > -math.inf, top, 0.0))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(b, hk, -1, keys), v).view(b, hk, h // hk, chunk, d) / torch.where(total > 0, total, 1.0)
    o = o.permute(0, 3, 1, 2, 4).reshape(b, chunk, h, d)
    row = torch.arange(rows, device=q.device)
    of = torch.searchsorted(starts[1:].contiguous(), row, right=True).clamp(max=b - 1)
    got = o[of, (row - starts[of]).clamp(max=chunk - 1)]
    return torch.where((row < starts[-1])[:, None, None], got, t["out"])


def _plain_score(t, top):
    """Sums in 64 bits: an entropy is a small difference of long ones."""
    x, tokens = t["logits"], t["tokens"]
    v = x.shape[1]
    x64 = x.double()
    e = torch.exp(x64 - x64.amax(-1, keepdim=True))
    total = e.sum(-1, keepdim=True)
    lse = x64.amax(-1, keepdim=True) + total.log()
    entropy = lse[:, 0] - (e * x64).sum(-1) / total[:, 0]
    given = (tokens >= 0) & (tokens < v)
    lp = torch.where(given, x64.gather(1, tokens.clamp(0, v - 1)[:, None])[:, 0] - lse[:, 0], 0.0)
    bits = x.view(torch.int32).long()
    order = torch.where(bits < 0, -(bits & 0x7fffffff), bits)               # rises with the logit; -0.0 as 0.0
    best = (order * (1 << 20) + (v - 1 - torch.arange(v, device=x.device))).topk(top, dim=-1).values
    ids = v - 1 - (best & ((1 << 20) - 1))
    return [lp.float(), entropy.float(), ids, (x64.gather(1, ids) - lse).float()]


def _plain_fork(t):
    parents, children, table, free = t["parents"].long(), t["children"].long(), t["tables"], t["free"]
    kc, vc = t["k"], t["v"]
    page, blocks = kc.shape[3], table.shape[1]
    n = t["lengths"][parents].long()
    full, rest = n // page, n % page
    need = (rest > 0).long()
    index = t["taken"].long() + torch.cumsum(need, 0) - need
    fresh = torch.where((need > 0) & (index < free.shape[0]), free[index.clamp(max=free.shape[0] - 1)], -1)
    at = torch.arange(blocks, device=table.device)
    source = table[parents].gather(1, (full * need)[:, None])[:, 0].long()      # with nothing to copy, the first page
    row = torch.where(at < full[:, None], table[parents], torch.where(at == full[:, None], fresh[:, None], -1))
    table[children] = row.int()
    t["lengths"][children] = n.int()
    moved = (torch.arange(page, device=table.device) < rest[:, None])[None, :, None, :, None]
    to = torch.where(fresh >= 0, fresh, source).long()
    for c in (kc, vc):
        c[:, to] = torch.where(moved, c[:, source], c[:, to])
    return [table, t["lengths"], (t["taken"] + need.sum()).int(), kc, vc]


def _used(t, page, pages):
    """Which pages a live sequence holds, and which entries of the tables are its."""
    table = t["tables"].long()
    live = torch.arange(table.shape[1], device=table.device) < ((t["lengths"].long() + page - 1) // page)[:, None]
    used = torch.zeros(pages + 1, dtype=torch.int32, device=table.device)
    used[torch.where(live, table, pages).reshape(-1)] = 1
    return used[:pages], live, table


def _plain_free(t, page):
    pages = t["free"].shape[0]
    used, _, _ = _used(t, page, pages)
    order = torch.argsort(used, stable=True)
    count = pages - used.sum()
    at = torch.arange(pages, device=used.device)
    return [torch.where(at < count, order, -1).int(), count.int().reshape(1)]


def _plain_compact(t):
    kc, vc, kn, vn = t["k"], t["v"], t["k_new"], t["v_new"]
    used, live, table = _used(t, kc.shape[3], kc.shape[1])
    rank = torch.cumsum(used, 0) - used
    order = torch.argsort(1 - used, stable=True)[:kn.shape[1]]
    held = (used[order] > 0)[None, :, None, None, None]
    for c, new in ((kc, kn), (vc, vn)):
        new.copy_(torch.where(held, c[:, order], new))
    return [torch.where(live, rank[table.clamp(min=0)], -1).int(), used.sum().int().reshape(1), kn, vn]


def run(s):
    if own:
        return _calls(s)
    case, kind = s["case"], s["case"]["kind"]
    t = {k: v.tensor for k, v in s.items() if k != "case"}
    if kind == "extend":
        return _plain_extend(t, case)
    if kind == "score":
        return _plain_score(t, case["top"])
    if kind == "fork":
        return _plain_fork(t)
    return _plain_free(t, case["page"]) if kind == "free" else _plain_compact(t)


# ----------------------------------------------------------------------------------------------
# what a pass cannot do without
# ----------------------------------------------------------------------------------------------

def work(case):
    """Where sizes come from the seed, their mean."""
    kind = case["kind"]
    size = {"f32": 4, "f16": 2, "bf16": 2}.get(case.get("type"), 4)
    if kind == "extend":
        b, h, hk, d, chunk, held = (case[k] for k in ("batch", "heads", "kv_heads", "dim", "chunk", "held"))
        seqs = [(chunk, held)]
        if case["ragged"]:
            seqs += [(chunk * i / b if 8 * (chunk * i // b) >= chunk else 0, held / 2) for i in range(1, b)]
        else:
            seqs = seqs * b
        read = seen = 0.0
        for c, p in seqs:
            if not c:
                continue
            w = case["window"] or c + p
            read += min(c + p, c + w)
            # rows see min(w, position + 1) keys: a rising part and a level one
            rise = min(max(w - p, 0), c)
            seen += rise * (p + (rise + 1) / 2) + (c - rise) * min(w, p + c)
        rows = sum(c for c, _ in seqs)
        return {"bytes": read * 2 * hk * d * size + read / case["page"] * 4 + 8.0 * rows * h * d + 8.0 * b,
                "flops": 4.0 * seen * h * d}
    if kind == "score":
        n, v, top = case["rows"], case["vocab"], case["top"]
        return {"bytes": n * (4.0 * v + 8 + 8 + 12 * top), "flops": 4.0 * n * v}
    if kind == "fork":
        p, e, page, top = case["parents"], case["each"], case["page"], case["length"]
        rest = (min(page, top) - 1) / 2                                     # rows of a part-filled page
        row = 2 * LAYERS * case["kv_heads"] * case["dim"] * size
        return {"bytes": (p + p * e) * rest * row + p * (e + 1) * (4.0 * _ceil(top, page) + 8), "flops": 0}
    b, top, page = case["batch"], case["length"], case["page"]
    entries = b * 0.75 * ((top + 1) / 2 / page + 0.5)                       # of sequences that have not ended
    pages = b * _ceil(top, page) + 3
    if kind == "free":
        return {"bytes": 4.0 * b + 4 * entries + 4 * max(0.0, pages - entries), "flops": 0}
    one = 2.0 * LAYERS * case["kv_heads"] * page * case["dim"] * size
    return {"bytes": 2 * 0.9 * entries * one + 4.0 * b + 4 * entries + 4 * b * _ceil(top, page), "flops": 0}


# ----------------------------------------------------------------------------------------------
# the same results in 64 bits, from the definitions
# ----------------------------------------------------------------------------------------------

def _exact_extend(case, t):
    h, hk, d, page = (case[k] for k in ("heads", "kv_heads", "dim", "page"))
    out = t["out"].double()
    n, starts = t["lengths"].tolist(), t["starts"].tolist()
    for b, total in enumerate(n):
        r0, r1 = starts[b], starts[b + 1]
        if r1 <= r0:
            continue
        ids = t["tables"][b, :_ceil(total, page)].long()
        pos = torch.arange(total - (r1 - r0), total, device="cuda")[:, None]
        at = torch.arange(total, device="cuda")[None]
        hidden = at > pos
        if case["window"]:
            hidden |= at <= pos - case["window"]
        for j in range(hk):
            k, v = (t[x][ids, j].double().reshape(-1, d)[:total] for x in "kv")
            kt = k.t().contiguous()
            for i in range(j * (h // hk), (j + 1) * (h // hk)):
                s = (t["q"][r0:r1, i].double() @ kt) / math.sqrt(d)
                out[r0:r1, i] = torch.softmax(s.masked_fill_(hidden, -math.inf), dim=1) @ v
    return out


def _exact_score(case, t):
    n, top = case["rows"], case["top"]
    lp = torch.zeros(n, dtype=torch.float64, device="cuda")
    entropy, best = torch.zeros_like(lp), torch.zeros(n, top, dtype=torch.float64, device="cuda")
    for r0 in range(0, n, 64):
        x = torch.log_softmax(t["logits"][r0:r0 + 64].double(), dim=1)
        tok = t["tokens"][r0:r0 + 64]
        picked = x.gather(1, tok.clamp(min=0)[:, None])[:, 0]
        lp[r0:r0 + 64] = torch.where(tok >= 0, picked, torch.zeros_like(picked))
        entropy[r0:r0 + 64] = torch.special.entr(x.exp()).sum(1)
        best[r0:r0 + 64] = x.sort(dim=1, descending=True).values[:, :top]
    return [lp, entropy, None, best]


def _exact_fork(case, t):
    page = case["page"]
    n, parents, children = (t[x].tolist() for x in ("lengths", "parents", "children"))
    table, free, taken = t["tables"].tolist(), t["free"].tolist(), int(t["taken"])
    caches = [t["k"].clone(), t["v"].clone()]
    for p, _ in zip(parents, children):
        full, rest = divmod(n[p], page)
        if rest:
            for new, old in zip(caches, (t["k"], t["v"])):
                new[:, free[taken], :, :rest] = old[:, table[p][full], :, :rest]
            taken += 1
    return [None, None, None] + caches              # moved, not computed: the values of the cache's own type are exact


def _exact_compact(case, t):
    page, n, table = case["page"], t["lengths"].tolist(), t["tables"].tolist()
    held = sorted({p for row, m in zip(table, n) for p in row[:_ceil(m, page)]})
    done = []
    for c, new in ((t["k"], t["k_new"]), (t["v"], t["v_new"])):
        new = new.clone()
        for i, p in enumerate(held):
            new[:, i] = c[:, p]
        done.append(new)
    return [None, None] + done


def exact(case, seed):
    kind = case["kind"]
    if kind == "free":
        return None
    t = {k: v.tensor for k, v in prepare(case, seed).items() if k != "case"}
    if kind == "extend":
        return _exact_extend(case, t)
    if kind == "score":
        return _exact_score(case, t)
    return _exact_fork(case, t) if kind == "fork" else _exact_compact(case, t)
