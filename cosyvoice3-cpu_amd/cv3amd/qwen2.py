"""Device-resident Qwen2 decode (the CosyVoice3 LM's token loop) on ``cv3_qwen2_decode_step``.

Restates the single-token path of cv3cpu/models/qwen2.py:139-179 and the head /
speech-embedding of cv3cpu/models/llm.py:68-77,121.  The reference samples
(llm.py:112-149); this path is greedy: argmax of the head logits with ties to
the lowest id, which is the first entry of the reference's stable
``np.argsort(-p)`` (llm.py:138).

Layout in HBM (L layers, D = hidden, dh = head_dim, I = intermediate):
  * per projection, one stacked int8 array for all layers: ``qkv`` [L*(H+2Hk)*dh, Kp]
    ([q; k; v] rows per layer), ``o`` [L*D, Kp], ``gate_up`` [L*2I, Kp]
    ([gate; up] rows per layer), ``down`` [L*D, Kp], each with its scales;
  * ``k_cache`` / ``v_cache`` [L, Hk, cap, dh] float32 (qwen2.py:74-121);
  * rotary tables cos / sin [cap, dh] built once on the host with the reference's
    float64 expressions (qwen2.py:46-56);
  * ``pos``, ``token``, ``history`` in device memory so that a captured graph of
    one step replays for every token.
"""

from __future__ import annotations

import ctypes
import threading
from typing import List, Optional, Tuple

import numpy as np

from . import _lib, paged
from .device import DeviceArray, Graph, synchronize, to_device

c_i64, c_vp = ctypes.c_int64, ctypes.c_void_p

# generate_batch: requests of one call of the block tables or the reordering, prompt tokens of one pass of the body
# (3.6 GB of rows at Qwen2-0.5B's sizes)
_TABLE_ROWS, _PROMPT_ROWS = 4096, 65536
# Prompts of so few tokens in all, that read so many numbers of keys, take one-token attention, a launch that starts sooner:
# generate_batch of one token after a prompt of 50 (24 layers, float32 cache) 2.52 ms, 2.64 by extend, of 200 3.04 and 3.21,
# two of 100 2.92 and 3.03, eight of 20 2.75 and 2.87; two of 200 4.05 and 4.07, eight of 50 3.84 and 3.83.
_FEW_ROWS, _FEW_NUMBERS = 256, 1 << 22
# Keys of one pass of score_batch: eight passes of the body and more, 13 GB of float32 cache at Qwen2-0.5B's sizes
_SCORE_KEYS = 1 << 19


class QWeight(ctypes.Structure):
    _fields_ = [("q", c_vp), ("scales", c_vp), ("rows", c_i64), ("k", c_i64), ("kp", c_i64), ("block", c_i64),
                ("scale_dtype", ctypes.c_int), ("kind", ctypes.c_int)]


class Model(ctypes.Structure):
    _fields_ = [("layers", c_i64), ("hidden", c_i64), ("heads", c_i64), ("kv_heads", c_i64), ("head_dim", c_i64),
                ("inter", c_i64), ("eps", ctypes.c_float),
                ("qkv", QWeight), ("o", QWeight), ("gate_up", QWeight), ("down", QWeight), ("head", QWeight),
                ("embedding", QWeight),
                ("qkv_bias", c_vp), ("ln1", c_vp), ("ln2", c_vp), ("norm", c_vp), ("head_bias", c_vp),
                ("rope_cos", c_vp), ("rope_sin", c_vp)]


class Persist(ctypes.Structure):
    _fields_ = [("words", c_vp), ("words_len", c_i64), ("err", c_vp), ("epoch_base", ctypes.c_uint32),
                ("workgroups", ctypes.c_int), ("cooperative", ctypes.c_int)]


class CodePlanes(ctypes.Structure):
    _fields_ = [("frag", c_vp), ("scales", c_vp), ("block", c_i64)]


class Planes(ctypes.Structure):
    _fields_ = [("qkv", CodePlanes), ("o", CodePlanes), ("gate_up", CodePlanes), ("down", CodePlanes),
                ("qkv_bias", c_vp)]


class Sampler(ctypes.Structure):
    _fields_ = [("top_p", ctypes.c_double), ("rep_threshold", ctypes.c_double), ("top_k", c_i64),
                ("win_size", c_i64), ("speech_token_size", c_i64), ("min_len", c_i64),
                ("strict_min_len", ctypes.c_int), ("ctl", c_vp)]


_M64 = (1 << 64) - 1


class State(ctypes.Structure):
    _fields_ = [("k_cache", c_vp), ("v_cache", c_vp), ("cap", c_i64), ("pos", c_vp), ("token", c_vp),
                ("history", c_vp), ("x", c_vp), ("logits", c_vp), ("workspace", c_vp),
                ("workspace_floats", c_i64)]


def rope_tables(dim: int, theta: float, n: int):
    """HF half-split cos/sin: float64 angles and cos/sin, stored float32 (qwen2.py:46-56)."""
    inv = 1.0 / (theta ** (np.arange(0, dim, 2, dtype=np.float64) / dim))
    ang = np.arange(n, dtype=np.float64)[:, None] * inv[None, :]
    ang = np.concatenate([ang, ang], axis=-1)
    return np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)


def _kind(w):
    return getattr(w, "kind", None)


def _host(a):
    return a.numpy() if isinstance(a, DeviceArray) else np.asarray(a)


def widen_q4_codes(packed: np.ndarray) -> np.ndarray:
    """q4 codes (quant.py:70-86: per 32-code block 16 bytes, byte j holding code j in its low
    nibble and code j + 16 in its high nibble, each + 8) as int8 codes n - 8, K in order."""
    b = np.ascontiguousarray(packed, dtype=np.uint8)
    rows, half = b.shape
    blocks = b.reshape(rows, half // 16, 16)
    codes = np.concatenate([blocks & 0x0F, blocks >> 4], axis=2).astype(np.int16) - 8
    return codes.reshape(rows, half * 2).astype(np.int8)


class _Stacked:
    """Rows of several q8 or q4 QTensors (per layer, in order) stacked into one device array.

    ``widen``: q4 rows are stored as int8 codes (n - 8) with their 32-code blocks and float16
    scales, i.e. the same weights, dequantised to the same floats, twice the bytes.  The decode
    step is latency-bound, and unpacking nibbles is VALU work on its critical path."""

    def __init__(self, per_layer: List[List[object]], widen: bool = False):
        qs, ss = [], []
        first = per_layer[0][0]
        self.k = int(first.shape[1])
        self.block = int(first.block)
        self.kind = _kind(first)
        sdt = np.dtype(_host(first.scales).dtype)
        for parts in per_layer:
            for w in parts:
                if _kind(w) not in ("q8", "q4"):
                    raise ValueError("the device decode takes q8 or q4 weights (the balanced and tiny profiles)")
                if (int(w.shape[1]) != self.k or int(w.block) != self.block or _host(w.scales).dtype != sdt
                        or _kind(w) != self.kind):
                    raise ValueError("stacked weights must share kind, K, block and scale dtype")
                qs.append(_host(w.q))
                ss.append(_host(w.scales))
        self.rows = sum(int(w.shape[0]) for w in per_layer[0])
        q = np.concatenate(qs, axis=0)
        s = np.concatenate(ss, axis=0)
        self.kp = int(s.shape[1]) * self.block  # q4 rows hold kp / 2 bytes
        self.source_nbytes = q.nbytes + s.nbytes   # the checkpoint's bytes (q4: packed nibbles)
        self.widened = bool(widen and self.kind == "q4")
        if self.widened:
            q = widen_q4_codes(q)
            self.kind = "q8"
        cpc = 32 if self.kind == "q4" else 16
        if self.kp % cpc or self.block % cpc:
            raise ValueError(f"padded K and block must be multiples of {cpc}")
        self.sf16 = sdt == np.dtype(np.float16)
        self.q = to_device(np.ascontiguousarray(q))
        self.scales = to_device(np.ascontiguousarray(s))

    def layer(self, layer: int, row0: int = 0, rows: Optional[int] = None):
        """linear_q arguments (kind, codes, scales, scale dtype, kp, block, n) of rows
        [row0, row0 + rows) of one layer."""
        rows = self.rows - row0 if rows is None else rows
        row_bytes = self.kp // 2 if self.kind == "q4" else self.kp
        nb = self.kp // self.block
        r = layer * self.rows + row0
        return (_lib.KIND_Q4 if self.kind == "q4" else _lib.KIND_Q8, self.q.ptr + r * row_bytes,
                self.scales.ptr + r * nb * (2 if self.sf16 else 4), _lib.F16 if self.sf16 else _lib.F32,
                self.kp, self.block, rows)

    def struct(self) -> QWeight:
        return QWeight(self.q.ptr, self.scales.ptr, self.rows, self.k, self.kp, self.block,
                       _lib.F16 if self.sf16 else _lib.F32, _lib.KIND_Q4 if self.kind == "q4" else _lib.KIND_Q8)

    def plane_arrays(self, rows: int):
        """(fragments, scales), empty, for ``rows`` rows of every layer: all the memory that ``planes`` takes."""
        layers, nc, ns = self.q.shape[0] // self.rows, ctypes.c_int64(), ctypes.c_int64()
        _lib.call("code_planes_elems", rows, self.k, self.block, ctypes.byref(nc), ctypes.byref(ns))
        return DeviceArray((layers, nc.value), np.uint16), DeviceArray((layers, ns.value))

    def planes(self, span: int = 0, limit: int = 0, row0: int = 0, rows: Optional[int] = None, arrays=None):
        """(fragments, scales) of every layer's rows (or rows [row0, row0 + rows)) for cv3_linear_code_planes, each
        layer packed on its own; ``span`` / ``limit`` interleave rows as cv3_pack_code_planes does."""
        rows = self.rows - row0 if rows is None else rows
        frag, scales = self.plane_arrays(rows) if arrays is None else arrays
        for l in range(frag.shape[0]):
            kind, q, sc, sdt, kp, block, n = self.layer(l, row0, rows)
            _lib.call("pack_code_planes", kind, q, n, self.k, sc, sdt, kp, block, span, limit,
                      frag.ptr + 2 * l * frag.shape[1], scales.ptr + 4 * l * scales.shape[1], None)
        return frag, scales

    @property
    def nbytes(self):
        """Bytes held in HBM (a widened q4 body: int8 codes)."""
        return self.q.nbytes + self.scales.nbytes


class DeviceQwen2:
    """Qwen2 body + CosyVoice3 LM head resident on the device, decoding greedily."""

    def __init__(self, weights, prefix: str = "llm.", cap: int = 1024, widen_q4: bool = False,
                 prompt_planes: bool = True):
        """A q4 body (the tiny profile) is held in HBM as the checkpoint's packed nibbles; the
        one-launch step decodes it at the int8 body's rate.  ``widen_q4`` holds it as int8
        codes with the same blocks and scales instead (identical weights, twice the bytes),
        which the five-kernel step reads a little faster.

        ``prompt_planes`` keeps the body a second time, laid out for ``prefill`` at two bytes a code
        (``prompt_nbytes``: 0.72 GB for Qwen2-0.5B beside 0.2 - 0.4 GB).  Without it, or without the
        memory for it, prompts run on the decode's rows (500 tokens 8.2 ms against 2.7)."""
        _lib.init()
        m = weights.meta["qwen2"]
        self.layers = int(m["num_hidden_layers"])
        self.hidden = int(m["hidden_size"])
        self.heads = int(m["num_attention_heads"])
        self.kv_heads = int(m["num_key_value_heads"])
        self.inter = int(m["intermediate_size"])
        self.eps = float(m.get("rms_norm_eps", 1e-6))
        self.theta = float(m.get("rope_theta", 1e6))
        self.head_dim = self.hidden // self.heads
        if cap % 64 or cap > 1024:
            raise ValueError("cache capacity must be a multiple of 64, at most 1024")
        self.cap = int(cap)
        body = prefix + "model."
        g = weights.get
        L = range(self.layers)
        lp = [f"{body}layers.{i}." for i in L]
        self.qkv = _Stacked([[g(p + f"self_attn.{x}_proj.weight") for x in "qkv"] for p in lp], widen_q4)
        self.o = _Stacked([[g(p + "self_attn.o_proj.weight")] for p in lp], widen_q4)
        self.gate_up = _Stacked([[g(p + "mlp.gate_proj.weight"), g(p + "mlp.up_proj.weight")] for p in lp], widen_q4)
        self.down = _Stacked([[g(p + "mlp.down_proj.weight")] for p in lp], widen_q4)
        self.head = _Stacked([[g(prefix + "llm_decoder.weight")]])
        self.emb = _Stacked([[g(prefix + "speech_embedding")]])
        f32 = lambda a: np.asarray(_host(a), np.float32)  # noqa: E731
        self.qkv_bias = to_device(np.concatenate([f32(g(p + f"self_attn.{x}_proj.bias")) for p in lp for x in "qkv"]))
        self.ln1 = to_device(np.concatenate([f32(g(p + "input_layernorm")) for p in lp]))
        self.ln2 = to_device(np.concatenate([f32(g(p + "post_attention_layernorm")) for p in lp]))
        self.norm = to_device(f32(g(body + "norm")))
        hb = prefix + "llm_decoder.bias"
        self.head_bias = to_device(f32(g(hb))) if hb in weights else None
        c, s = rope_tables(self.head_dim, self.theta, self.cap)
        self.rope_cos, self.rope_sin = to_device(c), to_device(s)
        self.vocab = self.head.rows
        self.model = Model(self.layers, self.hidden, self.heads, self.kv_heads, self.head_dim, self.inter,
                           self.eps, self.qkv.struct(), self.o.struct(), self.gate_up.struct(), self.down.struct(),
                           self.head.struct(), self.emb.struct(), self.qkv_bias.ptr, self.ln1.ptr, self.ln2.ptr,
                           self.norm.ptr, self.head_bias.ptr if self.head_bias is not None else None,
                           self.rope_cos.ptr, self.rope_sin.ptr)
        # state
        cache_shape = (self.layers, self.kv_heads, self.cap, self.head_dim)
        self.k_cache = DeviceArray(cache_shape).zero_()
        self.v_cache = DeviceArray(cache_shape).zero_()
        self.ints = DeviceArray((2 + self.cap,), np.int64).zero_()   # pos, token, history[cap]
        self.x = DeviceArray((self.hidden,))
        self.logits = DeviceArray((self.vocab,))
        nws = 1024 + self.heads * 16 * 64 + self.heads * 16 * 2 + self.inter + 64
        self.workspace = DeviceArray((nws,))
        p0 = self.ints.ptr
        self.state = State(self.k_cache.ptr, self.v_cache.ptr, self.cap, p0, p0 + 8, p0 + 16, self.x.ptr,
                           self.logits.ptr, self.workspace.ptr, nws)
        self._prompt, self._prompt_arrays = None, []
        # the body's projections for generate_batch, packed on its first call
        self._batch, self._batch_lock = None, threading.Lock()
        if prompt_planes:
            try:
                self._prompt = self._prompt_planes()
            except _lib.HIPError:    # out of memory
                self._prompt_arrays = []
        self._graph: Optional[Graph] = None
        self._pos_host = 0
        # sampler control block: [start, stop step + 1, PCG64 state hi, lo, inc hi, lo]
        self.ctl = DeviceArray((6,), np.int64).zero_()
        self._sampled_graphs = {}
        self._persist: Optional[Persist] = None   # exchange words of the one-launch step, made on first use
        # the one-launch step's launch: ordinary (the device runs nothing else meanwhile) or
        # hipLaunchCooperativeKernel, which guarantees co-residency at ~20 us more per token
        self.cooperative = False

    def _prompt_planes(self) -> Optional[Planes]:
        """The body's projections as code planes for ``prefill`` (cv3_qwen2_prefill), beside the decode's
        rows: q and k heads with their halves interleaved, so that a rotary pair is two neighbouring
        outputs, and gate beside up.  None for geometries it does not take."""
        D, I, dh = self.hidden, self.inter, self.head_dim
        ok = (dh == 64 and self.heads * dh == D and D % 64 == 0 and 256 <= D <= 1024 and I % 64 == 0 and I >= 256
              and self.heads % self.kv_heads == 0)
        for w in (self.qkv, self.o, self.gate_up, self.down):
            ok = ok and w.rows % 32 == 0 and (w.block in (32, 64) or w.block >= w.k) and w.kp % 16 == 0
        if not ok:
            return None
        turned = (self.heads + self.kv_heads) * dh
        p = Planes()
        for name, w, span, limit in (("qkv", self.qkv, dh, turned), ("o", self.o, 0, 0),
                                     ("gate_up", self.gate_up, 2 * I, 2 * I), ("down", self.down, 0, 0)):
            frag, scales = w.planes(span, limit)
            self._prompt_arrays += [frag, scales]
            setattr(p, name, CodePlanes(frag.ptr, scales.ptr, w.block))
        b = self.qkv_bias.numpy().reshape(self.layers, -1)
        qk = b[:, :turned].reshape(self.layers, -1, 2, dh // 2).transpose(0, 1, 3, 2).reshape(self.layers, -1)
        bias = to_device(np.concatenate([qk, b[:, turned:]], axis=1))
        self._prompt_arrays.append(bias)
        p.qkv_bias = bias.ptr
        return p

    @property
    def prompt_nbytes(self) -> int:
        """Bytes held in HBM for ``prefill``; o and down of them serve ``generate_batch`` too."""
        return sum(a.nbytes for a in self._prompt_arrays)

    @property
    def batch_nbytes(self) -> int:
        """Bytes held in HBM for ``generate_batch`` besides: none before its first call on several rows, or where there
        was no memory for them."""
        prompt = {a.ptr for a in self._prompt_arrays}
        return sum(a.nbytes for _, _, *arrays in (self._batch or {}).values() for a in arrays if a.ptr not in prompt)

    # -- weights streamed per token (the HBM roofline numerator) -----------
    def bytes_per_token(self, length: int) -> dict:
        """Algorithmic HBM bytes of one token at KV length ``length`` (keys read = length + 1): the
        checkpoint's weight bytes (a q4 body counts its packed nibbles even when held widened).
        ``body_held`` is what the kernels actually stream for the body: the widened int8 codes
        and their scales when a q4 body is held widened, else the same as ``body``."""
        body = self.qkv.source_nbytes + self.o.source_nbytes + self.gate_up.source_nbytes + self.down.source_nbytes
        held = self.qkv.nbytes + self.o.nbytes + self.gate_up.nbytes + self.down.nbytes
        kv = 2 * self.layers * self.kv_heads * (length + 1) * self.head_dim * 4
        small = 4 * (self.qkv_bias.size + self.ln1.size + self.ln2.size + self.norm.size)
        return {"body": body, "kv": kv, "norms_biases": small, "head": self.head.nbytes, "body_held": held}

    # -- state ------------------------------------------------------------
    def fill_cache(self, k: np.ndarray, v: np.ndarray):
        """Pre-fill positions [0, n) of every layer's cache from host (L, Hk, n, dh) arrays."""
        n = k.shape[2]
        if n >= self.cap:
            raise ValueError("prefill does not fit the cache")
        kc = np.zeros((self.layers, self.kv_heads, self.cap, self.head_dim), np.float32)
        vc = np.zeros_like(kc)
        kc[:, :, :n] = k
        vc[:, :, :n] = v
        self.k_cache.copy_from(kc)
        self.v_cache.copy_from(vc)

    def begin(self, token: int, pos: int):
        """Start decoding with input ``speech_embedding[token]`` at position ``pos``."""
        if not 0 <= pos < self.cap - 1:
            raise ValueError("position outside the cache")
        ints = np.zeros(2 + self.cap, np.int64)
        ints[0], ints[1] = pos, token
        self.ints.copy_from(ints)
        self._pos_host = pos
        _lib.call("qwen2_embed_token", ctypes.byref(self.model), ctypes.byref(self.state), None)

    def step(self, graph: bool = False):
        """Enqueue one greedy token (no host synchronisation)."""
        if self._pos_host + 1 >= self.cap:
            raise ValueError("the KV cache is full")
        if graph:
            if self._graph is None:
                g = Graph()
                with g:
                    _lib.call("qwen2_decode_step", ctypes.byref(self.model), ctypes.byref(self.state), None)
                self._graph = g
            self._graph.launch()
        else:
            _lib.call("qwen2_decode_step", ctypes.byref(self.model), ctypes.byref(self.state), None)
        self._pos_host += 1

    # -- prompt prefill (the body's multi-token forward) -----------------------
    def _linear(self, x: int, m: int, w: "_Stacked", layer: int, y: int, ldy: int, bias=None, row0: int = 0,
                rows: Optional[int] = None, epi=None):
        kind, q, sc, sdt, kp, block, n = w.layer(layer, row0, rows)
        _lib.call("linear_q", kind, x, m, w.k, w.k, q, sc, sdt, kp, block, n, bias, y, ldy,
                  ctypes.byref(epi) if epi is not None else None, None)

    def _after_attention(self, l: int, t: int, att, h, n, u, a, res, swiglu):
        """o_proj + residual, RMSNorm, SwiGLU, down + residual of layer l on t rows (qwen2.py:171-177)."""
        D, I = self.hidden, self.inter
        self._linear(att.ptr, t, self.o, l, h.ptr, D, epi=res)
        _lib.call("rms_norm", h.ptr, self.ln2.ptr + l * D * 4, n.ptr, t, D, self.eps, None)
        self._linear(n.ptr, t, self.gate_up, l, u.ptr, I, row0=I, rows=I)        # up
        self._linear(n.ptr, t, self.gate_up, l, a.ptr, I, row0=0, rows=I, epi=swiglu)  # u * silu(gate)
        self._linear(a.ptr, t, self.down, l, h.ptr, D, epi=res)

    def prefill(self, x, pos0: int = 0):
        """Qwen2Model.forward over T input embeddings at positions pos0 .. pos0 + T - 1
        (qwen2.py:139-179) on the device: RMSNorm, [q; k; v] projection with bias, half-split
        rotary, k and v appended to the cache, causal attention over the cache (mask
        ("causal", pos0) when T > 1), o_proj + residual, RMSNorm, SwiGLU, down + residual.
        On the bfloat16 matrix cores with the activations as planes (cv3_qwen2_prefill) where the
        geometry allows it, else layer by layer on the float32 ones.
        Leaves the head logits of the last position in ``logits`` and ``pos`` at that
        position, so ``select`` / ``generate_*_after_prefill`` draw the next token."""
        xd = x if isinstance(x, DeviceArray) else to_device(np.ascontiguousarray(x, np.float32))
        if xd.ndim != 2 or xd.shape[1] != self.hidden or xd.shape[0] < 1:
            raise ValueError(f"prefill takes (T, {self.hidden}) embeddings, got {xd.shape}")
        t = xd.shape[0]
        if pos0 < 0 or pos0 + t >= self.cap:
            raise ValueError("the prompt does not fit the KV cache")
        D, H, Hk, dh, I, cap = self.hidden, self.heads, self.kv_heads, self.head_dim, self.inter, self.cap
        if self._prompt is not None:
            if xd.ptr % 16:
                xd = xd.copy()
            work = [DeviceArray((t, D)), DeviceArray((t, D))]
            for k in (D, I):
                ne = ctypes.c_int64()
                _lib.call("x3_frag_elems", t, k, ctypes.byref(ne))
                work.append(DeviceArray((ne.value,), np.uint16))
            _lib.call("qwen2_prefill", ctypes.byref(self.model), ctypes.byref(self.state), ctypes.byref(self._prompt),
                      xd.ptr, t, pos0, *(w.ptr for w in work), None)
            self._pos_host = pos0 + t - 1
            return
        R = self.qkv.rows
        h = DeviceArray((t, D))
        _lib.call("copy_d2d", h.ptr, xd.ptr, t * D * 4, None)
        n = DeviceArray((t, D))
        qkv = DeviceArray((t, R))
        att = DeviceArray((t, D))
        u = DeviceArray((t, I))
        a = DeviceArray((t, I))
        res = _lib.epilogue(residual=h.ptr, ld_res=D)
        swiglu = _lib.epilogue(act="silu", gate=u.ptr, gate_stride=I, rows_per_gate=1)
        c64 = ctypes.c_int64 * 3
        for l in range(self.layers):
            _lib.call("rms_norm", h.ptr, self.ln1.ptr + l * D * 4, n.ptr, t, D, self.eps, None)
            self._linear(n.ptr, t, self.qkv, l, qkv.ptr, R, bias=self.qkv_bias.ptr + l * R * 4)
            _lib.call("rope_half", qkv.ptr, t * H, H, R, dh, self.rope_cos.ptr, self.rope_sin.ptr, pos0, None)
            _lib.call("rope_half", qkv.ptr + H * dh * 4, t * Hk, Hk, R, dh, self.rope_cos.ptr, self.rope_sin.ptr,
                      pos0, None)
            for j, cache in enumerate((self.k_cache, self.v_cache)):   # rows pos0 .. of layer l
                _lib.call("copy_strided", qkv.ptr + (H + j * Hk) * dh * 4,
                          cache.ptr + ((l * Hk) * cap + pos0) * dh * 4, Hk, t, dh, c64(dh, R, 1),
                          c64(cap * dh, dh, 1), None)
            kv = l * Hk * cap * dh * 4
            _lib.call("attention", qkv.ptr, self.k_cache.ptr + kv, self.v_cache.ptr + kv, att.ptr, 1, H, Hk, t,
                      pos0 + t, dh, c64(0, dh, R), c64(0, cap * dh, dh), c64(0, cap * dh, dh), c64(0, dh, D),
                      1.0 / np.sqrt(dh), 1 if t > 1 else 0, pos0, 0, None)
            self._after_attention(l, t, att, h, n, u, a, res, swiglu)
        _lib.call("rms_norm", h.ptr + (t - 1) * D * 4, self.norm.ptr, n.ptr, 1, D, self.eps, None)
        self._linear(n.ptr, 1, self.head, 0, self.logits.ptr, self.vocab,
                     bias=self.head_bias.ptr if self.head_bias is not None else None)
        p = np.array([pos0 + t - 1], np.int64)
        _lib.call("copy_h2d", self.ints.ptr, p.ctypes.data, 8, None)
        self._pos_host = pos0 + t - 1

    def select(self, smp: Optional["Sampler"] = None):
        """Draw the next token from the logits already in ``logits`` (greedy without a
        sampler), as a decode step's last kernel does."""
        _lib.call("qwen2_select", ctypes.byref(self.model), ctypes.byref(self.state),
                  ctypes.byref(smp) if smp is not None else None, None)
        self._pos_host += 1

    def step_sampled(self, smp: "Sampler", graph: bool = False, persistent: bool = False):
        """Enqueue one sampled token (no host synchronisation); ``persistent`` runs the
        body and head as one cooperative launch (cv3_qwen2_decode_step_persistent), then
        the draw (cv3_qwen2_select)."""
        if self._pos_host + 1 >= self.cap:
            raise ValueError("the KV cache is full")
        if persistent:
            self.step_persistent(select=False)
            _lib.call("qwen2_select", ctypes.byref(self.model), ctypes.byref(self.state), ctypes.byref(smp), None)
        elif graph:
            key = tuple(getattr(smp, f) for f, _ in Sampler._fields_)
            g = self._sampled_graphs.get(key)
            if g is None:
                g = Graph()
                with g:
                    _lib.call("qwen2_decode_step_sampled", ctypes.byref(self.model), ctypes.byref(self.state),
                              ctypes.byref(smp), None)
                self._sampled_graphs[key] = g
            g.launch()
        else:
            _lib.call("qwen2_decode_step_sampled", ctypes.byref(self.model), ctypes.byref(self.state),
                      ctypes.byref(smp), None)
        self._pos_host += 1

    def generate_sampled_after_prefill(self, max_len: int, min_len: int, sampling, speech_token_size: int,
                                       graph: bool = True, check_every: int = 16,
                                       persistent: bool = False) -> List[int]:
        """generate()'s loop after ``prefill``: the first token is drawn from the prompt's
        logits (llm.py:112-121 at i = 0), the rest by decode steps."""
        return self.generate_sampled(None, self._pos_host, max_len, min_len, sampling, speech_token_size, graph,
                                     check_every, persistent)

    def generate_sampled(self, first_token: Optional[int], pos: int, max_len: int, min_len: int, sampling,
                         speech_token_size: int, graph: bool = True, check_every: int = 16,
                         persistent: bool = False) -> List[int]:
        """The token loop of CosyVoice3LM.generate (llm.py:104-123) with its sampler
        (llm.py:125-149) on the device: up to max_len tokens from input
        speech_embedding[first_token] at position pos, ending before the first stop id.
        ``sampling`` has top_p, top_k, win_size, tau_r, strict_min_len and a NumPy
        PCG64 Generator ``rng``, whose state the device advances exactly as the
        reference's draws would and hands back.  The host looks for a stop every
        ``check_every`` tokens; steps after a stop change nothing.  ``first_token``
        None draws the first token from the logits already present (after ``prefill``,
        whose last position is ``pos``).  ``persistent`` decodes with the one-launch step
        (q8 weights) instead of the five-kernel step."""
        bg = sampling.rng.bit_generator
        st = bg.state
        if st.get("bit_generator") != "PCG64":
            raise ValueError("the device sampler draws from NumPy's PCG64 stream (np.random.default_rng)")
        if pos + max_len + 1 >= self.cap:
            raise ValueError("the generation does not fit the KV cache")
        if not sampling.top_p > 0 or int(sampling.top_k) < 1:
            raise ValueError("a draw needs top_p > 0 and top_k >= 1 (the nucleus would be empty)")
        s, inc = int(st["state"]["state"]), int(st["state"]["inc"])
        ctl = np.array([pos, 0, s >> 64, s & _M64, inc >> 64, inc & _M64], dtype=np.uint64).view(np.int64)
        self.ctl.copy_from(ctl)
        smp = Sampler(float(sampling.top_p), float(sampling.win_size * sampling.tau_r), int(sampling.top_k),
                      int(sampling.win_size), int(speech_token_size), int(min_len),
                      int(bool(getattr(sampling, "strict_min_len", False))), self.ctl.ptr)
        done = 0
        if first_token is None:
            self.select(smp)
            done = 1
        else:
            self.begin(first_token, pos)
        while done < max_len:
            n = min(check_every, max_len - done)
            for _ in range(n):
                self.step_sampled(smp, graph, persistent)
            done += n
            if int(self.ctl.numpy()[1]) != 0:
                break
        if persistent and self.persistent_error():
            raise RuntimeError("the one-launch decode step gave up waiting for an exchange")
        c = self.ctl.numpy().view(np.uint64)
        stop = int(c[1])
        count = stop - 1 if stop else max_len
        new = dict(st)
        new["state"] = {"state": (int(c[2]) << 64) | int(c[3]), "inc": (int(c[4]) << 64) | int(c[5])}
        bg.state = new
        ints = self.ints.numpy()
        self._pos_host = int(ints[0])
        return [int(t) for t in ints[2 + pos + 1: 2 + pos + 1 + count]]

    def generate_after_prefill(self, steps: int, graph: bool = True) -> List[int]:
        """Greedy tokens after ``prefill``: the argmax of the prompt's logits, then steps - 1
        decode steps."""
        pos = self._pos_host
        if pos + steps >= self.cap:
            raise ValueError("the generation does not fit the KV cache")
        self.select(None)
        for _ in range(steps - 1):
            self.step(graph)
        ints = self.ints.numpy()
        return [int(t) for t in ints[2 + pos + 1: 2 + pos + 1 + steps]]

    # -- the whole step as one cooperative launch --------------------------
    def step_persistent(self, select: bool = True):
        """Enqueue one token as a single launch of the whole step (cv3_qwen2_decode_step_persistent,
        cooperative if ``self.cooperative``): greedy selection inside (``select``), or logits only,
        for the sampler (``step_sampled(persistent=True)``)."""
        if self._pos_host + 1 >= self.cap:
            raise ValueError("the KV cache is full")
        need = ctypes.c_int64()
        _lib.call("qwen2_persist_words", ctypes.byref(self.model), 256, _lib.ptr(need))
        need = need.value
        if self._persist is None or self._persist.words_len < need:
            # fresh words are zero, the cleared state no epoch matches
            self._pwords = DeviceArray((need,), np.int64).zero_()
            self._perr = DeviceArray((1,), np.int64).zero_()
            base = self._persist.epoch_base if self._persist is not None else 0
            self._persist = Persist(self._pwords.ptr, need, self._perr.ptr, base, 0, 0)
        p = self._persist
        p.cooperative = 1 if self.cooperative else 0
        base = (p.epoch_base + 256) & 0xFFFFFFFF
        if base == 0:   # the launch counter wrapped: clear the words so no old epoch can match
            self._pwords.zero_()
            base = 256
        p.epoch_base = base
        _lib.call("qwen2_decode_step_persistent", ctypes.byref(self.model), ctypes.byref(self.state),
                  ctypes.byref(p), 1 if select else 0, None)
        self._pos_host += 1 if select else 0

    def persistent_error(self) -> bool:
        """True if a launch of the one-launch step gave up waiting (its results are invalid)."""
        return self._persist is not None and int(self._perr.numpy()[0]) != 0

    def generate_persistent(self, first_token: int, pos: int, steps: int) -> List[int]:
        """Greedy tokens with the one-launch step; raises if a launch gave up."""
        self.begin(first_token, pos)
        for _ in range(steps):
            self.step_persistent(True)
        if self.persistent_error():
            raise RuntimeError("the one-launch decode step gave up waiting for an exchange")
        ints = self.ints.numpy()
        return [int(t) for t in ints[2 + pos + 1: 2 + pos + 1 + steps]]

    def generate(self, first_token: int, pos: int, steps: int, graph: bool = True) -> List[int]:
        self.begin(first_token, pos)
        for _ in range(steps):
            self.step(graph)
        ints = self.ints.numpy()
        return [int(t) for t in ints[2 + pos + 1: 2 + pos + 1 + steps]]

    # -- several sequences, greedy or by beam search, over a paged cache ----
    def _batch_planes(self) -> dict:
        """The body's projections as code planes for rows of several sequences (cv3_linear_rows_planes), each in its own
        row order: two bytes a code beside the decode's rows (``batch_nbytes``), o and down shared with the prompt's.
        Empty for geometries that the planes do not take, or without the memory, which is asked for once: the decode's
        rows serve then (twice to four times the time of a step)."""
        with self._batch_lock:
            if self._batch is not None:
                return self._batch
            parts = {"qkv": (self.qkv, 0, None), "o": (self.o, 0, None), "gate": (self.gate_up, 0, self.inter),
                     "up": (self.gate_up, self.inter, self.inter), "down": (self.down, 0, None)}
            ok = all(w.k % 64 == 0 and w.k >= 256 and w.rows % 4 == 0 and (w.block in (32, 64) or w.block >= w.k)
                     and w.kp % 16 == 0 for w, _, _ in parts.values()) and self.inter % 4 == 0
            shared = {"o": 2, "down": 6} if self._prompt is not None else {}
            made = {n: tuple(self._prompt_arrays[at:at + 2]) for n, at in shared.items()} if ok else {}
            new = [n for n in parts if n not in made] if ok else []
            try:
                made.update({n: parts[n][0].plane_arrays(parts[n][2] or parts[n][0].rows) for n in new})
            except _lib.HIPError:    # out of memory
                made, new = {}, []
            for n in new:
                w, row0, rows = parts[n]
                w.planes(0, 0, row0, rows, made[n])
            synchronize()            # whole before a call on another thread's stream can read them
            self._batch = {n: (w, w.rows if rows is None else rows, *made[n]) for n, (w, _, rows) in parts.items() if made}
        return self._batch

    def _paged_layers(self, x: DeviceArray, pos, slots, tables, lengths, cos, sin, k: DeviceArray, v: DeviceArray,
                      starts=None):
        """The body over rows of any sequences (qwen2.py:139-179): each row's k and v go to its slot, and it sees the
        ``lengths`` keys of its own table row.  With ``starts`` the rows are several tokens of each sequence, the last at
        ``lengths`` - 1, and each sees its sequence up to itself.  Returns the residual stream."""
        t = x.shape[0]
        D, H, R, I = self.hidden, self.heads, self.qkv.rows, self.inter
        h, n, qkv = x.copy(), DeviceArray((t, D)), DeviceArray((t, R))
        q, att = DeviceArray((t, H, self.head_dim)), DeviceArray((t, H, self.head_dim))
        u, a = DeviceArray((t, I)), DeviceArray((t, I))
        res = _lib.epilogue(residual=h.ptr, ld_res=D)
        swiglu = _lib.epilogue(act="silu", gate=u.ptr, gate_stride=I, rows_per_gate=1)
        planes = self._batch_planes() if t > 1 else {}

        def linear(name, x, y, ldy, bias=None, epi=None):
            w, rows, frag, scales = planes[name]
            _lib.call("linear_rows_planes", _lib.KIND_Q4 if w.kind == "q4" else _lib.KIND_Q8, x, t, w.k, w.k,
                      frag.ptr + 2 * l * frag.shape[1], scales.ptr + 4 * l * scales.shape[1], w.block, rows, bias, y, ldy,
                      ctypes.byref(epi) if epi is not None else None, None)

        for l in range(self.layers):
            kl, vl = (c.rows(l, l + 1).reshape(c.shape[1:]) for c in (k, v))
            _lib.call("rms_norm", h.ptr, self.ln1.ptr + l * D * 4, n.ptr, t, D, self.eps, None)
            bias = self.qkv_bias.ptr + l * R * 4
            if planes:
                linear("qkv", n.ptr, qkv.ptr, R, bias)
            else:
                self._linear(n.ptr, t, self.qkv, l, qkv.ptr, R, bias=bias)
            paged.append(qkv, H, pos, slots, cos, sin, kl, vl, out=q)
            if starts is None:
                paged.attention(q, kl, vl, tables, lengths, out=att)
            else:
                paged.extend(q, kl, vl, tables, lengths, starts, out=att)
            if not planes:
                self._after_attention(l, t, att, h, n, u, a, res, swiglu)
                continue
            linear("o", att.ptr, h.ptr, D, None, res)
            _lib.call("rms_norm", h.ptr, self.ln2.ptr + l * D * 4, n.ptr, t, D, self.eps, None)
            linear("gate", n.ptr, a.ptr, I)
            linear("up", n.ptr, u.ptr, I)
            _lib.call("binary", 2, a.ptr, u.ptr, a.ptr, t * I, 0.0, 0.0, None)       # silu(gate) * up
            linear("down", a.ptr, h.ptr, D, None, res)
        return h

    def _ragged(self, x, before, new, tables: DeviceArray, slots, pos, cos, sin, k: DeviceArray, v: DeviceArray):
        """The body over ``new`` tokens of each sequence, after the ``before`` it holds (both the host's), in parts of rows
        that one launch serves: a sequence's earlier keys are in the cache, wherever the cut is.  ``x(t0, t1)`` are the
        rows' embeddings on the device.  Yields (t0, t1, residual stream)."""
        ends = np.cumsum(new, dtype=np.int64)
        begins, part = ends - new, min(_PROMPT_ROWS, (2**23 - 1) // self.heads)
        for t0 in range(0, int(ends[-1]), part):
            t1 = min(t0 + part, int(ends[-1]))
            at = np.flatnonzero((begins < t1) & (ends > t0))
            r = slice(int(at[0]), int(at[-1]) + 1)
            starts = np.clip(np.append(begins[r], ends[r][-1]), t0, t1) - t0
            upto = before[r] + np.minimum(ends[r], t1) - begins[r]
            yield t0, t1, self._paged_layers(x(t0, t1), pos.rows(t0, t1), slots.rows(t0, t1), tables.rows(r.start, r.stop),
                                             to_device(upto.astype(np.int32)), cos, sin, k, v,
                                             to_device(starts.astype(np.int32)))

    def _embedded(self, ids: DeviceArray, out: DeviceArray) -> DeviceArray:
        """Rows of the speech embedding for device ids (int64)."""
        kind, q, sc, sdt, kp, block, n = self.emb.layer(0)
        _lib.call("embedding", kind, q, sc, sdt, n, self.hidden, kp, block, ids.ptr, ids.size, out.ptr, None)
        return out

    @staticmethod
    def _reserve(held, beams: int, new: int, page: int):
        """Pages for ``held`` keys a prompt and ``new`` more a beam: ids (prompts, beams, blocks), -1 behind a prompt's
        last, and their number.  A prompt's whole pages are its beams' together, all others each beam's own."""
        held = held.astype(np.int64)
        shared, last = held // page, -(-(held + new) // page)
        used = shared + beams * (last - shared)
        base, j = (np.cumsum(used) - used)[:, None, None], np.arange(last.max())
        shared, last = shared[:, None, None], last[:, None, None]
        own = np.where(j < shared, base + j, base + shared + np.arange(beams)[None, :, None] * (last - shared) + j - shared)
        return np.where(j < last, own, -1).astype(np.int32), int(used.sum())

    @staticmethod
    def _slots(lengths: DeviceArray, new: DeviceArray, counts, page: int, tables: DeviceArray):
        """block_tables of reserved pages for any number of requests, ``counts`` the host's copy of ``new``: (total, slots,
        positions).  Pages are taken from nobody, so requests can be listed in parts."""
        n = lengths.shape[0]
        if n <= _TABLE_ROWS:
            total, _, _, slots, pos = paged.block_tables(lengths, new, page, None, None, tables, tokens=int(counts.sum()))
            return total, slots, pos
        ends = np.concatenate([[0], np.cumsum(counts, dtype=np.int64)])
        total, slots, pos = DeviceArray((n,), np.int32), DeviceArray((ends[-1],), np.int64), DeviceArray((ends[-1],), np.int32)
        for r0 in range(0, n, _TABLE_ROWS):
            r1 = min(r0 + _TABLE_ROWS, n)
            paged.block_tables(lengths.rows(r0, r1), new.rows(r0, r1), page, None, None, tables.rows(r0, r1),
                               out=(total.rows(r0, r1), None, DeviceArray((r1 - r0 + 1,), np.int32),
                                    slots.rows(ends[r0], ends[r1]), pos.rows(ends[r0], ends[r1])))
        return total, slots, pos

    def _head(self, h: DeviceArray) -> DeviceArray:
        """Head logits of every row (llm.py:74-77)."""
        n, logits = DeviceArray(h.shape), DeviceArray((h.shape[0], self.vocab))
        _lib.call("rms_norm", h.ptr, self.norm.ptr, n.ptr, h.shape[0], self.hidden, self.eps, None)
        self._linear(n.ptr, h.shape[0], self.head, 0, logits.ptr, self.vocab,
                     bias=self.head_bias.ptr if self.head_bias is not None else None)
        return logits

    def generate_batch(self, prompts, max_len: int, min_len: int = 0, speech_token_size: int = 6561, beams: int = 1,
                       page: int = 16, cache: str = "float32") -> List[Tuple[List[int], float]]:
        """Speech tokens for several prompts at once ((T, hidden) embeddings, of any lengths), from one pass of the
        weights a step: greedy, or by beam search with up to 16 ``beams`` a prompt.  Every prompt ends before its
        first stop id (speech_token_size .. + 199; none is chosen below ``min_len``) or after ``max_len`` tokens.
        Returns each prompt's best tokens and the sum of their log probabilities, the stop id's included.

        The sequences share nothing with this object's own cache: theirs is paged (``cache`` "float32", "float16" or
        "bfloat16") and not bound to 1024 positions.  A prompt's whole pages are held once for its beams; from there each
        beam has its own for ``max_len`` tokens.  There may be as many sequences (prompts times beams) as one launch
        serves: 2^23 over the query heads, or over the head's slices of 2048 logits (599 thousand for Qwen2-0.5B);
        memory ends before, at 27 KB of logits a sequence."""
        xs = [x.numpy() if isinstance(x, DeviceArray) else np.asarray(x, np.float32) for x in prompts]
        if any(x.ndim != 2 or x.shape[1] != self.hidden or x.shape[0] < 1 for x in xs):
            raise ValueError(f"prompts are (T, {self.hidden}) embeddings")
        stop = (int(speech_token_size), min(int(speech_token_size) + 200, self.vocab))
        if max_len < 1 or not 1 <= page <= 65536 or not 1 <= beams <= 16 or not 0 < stop[0] < stop[1]:
            raise ValueError("generation takes at least one token, pages of 1 to 65536 keys, 1 to 16 beams, and stop ids "
                             "inside the vocabulary")
        if self.vocab - (stop[1] - stop[0] if min_len > 0 else 0) < beams:
            raise ValueError(f"the vocabulary has fewer tokens to choose from than {beams} beams")
        if len(xs) * beams > (2**23 - 1) // max(self.heads, -(-self.vocab // 2048)):
            raise ValueError(f"{len(xs)} prompts of {beams} beams are too many for one call")
        if not xs:
            return []
        r, w, dh = len(xs), int(beams), self.head_dim
        held = np.array([x.shape[0] for x in xs], np.int32)
        most = int(held.max()) + max_len
        cos, sin = (to_device(a) for a in rope_tables(dh, self.theta, most))
        own_h, pages = self._reserve(held, w, max_len - 1, page)           # the last token's key is not asked for
        blocks = own_h.shape[2]
        k, v = paged.new_cache(pages, self.kv_heads, page, dh, cache, layers=self.layers)
        own, tables = to_device(own_h), to_device(own_h)
        # the prompts: every token a row that sees its own sequence up to itself
        first = to_device(own_h[:, 0])
        _, slots, pos = self._slots(to_device(np.zeros(r, np.int32)), to_device(held), held, page, first)
        ends, every = np.cumsum(held, dtype=np.int64), np.concatenate(xs).astype(np.float32)
        last = DeviceArray((r * w, self.hidden))
        n = len(every)
        upto = np.concatenate([np.arange(1, m + 1, dtype=np.int32) for m in held]) if n <= min(_FEW_ROWS, _PROMPT_ROWS) else None
        if upto is not None and int(upto.sum()) * self.kv_heads * dh <= _FEW_NUMBERS:
            runs = [(0, n, self._paged_layers(to_device(every), pos, slots, to_device(np.repeat(own_h[:, 0], held, axis=0)),
                                              to_device(upto), cos, sin, k, v))]
        else:
            runs = self._ragged(lambda t0, t1: to_device(every[t0:t1]), np.zeros(r, np.int64), held, first, slots, pos, cos,
                                sin, k, v)
        for t0, t1, h in runs:
            for i in np.flatnonzero((ends > t0) & (ends <= t1)):
                for j in range(w):
                    _lib.call("copy_d2d", last.ptr + (int(i) * w + j) * self.hidden * 4,
                              h.ptr + int(ends[i] - 1 - t0) * self.hidden * 4, self.hidden * 4, None)
        logits = self._head(last)
        scores_h = np.full((r, w), -np.inf, np.float32)                    # at first one beam a prompt lives
        scores_h[:, 0] = 0.0
        scores, done = to_device(scores_h), to_device(np.zeros((r, w), np.uint8))
        chosen, parents = DeviceArray((r, w), np.int64), DeviceArray((r, w), np.int32)
        each = np.ones(r * w, np.int32)
        lengths, ones, x = to_device(np.repeat(held, w)), to_device(each), DeviceArray((r * w, self.hidden))
        trail = []
        for i in range(max_len):
            paged.beam_select(logits.reshape(r, w, self.vocab), scores, done, stop, stop if i < min_len else (0, 0),
                              out=(chosen, parents, scores, done))
            trail.append((chosen.numpy(), parents.numpy()))
            if i + 1 == max_len or done.numpy().all():
                break
            for r0 in range(0, r if w > 1 else 0, _TABLE_ROWS):
                r1 = min(r0 + _TABLE_ROWS, r)
                paged.beam_reorder(parents.rows(r0, r1), tables.rows(r0, r1), own.rows(r0, r1), (held + i)[r0:r1], k, v)
            self._embedded(chosen, x)
            lengths, slots, pos = self._slots(lengths, ones, each, page, own.reshape(r * w, blocks))
            h = self._paged_layers(x, pos, slots, tables.reshape(r * w, blocks), lengths, cos, sin, k, v)
            logits = self._head(h)
        best, out = scores.numpy(), []
        for i in range(r):
            tokens, b = [], 0
            for ids, up in reversed(trail):
                tokens.append(int(ids[i, b]))
                b = int(up[i, b])
            tokens.reverse()
            ends = [j for j, t in enumerate(tokens) if stop[0] <= t < stop[1]]
            out.append((tokens[:ends[0]] if ends else tokens, float(best[i, 0])))
        return out

    # -- given continuations of several prompts ----
    def score_batch(self, prompts, continuations, top: int = 0, page: int = 16, cache: str = "float32"):
        """What given speech tokens are worth after their prompts: for each of several prompts ((T, hidden) embeddings, of
        any lengths) a list of continuations, each a list of token ids.  Returns as many lists, of (logprobs (n,), entropy
        (n,), ids (n, top) int64, values (n, top)) a continuation: each token's log probability after all before it, the
        entropy in nats of the distribution that it comes from, and that one's ``top`` (0 to 32) best tokens with their
        log probabilities, best first.

        A prompt is run once; its continuations go on from its cache (whole pages shared, a part-filled last one copied
        for each), and the tokens of all of them are rows of the same passes over the weights.  The cache is as in
        ``generate_batch``; prompts and continuations are taken up to 4096 sequences and 524288 keys (whole pages) at a
        time, a prompt with one continuation at least, and a prompt whose continuations are more is run for each part."""
        xs = [x.numpy() if isinstance(x, DeviceArray) else np.asarray(x, np.float32) for x in prompts]
        if any(x.ndim != 2 or x.shape[1] != self.hidden or x.shape[0] < 1 for x in xs):
            raise ValueError(f"prompts are (T, {self.hidden}) embeddings")
        texts = [[np.asarray(c) for c in cs] for cs in continuations]
        if len(texts) != len(xs):
            raise ValueError(f"{len(texts)} lists of continuations for {len(xs)} prompts")
        known = min(self.vocab, self.emb.rows)
        for c in (c for cs in texts for c in cs):
            if c.ndim != 1 or c.size and (c.dtype.kind not in "iu" or int(c.min()) < 0 or int(c.max()) >= known):
                raise ValueError(f"continuations are lists of token ids below {known}")
        if not 0 <= top <= min(32, self.vocab) or not 1 <= page <= 65536:
            raise ValueError("scores take 0 to 32 alternatives and pages of 1 to 65536 keys")
        if cache not in ("float32", "float16", "bfloat16"):
            raise ValueError(f"a cache is float32, float16 or bfloat16, not {cache}")
        none = tuple(np.zeros(s, t) for s, t in ((0, np.float32), (0, np.float32), ((0, top), np.int64), ((0, top), np.float32)))
        out = [[none] * len(cs) for cs in texts]
        group, size, keys = [], 0, 0        # (prompt, its continuations) of one pass
        for i, cs in enumerate(texts):
            some, n, at = [j for j, c in enumerate(cs) if c.size], xs[i].shape[0], 0
            # keys of the pages that a continuation adds to its prompt's
            more = [(-(-(n + cs[j].size - 1) // page) - n // page) * page for j in some]
            held = -(-n // page) * page
            while at < len(some):
                if group and (size + 2 > _TABLE_ROWS or keys + held + more[at] > _SCORE_KEYS):
                    self._score_group(xs, texts, group, top, page, cache, out)
                    group, size, keys = [], 0, 0
                take, size, keys = [], size + 1, keys + held
                while at < len(some) and (not take or (size < _TABLE_ROWS and keys + more[at] <= _SCORE_KEYS)):
                    take.append(some[at])
                    at, size, keys = at + 1, size + 1, keys + more[at]
                group.append((i, take))
        if group:
            self._score_group(xs, texts, group, top, page, cache, out)
        return out

    def _score_group(self, xs, texts, group, top: int, page: int, cache: str, out):
        """score_batch of up to 4096 sequences: the prompts are the first rows of the tables, their continuations the
        others."""
        r, D = len(group), self.hidden
        of = np.array([p for p, (_, js) in enumerate(group) for _ in js], np.int32)      # each continuation's prompt
        ids = [texts[i][j].astype(np.int64) for i, js in group for j in js]
        held = np.array([xs[i].shape[0] for i, _ in group], np.int64)
        count = np.array([c.size for c in ids], np.int64)
        # what a continuation adds to the cache: all but its last token
        total = held[of] + count - 1
        pages = int((-(-held // page)).sum() + (-(-total // page) - held[of] // page).sum())
        cos, sin = (to_device(a) for a in rope_tables(self.head_dim, self.theta, int(total.max())))
        k, v = paged.new_cache(pages, self.kv_heads, page, self.head_dim, cache, layers=self.layers)
        n = r + len(ids)
        tables = to_device(np.full((n, int((-(-total // page)).max())), -1, np.int32))
        free = to_device(np.arange(pages, dtype=np.int32))
        row = 4 * D
        states = DeviceArray((int(count.sum()), D))         # the residual stream that each token is drawn from
        ends = np.cumsum(count)

        def run(lengths, before, new, taken, x, keep):
            lengths, taken, _, slots, pos = paged.block_tables(lengths, to_device(new.astype(np.int32)), page, free, taken,
                                                               tables, tokens=int(new.sum()))
            for t0, t1, h in self._ragged(x, before, new, tables, slots, pos, cos, sin, k, v) if new.any() else ():
                keep(t0, t1, h)
            return lengths, taken

        every = np.concatenate([xs[i] for i, _ in group]).astype(np.float32)
        last = np.cumsum(held) - 1

        def keep_last(t0, t1, h):
            for c in np.flatnonzero((last[of] >= t0) & (last[of] < t1)):
                _lib.call("copy_d2d", states.ptr + int(ends[c] - count[c]) * row, h.ptr + int(last[of[c]] - t0) * row, row, None)

        zero = np.zeros(n, np.int64)
        lengths, taken = run(to_device(zero.astype(np.int32)), zero, np.append(held, zero[r:]), to_device(np.zeros(1, np.int32)),
                             lambda t0, t1: to_device(every[t0:t1]), keep_last)
        taken = paged.fork(to_device(of), to_device(np.arange(r, n, dtype=np.int32)), tables, lengths, free, taken, k, v)
        fed = np.concatenate([c[:-1] for c in ids])
        at = np.cumsum(count - 1)                           # each continuation's end among the tokens that are fed

        def keep_all(t0, t1, h):
            for c in np.flatnonzero((at - count + 1 < t1) & (at > t0)):
                a, b = max(int(at[c] - count[c] + 1), t0), min(int(at[c]), t1)
                _lib.call("copy_d2d", states.ptr + int(ends[c] - (at[c] - a)) * row, h.ptr + (a - t0) * row, (b - a) * row, None)

        run(lengths, np.append(held, held[of]), np.append(zero[:r], count - 1), taken,
            lambda t0, t1: self._embedded(to_device(fed[t0:t1]), DeviceArray((t1 - t0, D))), keep_all)
        tokens, found = np.concatenate(ids), []
        for t0 in range(0, len(tokens), _PROMPT_ROWS):
            t1 = min(t0 + _PROMPT_ROWS, len(tokens))
            got = paged.token_logprobs(self._head(states.rows(t0, t1)), to_device(tokens[t0:t1]), top)
            found.append([g.numpy() for g in got])
        found = [np.concatenate(f) for f in zip(*found)]
        c = 0
        for i, js in group:
            for j in js:
                out[i][j] = tuple(f[ends[c] - count[c]:ends[c]].copy() for f in found)
                c += 1
