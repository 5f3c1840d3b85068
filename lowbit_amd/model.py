"""A device-resident decoder (Qwen2 / Llama architecture) on the fused GEMMs.

The reference runs this model in numpy with one ctypes GEMM per linear layer
(src/lowbit/model.py:300-470): every layer crosses the host boundary four
times. Here everything stays in HBM: token ids, activations, the KV cache, the
quantized weights (`to_device` handles) and the greedy argmax. Linear layers
call the library's GEMMs on device pointers (the decode kernels at one token,
the matrix-core kernels on t16 tiles for a prompt); the rest of a layer is the
library's decoder-layer kernels (`lbd_embed`, `lbd_rmsnorm`, `lbd_qkv_rope`,
`lbd_attention`, `lbd_swiglu`, `lbd_add`, `lbd_argmax`).

The decode position lives in device memory and the argmax writes the next token
id where the embedding lookup reads it, so one decode step is a fixed sequence
of launches: `generate` records it once as a HIP graph and replays it per token.

A one-token step (fused=True, the default) runs five launches per layer: each
linear layer is one fused GEMV (`lbd_gemv_*_fused`) whose prologue applies the
RMSNorm (q/k/v, gate/up, LM head) to its activation row and whose epilogue adds
the q/k/v bias or the residual in place, or (gate/up) writes the SwiGLU of each
gate/up output pair, so the down projection reads its activations ready-made;
the rotary embedding and the KV-cache write run inside the one-token attention,
which cuts each head's keys into slices on many compute units
(`lbd_attention_slices`) whose partial sums the o projection's prologue merges
(caches of more than 8 slices take `lbd_attention_decode_ws`, which merges in a
launch of its own); the LM head's epilogue folds the greedy argmax into a
64-bit key that `lbd_argmax_finalize` turns into the next token. Prompts (T > 1)
run the unfused sequence on the matrix-core GEMMs.

With a paged 8-bit cache (`new_cache(.., kv="e4m3")`, KV8Cache) the rotary embedding and
the cache write are `lbd_kv8_append` and the attention `lbd_kv8_attention`, in prompts
and steps alike; such a cache may hold several sequences, which `forward_batch` and
`generate_batch` run together.

Same architecture and arithmetic as the reference model: RMSNorm in fp32, q/k/v
projections concatenated along N and gate/up rows interleaved in (gate i, up i)
pairs (quantization is per output row, so no quantized value changes), rotary embedding in the "rotate_half"
convention from float32 cos/sin tables built in float64, grouped-query causal
attention with a KV cache, SwiGLU MLP, tied or untied LM head (quantized like
the other linears). Norm weights, biases, the embedding table and the KV cache
stay fp32. Backends: "w4a16", "w4a8", "mxfp4" (the reference's "fp32" backend is
numpy sgemm and has no counterpart here).
"""
from __future__ import annotations

import ctypes as C
import time
from dataclasses import dataclass

import numpy as np

from . import formats as F
from . import kernels as K

BACKENDS = ("w4a16", "w4a8", "mxfp4")
_KIND = {"w4a16": 0, "mxfp4": 1, "w4a8": 2}
ARGMAX_SLOTS = 1024  # LBD_ARGMAX_SLOTS of include/lowbit_hip.h


# ---------------------------------------------------------------- config (src/lowbit/model.py:42-77)

@dataclass
class ModelConfig:
    vocab_size: int
    hidden_size: int
    intermediate_size: int
    num_layers: int
    num_heads: int
    num_kv_heads: int
    head_dim: int
    rms_norm_eps: float = 1e-6
    rope_theta: float = 10000.0
    tie_word_embeddings: bool = False
    qkv_bias: bool = False
    max_position: int = 4096
    name: str = "custom"


def tiny_config(**over) -> ModelConfig:
    """The reference's test model shape (src/lowbit/model.py:483-489), overridable."""
    base = dict(vocab_size=97, hidden_size=256, intermediate_size=384, num_layers=2,
                num_heads=4, num_kv_heads=2, head_dim=64, rms_norm_eps=1e-6,
                rope_theta=10000.0, tie_word_embeddings=True, qkv_bias=True,
                max_position=256, name="tiny")
    base.update(over)
    return ModelConfig(**base)


def qwen2_config(**over) -> ModelConfig:
    """a Qwen2.5-0.5B-shaped decoder (hidden 896, 24 layers, 14 / 2
    heads, MLP 4864, vocab 151936, RMSNorm + RoPE, q/k/v bias, tied embeddings)."""
    base = dict(vocab_size=151936, hidden_size=896, intermediate_size=4864, num_layers=24,
                num_heads=14, num_kv_heads=2, head_dim=64, rms_norm_eps=1e-6,
                rope_theta=1000000.0, tie_word_embeddings=True, qkv_bias=True,
                max_position=32768, name="qwen2-0.5b-shape")
    base.update(over)
    return ModelConfig(**base)


def random_weights(cfg: ModelConfig, seed: int = 0, scale: float = 0.05, float32_draws: bool = False) -> dict:
    """Random weights under the checkpoint tensor names, drawn as the reference's test
    helper draws them (src/lowbit/model.py:492-513): N(0, scale^2), embeddings x20,
    norm weights 1 + N(0, scale^2). float32_draws=True draws float32 normals directly
    (same distribution, other values, several times faster at 0.5B parameters)."""
    rng = np.random.default_rng(seed)
    if float32_draws:
        r = lambda *s: rng.standard_normal(s, dtype=np.float32) * np.float32(scale)  # noqa: E731
    else:
        r = lambda *s: (rng.standard_normal(s) * scale).astype(np.float32)  # noqa: E731
    h, i, D = cfg.hidden_size, cfg.intermediate_size, cfg.head_dim
    W = {"model.embed_tokens.weight": r(cfg.vocab_size, h) * 20,
         "model.norm.weight": 1 + r(h)}
    for li in range(cfg.num_layers):
        p = f"model.layers.{li}."
        W[p + "input_layernorm.weight"] = 1 + r(h)
        W[p + "post_attention_layernorm.weight"] = 1 + r(h)
        for nm, n in (("q", cfg.num_heads * D), ("k", cfg.num_kv_heads * D),
                      ("v", cfg.num_kv_heads * D)):
            W[p + f"self_attn.{nm}_proj.weight"] = r(n, h)
            if cfg.qkv_bias:
                W[p + f"self_attn.{nm}_proj.bias"] = r(n)
        W[p + "self_attn.o_proj.weight"] = r(h, cfg.num_heads * D)
        W[p + "mlp.gate_proj.weight"] = r(i, h)
        W[p + "mlp.up_proj.weight"] = r(i, h)
        W[p + "mlp.down_proj.weight"] = r(h, i)
    if not cfg.tie_word_embeddings:
        W["lm_head.weight"] = r(cfg.vocab_size, h)
    return W


def rope_tables(head_dim: int, n_pos: int, theta: float) -> tuple[np.ndarray, np.ndarray]:
    """float32 cos / sin [n_pos, head_dim/2], angles in float64 (src/lowbit/model.py:195-198)."""
    inv = 1.0 / theta ** (np.arange(0, head_dim, 2, dtype=np.float64) / head_dim)
    ang = np.arange(n_pos, dtype=np.float64)[:, None] * inv[None]
    return np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)


# ---------------------------------------------------------------- device state

def _buf(nbytes: int) -> K.DeviceBuffer:
    return K.DeviceBuffer(max(16, int(nbytes)))


class KVCache:
    """Per-layer fp32 K and V [KV, capacity, D] in HBM; `length` tokens are valid."""

    def __init__(self, cfg: ModelConfig, capacity: int):
        if capacity > 16000:
            raise ValueError("KV cache capacity above 16000 positions")
        self.capacity = int(capacity)
        nb = cfg.num_kv_heads * self.capacity * cfg.head_dim * 4
        self.k = [_buf(nb) for _ in range(cfg.num_layers)]
        self.v = [_buf(nb) for _ in range(cfg.num_layers)]
        self.length = 0
        # partial sums of the one-token attention's key slices (the layers use it
        # in turn on the model's stream)
        wb = K.lib().lbd_attention_decode_work_bytes(cfg.num_heads, cfg.head_dim, self.capacity)
        self.attn_work = _buf(wb)
        # the o projection's prologue merges up to 8 slices of 4096 / head_dim keys
        # over rows of at most 2048 elements; longer caches take the merge launch
        slices = wb // (cfg.num_heads * (cfg.head_dim + 4) * 4)
        self.fused_merge = slices <= 8 and cfg.num_heads * cfg.head_dim <= 2048


class KV8Cache:
    """K and V of one or more sequences in pages of a shared pool, 8 bits an element (E4M3
    codes, an E8M0 exponent for each page and KV head; lbd_kv8_* of include/lowbit_hip.h):
    a quarter of KVCache's bytes, no bound of 16000 positions, and sequences take pages as
    they grow. `lengths[s]` tokens of sequence s are valid. `capacity` positions a sequence;
    `pages` in the pool (default: enough for every sequence at its capacity)."""

    def __init__(self, cfg: ModelConfig, capacity: int, sequences: int = 1, page: int = 32, pages: int | None = None):
        if capacity <= 0 or sequences <= 0 or (pages is not None and pages <= 0):
            raise ValueError("capacity, sequences and pages must be positive")
        if page not in (16, 32, 64, 128):
            raise ValueError("pages hold 16, 32, 64 or 128 tokens")
        if cfg.head_dim not in (32, 64, 128):
            raise ValueError("the 8-bit cache takes heads of 32, 64 or 128")
        self.capacity, self.page = int(capacity), int(page)
        self.max_pages = -(-self.capacity // self.page)
        self.pages = int(sequences * self.max_pages if pages is None else pages)
        kv, d = cfg.num_kv_heads, cfg.head_dim
        codes, exps = self.pages * kv * self.page * d, self.pages * kv
        self.layers = []  # (lbd_kv8_pool, its buffers) of each layer; the layers share the page table
        for _ in range(cfg.num_layers):
            b = [_buf(codes), _buf(codes), _buf(exps), _buf(exps)]
            self.layers.append((K.LbdKv8Pool(*(x.ptr for x in b), self.pages, self.page, kv, d), b))
        self.lengths = np.zeros(sequences, np.int64)
        self._held = np.zeros(sequences, np.int64)  # pages of each sequence
        self._free = list(range(self.pages - 1, -1, -1))
        self._table = np.full((sequences, self.max_pages), -1, np.int32)
        self._dirty = True
        self.table = _buf(self._table.nbytes)
        self.past, self.q_start = _buf(4 * sequences), _buf(4 * (sequences + 1))
        self.one = K.DeviceBuffer.from_array(np.array([0, 1], np.int32))  # q_start of a one-token step
        self.work = _buf(16)

    @property
    def length(self) -> int:
        """Valid tokens of a cache of one sequence."""
        if len(self.lengths) != 1:
            raise ValueError("a cache of several sequences has lengths, not one length")
        return int(self.lengths[0])

    @length.setter
    def length(self, n: int):
        if len(self.lengths) != 1:
            raise ValueError("a cache of several sequences has lengths, not one length")
        self.truncate(0, n)

    def truncate(self, seq: int, n: int = 0):
        """Sequence `seq` keeps its first n tokens (pages past them return to the pool). The page that
        the last of them lies in keeps its blocks' exponents: tokens that are appended to it later
        are rounded in the unit that the dropped ones called for, and a block that a dropped token
        made NaN stays NaN until the page is begun again (n a multiple of the page: at once)."""
        if not 0 <= n <= self.lengths[seq]:
            raise ValueError(f"sequence {seq} does not hold {n} tokens")
        self.commit(seq, n)

    def commit(self, seq: int, n: int):
        """The first n positions of sequence `seq` hold its tokens, as a pass over positions that reserve
        gave it has written them (pages past them return to the pool)."""
        keep = -(-int(n) // self.page)
        if n < 0 or keep > self._held[seq]:
            raise ValueError(f"sequence {seq} has no pages for {n} tokens")
        gone = self._table[seq, keep:self._held[seq]]
        self._free.extend(int(p) for p in gone[::-1])
        if len(gone):
            gone[:] = -1
            self._dirty = True
        self._held[seq], self.lengths[seq] = keep, n

    def reserve(self, seq: int, n: int):
        """Pages for the first n positions of sequence `seq`."""
        if n > self.capacity:
            raise ValueError(f"KV cache full ({n} > {self.capacity})")
        need, has = -(-int(n) // self.page), int(self._held[seq])
        if need - has > len(self._free):
            raise ValueError(f"KV cache full (no {need - has} pages left for sequence {seq})")
        for i in range(has, need):
            self._table[seq, i] = self._free.pop()
            self._dirty = True
        self._held[seq] = max(need, has)

    def upload(self):
        """The page table to the device, where it changed."""
        if self._dirty:
            _check(K.lib().lb_memcpy_h2d(self.table.ptr, self._table.ctypes.data, self._table.nbytes), "table upload")
            self._dirty = False

    def batch(self, q_start: int, past: int, seqs: int, max_new: int, rows: int) -> K.LbdKv8Batch:
        """The lbd_kv8_batch of the first `seqs` sequences (room: the workspace that its attention takes)."""
        return K.LbdKv8Batch(q_start, past, self.table.ptr, seqs, self.max_pages, max_new, rows)

    def room(self, b: K.LbdKv8Batch, heads: int):
        """Grow `work` to what the attention of this batch takes (no call may be in flight)."""
        need = K.lib().lbd_kv8_attention_work_bytes(C.byref(self.layers[0][0]), C.byref(b), heads)
        if need > self.work.nbytes:
            self.work = _buf(need)


@dataclass
class _Layer:
    ln1: K.DeviceBuffer
    qkv: object
    qkv_bias: K.DeviceBuffer | None
    o: object
    ln2: K.DeviceBuffer
    gate_up: object
    down: object


def _check(rc: int, what: str) -> int:
    if rc < 0:
        K._err(rc, what)
    return rc


class Model:
    """Device-resident decoder with the reference Model's constructor and calls
    (src/lowbit/model.py:300-470): `forward(tokens, cache, logits)` and greedy
    `generate(prompt, n_new, cache, timings)`."""

    def __init__(self, cfg: ModelConfig, weights: dict, backend: str = "w4a8", asym: bool = False,
                 quantize_lm_head: bool = True, int4_scale: str = "absmax", max_tokens: int = 512,
                 quantize_on_device: bool = True, fused: bool = True):
        if backend not in BACKENDS:
            raise ValueError(f"backend must be one of {BACKENDS}")
        if not quantize_lm_head:
            raise ValueError("the LM head is quantized like the other linears on the device")
        blk = F.MXBLOCK if backend == "mxfp4" else F.GROUP
        for k in (cfg.hidden_size, cfg.intermediate_size, cfg.num_heads * cfg.head_dim):
            if k % blk:
                raise ValueError(f"layer width {k} is not a multiple of the {backend} block ({blk})")
        self.cfg, self.backend, self.asym = cfg, backend, asym
        self.L = K.lib()
        s = C.c_void_p()
        _check(self.L.lb_stream_create(C.byref(s)), "stream")
        self.stream = s.value
        g = lambda n: np.ascontiguousarray(weights[n], np.float32)  # noqa: E731
        up = K.DeviceBuffer.from_array

        def lin(w):
            # the device packers write the host packers' bytes; packing on the device
            # only saves the host time (seconds per 100M weights)
            if quantize_on_device:
                if backend == "mxfp4":
                    return K.quantize_mxfp4_device(w)
                return K.quantize_int4_device(w, asym=asym, scale=int4_scale)
            wq = F.quantize_mxfp4(w) if backend == "mxfp4" else F.quantize_int4(w, asym=asym, scale=int4_scale)
            return K.to_device(wq)

        self.embed = up(g("model.embed_tokens.weight"))
        self.layers: list[_Layer] = []
        for i in range(cfg.num_layers):
            p = f"model.layers.{i}."
            a = p + "self_attn."
            wqkv = np.concatenate([g(a + "q_proj.weight"), g(a + "k_proj.weight"), g(a + "v_proj.weight")], 0)
            bqkv = (np.concatenate([g(a + "q_proj.bias"), g(a + "k_proj.bias"), g(a + "v_proj.bias")])
                    if cfg.qkv_bias else None)
            # row 2i: gate i, row 2i + 1: up i (the pairs of the glu epilogue)
            wgu = np.stack([g(p + "mlp.gate_proj.weight"), g(p + "mlp.up_proj.weight")], 1).reshape(
                2 * cfg.intermediate_size, -1)
            self.layers.append(_Layer(up(g(p + "input_layernorm.weight")), lin(wqkv),
                                      None if bqkv is None else up(bqkv), lin(g(a + "o_proj.weight")),
                                      up(g(p + "post_attention_layernorm.weight")), lin(wgu),
                                      lin(g(p + "mlp.down_proj.weight"))))
        self.norm = up(g("model.norm.weight"))
        head = (g("model.embed_tokens.weight") if cfg.tie_word_embeddings or "lm_head.weight" not in weights
                else g("lm_head.weight"))
        self.lm_head = lin(head)
        cos, sin = rope_tables(cfg.head_dim, cfg.max_position, cfg.rope_theta)
        self.cos, self.sin = up(cos), up(sin)
        self._alloc(max_tokens)
        self.tok = _buf(4 * max(max_tokens, 1))
        self.pos = _buf(4)
        self.hist: K.DeviceBuffer | None = None
        # argmax key slots of the fused LM head; lbd_argmax_finalize clears them
        self.key = _buf(8 * ARGMAX_SLOTS)
        _check(self.L.lb_memset_d(self.key.ptr, 0, 8 * ARGMAX_SLOTS), "key clear")
        # one-token steps fuse when every linear takes the small-M kernels and the
        # attention shape fits the one-token kernel
        D = cfg.head_dim
        widths = {cfg.hidden_size, cfg.intermediate_size, cfg.num_heads * D}
        prm = K._Params(-1, 0, 0, 0, 0, 0, 0)
        self.fused = bool(fused) and D in (32, 64, 128) and cfg.num_heads // cfg.num_kv_heads <= 16 and all(
            self.L.lbd_gemm_path(_KIND[backend], 1, k, C.byref(prm)) == K.ISA_GFX950 for k in widths)

    # ------------------------------------------------------------ buffers

    def _alloc(self, T: int):
        cfg = self.cfg
        h, I, D = cfg.hidden_size, cfg.intermediate_size, cfg.head_dim
        qkvw = (cfg.num_heads + 2 * cfg.num_kv_heads) * D
        self.tmax = T
        self.x, self.h, self.o = _buf(T * h * 4), _buf(T * h * 4), _buf(T * h * 4)
        self.qkv, self.att = _buf(T * qkvw * 4), _buf(T * cfg.num_heads * D * 4)
        self.gu, self.m = _buf(T * 2 * I * 4), _buf(T * I * 4)
        self.logits = _buf(cfg.vocab_size * 4)
        kmax = max(h, I, cfg.num_heads * D)
        # room for the K split of the bf16x3 prefill GEMMs (rows of 8192+ elements), so
        # the model's matrix-core GEMMs are the launches lb.gemm_* and bench.py time
        kind = 1 if self.backend == "mxfp4" else 0
        lin = [w for ly in self.layers for w in (ly.qkv, ly.o, ly.gate_up, ly.down)] + [self.lm_head]
        split = max(self.L.lbd_bf16x3_workspace_bytes_split(kind, T, w.n, w.kp) for w in lin)
        self.ws = _buf(max(self.L.lbd_w4a8_workspace_bytes(T, kmax), self.L.lbd_bf16x3_workspace_bytes(T, kmax),
                           split))

    @property
    def linear_weight_bytes(self) -> int:
        return sum(x.nbytes for L in self.layers for x in (L.qkv, L.o, L.gate_up, L.down)) + self.lm_head.nbytes

    def new_cache(self, max_len: int, kv: str = "fp32", sequences: int = 1, page: int = 32,
                  pages: int | None = None) -> "KVCache | KV8Cache":
        """A cache of max_len positions: kv="fp32" (one sequence), or kv="e4m3", the paged 8-bit
        cache of `sequences` sequences (KV8Cache)."""
        if kv == "fp32":
            if sequences != 1 or pages is not None:
                raise ValueError("the fp32 cache holds one sequence, without pages")
            return KVCache(self.cfg, max_len)
        if kv != "e4m3":
            raise ValueError(f"kv must be 'fp32' or 'e4m3', not {kv!r}")
        return KV8Cache(self.cfg, max_len, sequences, page, pages)

    # ------------------------------------------------------------ one step

    def _linear(self, w, x: int, m: int, y: int):
        """y[m, n] = x[m, k] . w^T on the stream: decode kernels on the row-major
        copy, or the matrix-core kernels on the t16 copy (repacked on first use)."""
        L, prm = self.L, K._Params(-1, 0, 0, 0, 0, 0, 0)
        mfma = _check(L.lbd_gemm_path(_KIND[self.backend], m, w.kp, C.byref(prm)), "lbd_gemm_path") \
            == K.ISA_GFX950_MFMA
        s, ws = self.stream, self.ws
        if self.backend == "mxfp4":
            if mfma:
                qwt, et = w.tiles()
                rc = L.lbd_gemm_mxfp4_t16(x, m, w.kp, qwt.ptr, et.ptr, w.n, y, C.byref(prm), ws.ptr, ws.nbytes, s)
            else:
                rc = L.lbd_gemm_mxfp4(x, m, w.kp, w.qw.ptr, w.e8m0.ptr, w.n, y, C.byref(prm), s)
        else:
            zp = None if w.zeros is None else w.zeros.ptr
            if mfma and self.backend == "w4a16":
                rc = K.gemm_w4a16_tiles(w, x, m, y, prm, ws.ptr, ws.nbytes, s)
            elif mfma:
                qwt, st, zt = w.tiles()
                rc = L.lbd_gemm_w4a8_t16(x, m, w.kp, qwt.ptr, st.ptr, None if zt is None else zt.ptr, w.n, y,
                                         C.byref(prm), ws.ptr, ws.nbytes, s)
            elif self.backend == "w4a16":
                rc = L.lbd_gemm_w4a16(x, m, w.kp, w.qw.ptr, w.scales.ptr, zp, w.n, y, C.byref(prm), s)
            else:
                rc = L.lbd_gemm_w4a8(x, m, w.kp, w.qw.ptr, w.scales.ptr, zp, w.n, y, C.byref(prm), ws.ptr,
                                     ws.nbytes, s)
        _check(rc, f"{self.backend} linear")

    def _fused_linear(self, w, x: int | None, y: int, norm: int | None = None, glu: bool = False,
                      bias: int | None = None, res: int | None = None, key: int | None = None,
                      attn: tuple | None = None):
        """y[0, n] = res[n] + (act(x) . w^T)[n] + bias[n] for one token, one launch;
        act is the RMSNorm with weights `norm` (or the identity). With glu the rows
        of w are (gate, up) pairs and y[0, p] = silu(gate) * up of pair p. With
        attn = (partials, cache capacity) the activation row is the one-token
        attention merged from its key-slice partials (x unused)."""
        part, cap = attn if attn else (None, 0)
        f = K.LbdFusion(norm, self.cfg.rms_norm_eps if norm else 0.0, 0, bias, res, key, int(glu), part, cap,
                        self.cfg.head_dim if attn else 0)
        L, s = self.L, self.stream
        if self.backend == "mxfp4":
            rc = L.lbd_gemv_mxfp4_fused(x, 1, w.kp, w.qw.ptr, w.e8m0.ptr, w.n, y, C.byref(f), s)
        else:
            zp = None if w.zeros is None else w.zeros.ptr
            fn = L.lbd_gemv_w4a16_fused if self.backend == "w4a16" else L.lbd_gemv_w4a8_fused
            rc = fn(x, 1, w.kp, w.qw.ptr, w.scales.ptr, zp, w.n, y, C.byref(f), s)
        _check(rc, f"fused {self.backend} linear")

    def _step_fused(self, cache: KVCache, logits: str, argmax_hist: bool):
        """Enqueue one forward of the single token in self.tok at position *pos,
        five launches per layer."""
        cfg, L, s = self.cfg, self.L, self.stream
        h, H, KV, D = cfg.hidden_size, cfg.num_heads, cfg.num_kv_heads, cfg.head_dim
        x = self.x.ptr
        _check(L.lbd_embed(self.embed.ptr, cfg.vocab_size, h, self.tok.ptr, 1, x, s), "embed")
        for li, ly in enumerate(self.layers):
            self._fused_linear(ly.qkv, x, self.qkv.ptr, norm=ly.ln1.ptr,
                               bias=None if ly.qkv_bias is None else ly.qkv_bias.ptr)
            if isinstance(cache, KV8Cache):
                self._attend_kv8(cache, li, None)
                self._fused_linear(ly.o, self.att.ptr, x, res=x)
            elif cache.fused_merge:
                # key slices, merged in the o projection's prologue
                _check(L.lbd_attention_slices(self.qkv.ptr, H, KV, D, self.cos.ptr, self.sin.ptr, self.pos.ptr,
                                              cfg.max_position, cache.k[li].ptr, cache.v[li].ptr, cache.capacity,
                                              cache.attn_work.ptr, cache.attn_work.nbytes, s), "attention slices")
                self._fused_linear(ly.o, None, x, res=x, attn=(cache.attn_work.ptr, cache.capacity))
            else:
                _check(L.lbd_attention_decode_ws(self.qkv.ptr, H, KV, D, self.cos.ptr, self.sin.ptr, self.pos.ptr,
                                                 cfg.max_position, cache.k[li].ptr, cache.v[li].ptr, cache.capacity,
                                                 self.att.ptr, cache.attn_work.ptr, cache.attn_work.nbytes, s),
                       "attention decode")
                self._fused_linear(ly.o, self.att.ptr, x, res=x)
            self._fused_linear(ly.gate_up, x, self.m.ptr, norm=ly.ln2.ptr, glu=True)
            self._fused_linear(ly.down, self.m.ptr, x, res=x)
        if logits == "none":
            _check(L.lbd_rmsnorm(x, self.norm.ptr, 1, h, cfg.rms_norm_eps, self.h.ptr, s), "rmsnorm")
        elif logits == "last":
            key = self.key.ptr if argmax_hist else None
            self._fused_linear(self.lm_head, x, self.logits.ptr, norm=self.norm.ptr, key=key)
            if argmax_hist:
                hist = self.hist.ptr if self.hist is not None else None
                n = self.hist.nbytes // 4 if self.hist is not None else 0
                _check(L.lbd_argmax_finalize(self.key.ptr, self.tok.ptr, self.pos.ptr, 1, hist, n, s),
                       "argmax finalize")
        else:
            self._fused_linear(self.lm_head, x, self.all_logits.ptr, norm=self.norm.ptr)

    def _attend_kv8(self, cache: KV8Cache, li: int, bias: int | None):
        """Layer li's append of the rows in self.qkv (rotated in place) and their attention, by the
        batch that _plan_kv8 or forward_batch left in self.batch."""
        cfg, L, s = self.cfg, self.L, self.stream
        H, D = cfg.num_heads, cfg.head_dim
        width, pool, b = (H + 2 * cfg.num_kv_heads) * D, C.byref(cache.layers[li][0]), C.byref(self.batch)
        _check(L.lbd_kv8_append(pool, b, self.qkv.ptr, width, bias, H, self.cos.ptr, self.sin.ptr, cfg.max_position,
                                self.qkv.ptr, width, s), "kv8 append")
        _check(L.lbd_kv8_attention(pool, b, self.qkv.ptr, width, H, self.att.ptr, H * D, cache.work.ptr,
                                   cache.work.nbytes, s), "kv8 attention")

    def _plan_kv8(self, cache, T: int):
        """The batch of T tokens of a one-sequence 8-bit cache at position *pos."""
        if not isinstance(cache, KV8Cache):
            return
        q_start = cache.one
        if T > 1:
            a, q_start = np.array([0, T], np.int32), cache.q_start
            _check(self.L.lb_memcpy_h2d(q_start.ptr, a.ctypes.data, 8), "q_start upload")
        self.batch = cache.batch(q_start.ptr, self.pos.ptr, 1, T, T)
        cache.room(self.batch, self.cfg.num_heads)

    def _layers(self, T: int, cache):
        """The T tokens in self.tok through every layer and the last norm, into self.h."""
        cfg, L, s = self.cfg, self.L, self.stream
        h, I, H, KV, D = cfg.hidden_size, cfg.intermediate_size, cfg.num_heads, cfg.num_kv_heads, cfg.head_dim
        qkvw = (H + 2 * KV) * D
        _check(L.lbd_embed(self.embed.ptr, cfg.vocab_size, h, self.tok.ptr, T, self.x.ptr, s), "embed")
        for li, ly in enumerate(self.layers):
            _check(L.lbd_rmsnorm(self.x.ptr, ly.ln1.ptr, T, h, cfg.rms_norm_eps, self.h.ptr, s), "rmsnorm")
            self._linear(ly.qkv, self.h.ptr, T, self.qkv.ptr)
            bias = None if ly.qkv_bias is None else ly.qkv_bias.ptr
            if isinstance(cache, KV8Cache):
                self._attend_kv8(cache, li, bias)
            else:
                _check(L.lbd_qkv_rope(self.qkv.ptr, bias, T, H, KV, D, self.cos.ptr, self.sin.ptr, self.pos.ptr,
                                      cfg.max_position, cache.k[li].ptr, cache.v[li].ptr, cache.capacity, s),
                       "qkv rope")
                _check(L.lbd_attention(self.qkv.ptr, qkvw, cache.k[li].ptr, cache.v[li].ptr, T, H, KV, D,
                                       self.pos.ptr, cache.capacity, self.att.ptr, s), "attention")
            self._linear(ly.o, self.att.ptr, T, self.o.ptr)
            _check(L.lbd_add(self.x.ptr, self.o.ptr, T * h, s), "add")
            _check(L.lbd_rmsnorm(self.x.ptr, ly.ln2.ptr, T, h, cfg.rms_norm_eps, self.h.ptr, s), "rmsnorm")
            self._linear(ly.gate_up, self.h.ptr, T, self.gu.ptr)
            _check(L.lbd_swiglu_pairs(self.gu.ptr, T, I, self.m.ptr, s), "swiglu")
            self._linear(ly.down, self.m.ptr, T, self.o.ptr)
            _check(L.lbd_add(self.x.ptr, self.o.ptr, T * h, s), "add")
        _check(L.lbd_rmsnorm(self.x.ptr, self.norm.ptr, T, h, cfg.rms_norm_eps, self.h.ptr, s), "rmsnorm")

    def _step(self, T: int, cache: KVCache, logits: str, argmax_hist: bool):
        """Enqueue one forward of the T tokens in self.tok at position *pos."""
        if T == 1 and self.fused:
            return self._step_fused(cache, logits, argmax_hist)
        cfg, L, s = self.cfg, self.L, self.stream
        h = cfg.hidden_size
        self._layers(T, cache)
        if logits == "none":
            return
        if logits == "last":
            self._linear(self.lm_head, self.h.ptr + (T - 1) * h * 4, 1, self.logits.ptr)
            if argmax_hist:
                hist = self.hist.ptr if self.hist is not None else None
                n = self.hist.nbytes // 4 if self.hist is not None else 0
                _check(L.lbd_argmax(self.logits.ptr, cfg.vocab_size, self.tok.ptr, self.pos.ptr, T, hist, n, s),
                       "argmax")
        else:
            self._linear(self.lm_head, self.h.ptr, T, self.all_logits.ptr)

    def _tokens(self, tokens) -> np.ndarray:
        """int32 ids as numpy indexing reads them: negatives count from the end,
        anything outside [-vocab, vocab) raises IndexError (src/lowbit/model.py:398)."""
        t = np.asarray(tokens, np.int64).reshape(-1)
        if t.size == 0:
            raise ValueError("no tokens")
        V = self.cfg.vocab_size
        if (t.min() < -V or t.max() >= V):
            raise IndexError(f"token id out of range for a vocabulary of {V}")
        return np.ascontiguousarray(np.where(t < 0, t + V, t), np.int32)

    def _set_pos(self, p: int):
        a = np.array([p], np.int32)
        _check(self.L.lb_memcpy_h2d(self.pos.ptr, a.ctypes.data, 4), "pos upload")

    @staticmethod
    def _set_length(cache, n: int):
        """A one-sequence cache after a pass that has written its first n tokens."""
        if isinstance(cache, KV8Cache):
            cache.commit(0, n)
        else:
            cache.length = n

    def _sync(self):
        _check(self.L.lb_stream_synchronize(self.stream), "synchronize")

    # ------------------------------------------------------------ public calls

    def forward(self, tokens, cache: KVCache | None = None, logits: str = "last") -> np.ndarray:
        """Run tokens [T] at positions cache.length.. (0 without a cache); logits="last"
        returns [V], "all" [T, V], "none" the final hidden states [T, hidden]
        (src/lowbit/model.py:380-435)."""
        cfg = self.cfg
        tokens = self._tokens(tokens)
        T = int(tokens.shape[0])
        own = cache is None
        cache = cache or self.new_cache(T)
        pos = cache.length
        if pos + T > cache.capacity:
            raise ValueError(f"KV cache full ({pos}+{T} > {cache.capacity})")
        if T > self.tmax:
            self._alloc(T)
            self.tok = _buf(4 * T)
        self._sync()
        if isinstance(cache, KV8Cache):
            cache.reserve(0, pos + T)
            cache.upload()
            self._plan_kv8(cache, T)
        _check(self.L.lb_memcpy_h2d(self.tok.ptr, tokens.ctypes.data, 4 * T), "token upload")
        self._set_pos(pos)
        if logits == "all":
            self.all_logits = _buf(T * cfg.vocab_size * 4)
        self._step(T, cache, logits, argmax_hist=False)
        self._sync()
        if not own:
            self._set_length(cache, pos + T)
        if logits == "last":
            return self.logits.to_array((cfg.vocab_size,), np.float32)
        if logits == "all":
            return self.all_logits.to_array((T, cfg.vocab_size), np.float32)
        return self.h.to_array((T, cfg.hidden_size), np.float32)

    def generate(self, prompt, n_new: int, cache: KVCache | None = None, timings: dict | None = None,
                 graph: bool = True) -> list[int]:
        """Greedy decoding: prefill the prompt, then n_new tokens one at a time
        (src/lowbit/model.py:437-458): n_new tokens come out of one prefill and
        n_new - 1 decode forwards. The argmax runs on the device and feeds the next
        step's embedding lookup; the decode steps replay one recorded HIP graph
        (graph=False launches them one by one). timings["decode_s"] includes the
        recording of the graph."""
        prompt = self._tokens(prompt)
        T = len(prompt)
        steps = max(0, n_new - 1)
        cache = cache or self.new_cache(T + n_new)
        start = cache.length
        if start + T + steps > cache.capacity:
            raise ValueError(f"KV cache full ({start}+{T}+{steps} > {cache.capacity})")
        if T > self.tmax:
            self._alloc(T)
            self.tok = _buf(4 * T)
        # hist[p] = the token generated at position p - 1; the last one lands at start + T + steps
        self.hist = _buf(4 * (cache.capacity + 1))
        L = self.L
        self._sync()
        if isinstance(cache, KV8Cache):  # the whole answer's pages, so that the recorded step never changes
            cache.reserve(0, start + T + steps)
            cache.upload()
            self._plan_kv8(cache, T)
        _check(L.lb_memcpy_h2d(self.tok.ptr, prompt.ctypes.data, 4 * T), "token upload")
        self._set_pos(start)
        t0 = time.perf_counter()
        self._step(T, cache, "last", argmax_hist=True)
        self._sync()
        t1 = time.perf_counter()
        if steps:
            self._plan_kv8(cache, 1)
        if steps and graph:
            # every linear of a one-token step takes the decode kernels (M = 1),
            # which allocate nothing, so the step can be recorded
            s, ex = self.stream, C.c_void_p()
            _check(L.lb_stream_begin_capture(s), "begin capture")
            try:
                self._step(1, cache, "last", argmax_hist=True)
            finally:
                _check(L.lb_stream_end_capture(s, C.byref(ex)), "end capture")
            try:
                for _ in range(steps):
                    _check(L.lb_graph_launch(ex.value, s), "graph launch")
                self._sync()
            finally:
                L.lb_graph_destroy(ex.value)
        else:
            for _ in range(steps):
                self._step(1, cache, "last", argmax_hist=True)
            self._sync()
        t2 = time.perf_counter()
        self._set_length(cache, start + T + steps)
        out = self.hist.to_array((cache.capacity + 1,), np.int32)[start + T:start + T + n_new]
        if timings is not None:
            timings["prefill_s"] = t1 - t0
            timings["decode_s"] = t2 - t1
            timings["decode_forwards"] = steps
        return [int(v) for v in out]

    # ------------------------------------------------------------ several sequences

    def forward_batch(self, tokens: list, cache: KV8Cache) -> np.ndarray:
        """Run tokens[s] (possibly none) of each sequence s of an 8-bit cache behind what it holds:
        prompts, chunks of prompts and single tokens in one pass. Returns the logits [S, V] of each
        sequence's last token; rows of sequences without tokens are NaN."""
        cfg, L = self.cfg, self.L
        S = len(cache.lengths) if isinstance(cache, KV8Cache) else -1
        if len(tokens) != S:
            raise ValueError("forward_batch takes a KV8Cache and a list of tokens for each of its sequences")
        rows = [self._tokens(t) if len(t) else np.zeros(0, np.int32) for t in tokens]
        news = np.array([len(r) for r in rows])
        T, last = int(news.sum()), int(news.max(initial=0))
        if T == 0:
            raise ValueError("no tokens")
        try:
            for i in range(S):
                cache.reserve(i, int(cache.lengths[i] + news[i]))
        except ValueError:
            for i in range(S):  # what the others had taken goes back
                cache.commit(i, int(cache.lengths[i]))
            raise
        self._sync()
        if max(T, S) > self.tmax:
            self._alloc(max(T, S))
            self.tok = _buf(4 * max(T, S))
        cache.upload()
        starts = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
        ends = np.where(news > 0, starts[1:] - 1, 0).astype(np.int32)
        past, tok = cache.lengths.astype(np.int32), np.concatenate(rows).astype(np.int32)
        for buf, a in ((cache.q_start, starts), (cache.past, past), (self.tok, tok)):
            _check(L.lb_memcpy_h2d(buf.ptr, a.ctypes.data, a.nbytes), "batch upload")
        self.batch = cache.batch(cache.q_start.ptr, cache.past.ptr, S, last, T)
        cache.room(self.batch, cfg.num_heads)
        self._layers(T, cache)
        # the sequences' last rows, gathered, through the LM head
        index, rows_h = K.DeviceBuffer.from_array(ends), _buf(S * cfg.hidden_size * 4)
        out = _buf(S * cfg.vocab_size * 4)
        _check(L.lbd_embed(self.h.ptr, T, cfg.hidden_size, index.ptr, S, rows_h.ptr, self.stream), "row gather")
        self._linear(self.lm_head, rows_h.ptr, S, out.ptr)
        self._sync()
        cache.lengths += news
        y = out.to_array((S, cfg.vocab_size), np.float32)
        y[news == 0] = np.nan
        return y

    def generate_batch(self, prompts: list, n_new: int, cache: KV8Cache | None = None) -> list[list[int]]:
        """Greedy decoding of several prompts together: all prompts in one pass, then one token of
        every sequence a pass (the argmax on the host)."""
        if not len(prompts) or not all(len(p) for p in prompts):
            raise ValueError("no tokens")
        if n_new <= 0:
            return [[] for _ in prompts]
        if cache is None:
            cache = self.new_cache(max(len(p) for p in prompts) + n_new, kv="e4m3", sequences=len(prompts))
        out = [[] for _ in prompts]
        y = self.forward_batch(list(prompts), cache)
        for i in range(n_new):
            tok = y.argmax(1)
            for o, v in zip(out, tok):
                o.append(int(v))
            if i + 1 < n_new:
                y = self.forward_batch([[int(v)] for v in tok], cache)
        return out
