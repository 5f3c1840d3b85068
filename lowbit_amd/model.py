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
`generate_batch` run together. With ModelConfig.window the attention sees a sliding window and
the first `sinks` positions (`lbd_kv8_attention_window`, on such a cache only), and pages
behind the window go back to the pool. `generate_beams` searches with beams: a prompt's beams
are sequences of one cache that share their pages (`lbd_beam_select`, `lbd_kv8_reorder`).

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
    window: int = 0  # positions that a token sees, itself among them; 0: all (no reference counterpart)
    sinks: int = 0   # with a window: first positions that stay visible


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
        if cfg.window:
            raise ValueError("a sliding window takes the 8-bit cache (kv='e4m3')")
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


def _pages_at(n, page: int, cfg):
    """Pages that a sequence of n tokens (an array) holds while its next one is written: with a window those that it
    sees. `cfg`: what has `window` and `sinks`."""
    first, last = -(-cfg.sinks // page), n // page + 1
    return last - (np.maximum(np.maximum(n - cfg.window + 1, 0) // page - first, 0) if cfg.window else 0)


class KV8Cache:
    """K and V of one or more sequences in pages of a shared pool, 8 bits an element (E4M3
    codes, an E8M0 exponent for each page and KV head; lbd_kv8_* of include/lowbit_hip.h):
    a quarter of KVCache's bytes, no bound of 16000 positions, and sequences take pages as
    they grow. `lengths[s]` tokens of sequence s are valid. `capacity` positions a sequence;
    `pages` in the pool (default: enough for every sequence at its capacity).

    Sequences may share pages (`fork`): a page belongs to all that hold it, and the first that is
    about to write to one that others hold takes a copy. With a window pages that no later token
    sees go back to the pool (`slide`)."""

    def __init__(self, cfg: ModelConfig, capacity: int, sequences: int = 1, page: int = 32, pages: int | None = None):
        if capacity <= 0 or sequences <= 0 or (pages is not None and pages <= 0):
            raise ValueError("capacity, sequences and pages must be positive")
        if page not in (16, 32, 64, 128):
            raise ValueError("pages hold 16, 32, 64 or 128 tokens")
        if cfg.head_dim not in (32, 64, 128):
            raise ValueError("the 8-bit cache takes heads of 32, 64 or 128")
        self.capacity, self.page = int(capacity), int(page)
        self.window, self.sinks = int(cfg.window), int(cfg.sinks)
        self.max_pages = -(-self.capacity // self.page)
        self.pages = int(sequences * self.max_pages if pages is None else pages)
        self._kv, self._d = cfg.num_kv_heads, cfg.head_dim
        self.layers = []  # (lbd_kv8_pool, its buffers) of each layer; the layers share the page table
        self._set_layers([self._new_layer(self.pages) for _ in range(cfg.num_layers)])
        self.lengths = np.zeros(sequences, np.int64)
        self._held = np.zeros(sequences, np.int64)  # pages of each sequence
        self._hole = np.zeros((sequences, 2), np.int64)  # of them those given back by slide
        self._refs = np.zeros(self.pages, np.int64)  # sequences that hold each page
        self._free = list(range(self.pages - 1, -1, -1))
        self._table = np.full((sequences, self.max_pages), -1, np.int32)
        self._dirty = True
        self._copies: list[list] = []  # (page, its copy) that upload makes, in batches one after the other
        self.table = _buf(self._table.nbytes)
        self.past, self.q_start = _buf(4 * sequences), _buf(4 * (sequences + 1))
        self.one = K.DeviceBuffer.from_array(np.array([0, 1], np.int32))  # q_start of a one-token step
        self.work = _buf(16)

    def _new_layer(self, pages: int) -> list:
        codes, exps = pages * self._kv * self.page * self._d, pages * self._kv
        return [_buf(codes), _buf(codes), _buf(exps), _buf(exps)]

    def _set_layers(self, buffers: list):
        self.layers = [(K.LbdKv8Pool(*(x.ptr for x in b), self.pages, self.page, self._kv, self._d), b) for b in buffers]
        self.pools = (K.LbdKv8Pool * len(buffers))(*(p for p, _ in self.layers))

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
        made NaN stays NaN until the page is begun again (n a multiple of the page: at once). With a
        window, what the next token would see must not have been given back."""
        if not 0 <= n <= self.lengths[seq]:
            raise ValueError(f"sequence {seq} does not hold {n} tokens")
        a, b = self._hole[seq]
        if b > a and n > a * self.page and n - self.window + 1 < b * self.page:
            raise ValueError(f"pages of sequence {seq} that position {n} sees have been given back")
        self.commit(seq, n)

    def commit(self, seq: int, n: int):
        """The first n positions of sequence `seq` hold its tokens, as a pass over positions that reserve
        gave it has written them (pages past them return to the pool)."""
        keep = -(-int(n) // self.page)
        if n < 0 or keep > self._held[seq]:
            raise ValueError(f"sequence {seq} has no pages for {n} tokens")
        self._drop(seq, keep, int(self._held[seq]))
        if keep <= self._hole[seq, 0]:
            self._hole[seq] = 0
        self._held[seq], self.lengths[seq] = keep, n

    def _drop(self, seq: int, first: int, last: int):
        """Sequence `seq` no longer holds its pages first .. last - 1."""
        part = self._table[seq, first:last]
        gone = part[part >= 0]
        for p in gone[::-1]:
            self._refs[p] -= 1
            if not self._refs[p]:
                self._free.append(int(p))
        if len(gone):
            part[:] = -1
            self._dirty = True

    def _take(self) -> int:
        p = self._free.pop()
        self._refs[p] = 1
        return p

    def reserve(self, seq: int, n: int):
        """Pages for the first n positions of sequence `seq`, the one that its next token goes to its own."""
        if n > self.capacity:
            raise ValueError(f"KV cache full ({n} > {self.capacity})")
        need, has = -(-int(n) // self.page), int(self._held[seq])
        at, used = divmod(int(self.lengths[seq]), self.page)
        shared = n > self.lengths[seq] and used and self._refs[self._table[seq, at]] > 1
        more = max(need - has, 0) + bool(shared)
        if more > len(self._free):
            raise ValueError(f"KV cache full (no {more} pages left for sequence {seq})")
        if shared:
            p, mine = int(self._table[seq, at]), self._take()
            self._refs[p] -= 1
            self._table[seq, at] = mine
            self._dirty = True
            # copies of one batch are made at once: none may read or write what another writes
            if not self._copies or any(mine in pair or p == pair[1] for pair in self._copies[-1]):
                self._copies.append([])
            self._copies[-1].append((p, mine))
        for i in range(has, need):
            self._table[seq, i] = self._take()
            self._dirty = True
        self._held[seq] = max(need, has)

    def fork(self, dst: int, src: int):
        """Sequence `dst` becomes what `src` is (what it held returns to the pool): it shares its pages, none
        is copied until one of them writes to it."""
        dst, src = (range(len(self.lengths))[i] for i in (dst, src))  # negative ones count from the end
        if dst == src:
            raise ValueError("a sequence cannot be forked onto itself")
        self.commit(dst, 0)
        n = -(-int(self.lengths[src]) // self.page)
        self._table[dst, :n] = self._table[src, :n]
        for p in self._table[dst, :n]:
            if p >= 0:
                self._refs[p] += 1
        self._dirty = True
        self._held[dst], self.lengths[dst], self._hole[dst] = n, self.lengths[src], self._hole[src]

    def slide(self, seq: int):
        """Pages that no token behind the sequence's last one sees return to the pool (with a window; the
        model's passes call it)."""
        if not self.window:
            return
        a, b = -(-self.sinks // self.page), max(int(self.lengths[seq]) - self.window + 1, 0) // self.page
        if b > max(a, self._hole[seq, 1]):  # what was given back before is not looked at again
            self._drop(seq, max(a, int(self._hole[seq, 1])), b)
            self._hole[seq] = a, b

    def compact(self) -> int:
        """The pages in use moved to the front of the pool; returns how many they are."""
        self.upload()
        held = np.flatnonzero(self._refs)
        n = len(held)
        src = held[held >= n]
        dst = np.setdiff1d(np.arange(n), held)
        if len(src):
            to = np.arange(self.pages, dtype=np.int32)
            to[src] = dst
            self._copy(list(zip(src.tolist(), dst.tolist())), None)
            self._table = np.where(self._table >= 0, to[self._table], -1).astype(np.int32)
            self._refs[dst] = self._refs[src]
            self._refs[src] = 0
            self._dirty = True
            _check(K.lib().lb_dev_synchronize(), "synchronize")
        self._free = list(range(self.pages - 1, n - 1, -1))
        return n

    def resize(self, pages: int):
        """A pool of `pages` pages; where it shrinks the pages in use are compacted first and have to fit. One
        buffer of a layer at a time, so that there is room for little more than the larger of the two pools; if
        there is not, what is in use stays, in a pool of the fewer pages."""
        if pages <= 0 or pages < np.count_nonzero(self._refs):
            raise ValueError(f"{np.count_nonzero(self._refs)} pages are in use")
        if pages < self.pages:
            self.compact()
        else:
            self.upload()
        _check(K.lib().lb_dev_synchronize(), "synchronize")
        keep, buffers = min(int(pages), self.pages), [b for _, b in self.layers]
        code, self.pages = self._kv * self.page * self._d, keep
        try:
            for b in buffers:
                for i, of_page in enumerate((code, code, self._kv, self._kv)):
                    b[i] = self._resized(b[i], keep * of_page, int(pages) * of_page)
            self.pages = int(pages)
        finally:
            self._set_layers(buffers)
            self._refs = np.concatenate([self._refs[:keep], np.zeros(self.pages - keep, np.int64)])
            self._free = [int(p) for p in np.flatnonzero(self._refs == 0)[::-1]]

    @staticmethod
    def _resized(old, keep: int, nbytes: int):
        """A buffer of nbytes that begins as `old` does."""
        new = _buf(nbytes)
        _check(K.lib().lb_memcpy_d2d(new.ptr, old.ptr, keep), "pool copy")
        _check(K.lib().lb_dev_synchronize(), "synchronize")
        return new

    def _copy(self, pairs: list, stream):
        """Pages copied in every layer, on `stream`."""
        most, self._moved = 1 << 24, []  # pairs of a call; their arrays live until the next copies
        for at in range(0, len(pairs), most):
            a = [K.DeviceBuffer.from_array(np.array(x, np.int32)) for x in zip(*pairs[at:at + most])]
            self._moved.append(a)
            _check(K.lib().lbd_kv8_copy_pages(self.pools, len(self.layers), a[0].ptr, a[1].ptr,
                                              min(most, len(pairs) - at), stream), "page copies")

    def upload(self, stream=None):
        """The page table to the device, where it changed, and the copies that forks called for."""
        for batch in self._copies:
            self._copy(batch, stream)
            _check(K.lib().lb_stream_synchronize(stream), "synchronize")
        self._copies = []
        if self._dirty:
            _check(K.lib().lb_memcpy_h2d(self.table.ptr, self._table.ctypes.data, self._table.nbytes), "table upload")
            self._dirty = False

    def batch(self, q_start: int, past: int, seqs: int, max_new: int, rows: int, table: int | None = None) -> K.LbdKv8Batch:
        """The lbd_kv8_batch of the first `seqs` sequences (room: the workspace that its attention takes)."""
        return K.LbdKv8Batch(q_start, past, table or self.table.ptr, seqs, self.max_pages, max_new, rows)

    def room(self, b: K.LbdKv8Batch, heads: int):
        """Grow `work` to what the attention of this batch takes (no call may be in flight)."""
        L, pool, b = K.lib(), C.byref(self.layers[0][0]), C.byref(b)
        need = (L.lbd_kv8_attention_window_work_bytes(pool, b, heads, self.window, self.sinks) if self.window
                else L.lbd_kv8_attention_work_bytes(pool, b, heads))
        if need > self.work.nbytes:
            self.work = _buf(need)

    def beam_pages(self, seq: int, end: int, steps: int, beams: int) -> np.ndarray:
        """Pages that beams behind the first `end` tokens of sequence `seq` take beyond those it holds: with a window
        at each of their steps, for the next two, less what the sequence has given back by then."""
        last, full = -(-(end + steps) // self.page), end // self.page
        j = np.arange(max(last, int(self._held[seq])))
        held = (j < self._held[seq]) & (self._table[seq, :len(j)] >= 0)
        alone = held & (self._refs[np.where(held, self._table[seq, :len(j)], 0)] == 1)
        upto = lambda x: np.concatenate([[0], np.cumsum(x)])  # noqa: E731
        takes, alone = upto(np.where(j < full, 1, beams) - held), upto(alone)
        if not self.window:
            return takes[[last]]
        at = end + np.arange(max(steps, 1))
        b = np.maximum(at - self.window + 1, 0) // self.page  # pages in sight: those of the sinks, and b .. to - 1
        a, to = np.minimum(-(-self.sinks // self.page), b), -(-np.minimum(at + 2, end + steps) // self.page)
        return takes[a] + takes[to] - takes[b] - (alone[b] - alone[a])

    def beam_room(self, beams: int, steps: int, first: int) -> tuple:
        """Pages for the next tokens of `beams` places a prompt, those without a sequence among them where one has
        one: (the steps that they suffice for, all of them without a window, else a number as odd as `first` where
        it is not all; [sequences, max_pages] each place's own pages from the one in writing on, else -1)."""
        live, held = self.lengths > 0, self._held
        length = np.repeat(self.lengths.reshape(-1, beams).max(1), beams)  # (one within a prompt)
        tail = length // self.page

        def last(n):
            return np.where(length > 0, -(-(length + n) // self.page), 0)

        def takes(n):
            return int(np.maximum(last(n) - np.where(live, held, tail), 0).sum())

        n = steps
        if self.window and takes(n) > len(self._free):
            n = 0
            for bit in range(steps.bit_length() - 1, -1, -1):
                if n + (1 << bit) < steps and takes(n + (1 << bit)) <= len(self._free):
                    n += 1 << bit
            n -= n % 2 != first
        if takes(n) > len(self._free) or (steps and n <= 0):
            raise ValueError("KV cache full")
        own, to = np.full(self._table.shape, -1, np.int32), last(n)
        for i in np.flatnonzero(length):
            if live[i]:
                self.reserve(i, int(length[i]) + n)
                own[i, tail[i]:to[i]] = self._table[i, tail[i]:to[i]]
            else:
                own[i, tail[i]:to[i]] = [self._take() for _ in range(tail[i], to[i])]
        return n, own

    def adopt(self, table: np.ndarray, lengths: np.ndarray):
        """The sequences become those of a page table and their lengths (negative: none): every page belongs
        to the sequences that name it, the others are free."""
        self.lengths = np.maximum(np.asarray(lengths, np.int64), 0)
        self._held = -(-self.lengths // self.page)
        self._table = np.where(np.arange(self.max_pages) < self._held[:, None], table, -1).astype(np.int32)
        self._refs = np.bincount(self._table[self._table >= 0], minlength=self.pages).astype(np.int64)
        self._free = [int(p) for p in np.flatnonzero(self._refs == 0)[::-1]]
        self._hole[self.lengths == 0] = 0
        self._dirty = True


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
        if cfg.window < 0 or cfg.sinks < 0 or (cfg.sinks and not cfg.window):
            raise ValueError("window and sinks must not be negative, and sinks go with a window")
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

    def new_cache(self, max_len: int, kv: str | None = None, sequences: int = 1, page: int = 32,
                  pages: int | None = None) -> "KVCache | KV8Cache":
        """A cache of max_len positions: kv="fp32" (one sequence; the default without a window), or
        kv="e4m3", the paged 8-bit cache of `sequences` sequences (KV8Cache)."""
        kv = kv or ("e4m3" if self.cfg.window else "fp32")
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
        if cache.window:
            _check(L.lbd_kv8_attention_window(pool, b, self.qkv.ptr, width, H, cache.window, cache.sinks, self.att.ptr,
                                              H * D, cache.work.ptr, cache.work.nbytes, s), "kv8 window attention")
        else:
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
            cache.slide(0)
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
            cache.upload(self.stream)
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
        recording of the graph. With a window the steps take what pages the pool has, and
        where these run out those behind the window go back to it."""
        prompt = self._tokens(prompt)
        T = len(prompt)
        steps = max(0, n_new - 1)
        cache = cache or self._window_cache([T], T + n_new) or self.new_cache(T + n_new)
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
        if isinstance(cache, KV8Cache):  # the whole answer's pages where there is no window
            if cache.window and steps:
                need = int(_pages_at(np.arange(start + T, start + T + steps), cache.page, cache).max())
                if need > len(cache._free) + np.count_nonzero(cache._table[0] >= 0):
                    raise ValueError(f"KV cache full (a window of {need} pages)")
            cache.reserve(0, start + T + (0 if cache.window else steps))
            cache.upload(self.stream)
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
                for n in self._runs(cache, start + T, steps):
                    for _ in range(n):
                        _check(L.lb_graph_launch(ex.value, s), "graph launch")
                    self._sync()
            finally:
                L.lb_graph_destroy(ex.value)
        else:
            for n in self._runs(cache, start + T, steps):
                for _ in range(n):
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

    def _runs(self, cache, at: int, steps: int):
        """`steps` steps of a one-sequence cache from position `at` on in runs for which it has pages: the device
        is idle between them, when pages behind a window go back and the next ones are taken."""
        end = at + steps
        while at < end:
            n = end - at
            if isinstance(cache, KV8Cache) and cache.window:
                cache.commit(0, at)
                cache.slide(0)
                n = min(end, (int(cache._held[0]) + len(cache._free)) * cache.page) - at
                cache.reserve(0, at + n)
                cache.upload(self.stream)
            yield n
            at += n

    def _window_cache(self, prompts: list, capacity: int) -> "KV8Cache | None":
        """With a window, a cache for prompts of these lengths whose pool holds them and then their answers' windows
        (with eight pages more each, so that pages seldom run out)."""
        if not self.cfg.window:
            return None
        page = 32
        most = int(_pages_at(np.arange(capacity), page, self.cfg).max()) + 8
        pages = sum(min(-(-capacity // page), max(-(-n // page), most)) for n in prompts)
        return self.new_cache(capacity, "e4m3", len(prompts), page, pages)

    # ------------------------------------------------------------ several sequences

    def _pass(self, tokens: list, cache: KV8Cache) -> tuple:
        """tokens[s] of each sequence behind what it holds; (how many each had, the device's logits
        [sequences, V] of their last ones, enqueued: rows of sequences without tokens are no one's)."""
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
        self._rows(max(T, S))
        cache.upload(self.stream)
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
        for i in np.flatnonzero(news):
            cache.lengths[i] += news[i]
            cache.slide(i)
        return news, out

    def _rows(self, n: int):
        """Buffers of at least n rows (no call may be in flight)."""
        if n > self.tmax:
            self._alloc(n)
            self.tok = _buf(4 * n)

    def forward_batch(self, tokens: list, cache: KV8Cache) -> np.ndarray:
        """Run tokens[s] (possibly none) of each sequence s of an 8-bit cache behind what it holds:
        prompts, chunks of prompts and single tokens in one pass. Returns the logits [S, V] of each
        sequence's last token; rows of sequences without tokens are NaN."""
        news, out = self._pass(tokens, cache)
        y = out.to_array((len(news), self.cfg.vocab_size), np.float32)
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
            lengths = [len(p) for p in prompts]
            cache = self._window_cache(lengths, max(lengths) + n_new) or self.new_cache(
                max(lengths) + n_new, kv="e4m3", sequences=len(prompts))
        out = [[] for _ in prompts]
        y = self.forward_batch(list(prompts), cache)
        for i in range(n_new):
            tok = y.argmax(1)
            for o, v in zip(out, tok):
                o.append(int(v))
            if i + 1 < n_new:
                y = self.forward_batch([[int(v)] for v in tok], cache)
        return out

    def generate_beams(self, prompts: list, n_new: int, beams: int = 4, eos: int = -1, length_penalty: float = 1.0,
                       cache: KV8Cache | None = None, graph: bool = True) -> list[list[tuple[list[int], float]]]:
        """Beam search (lbd_beam_select): the `beams` best continuations of n_new tokens of each prompt by the
        sum of their log-probabilities, as (tokens, sum), best first by sum / length ** length_penalty. A beam
        that takes token `eos` has ended (its tokens end there): it keeps its sum and its place among the
        prompt's as long as no `beams` others exceed it. Fewer beams come back where the vocabulary offers no
        more.

        Beam w of prompt p is sequence p * beams + w of the cache (default: one of its own); a given cache may
        hold tokens in the first sequence of each prompt, which the prompt continues, and the others must be
        empty. Beams share the pages of what they have in common. Afterwards the sequences hold the
        beams in the order of their sums, all but their last token; ended beams hold nothing.

        The search stays on the device: selection, the page tables' new order and the next token's embedding
        read each other's results, and the steps replay one recorded HIP graph of two (graph=False launches
        them one by one). With eos the host looks every 32 steps whether all beams have ended. With a window the
        steps take what pages the pool has, and where these run out the host gives back those behind the window
        (an error after that leaves the sequences empty, one before it the prompts)."""
        cfg = self.cfg
        G, W, V, eos = len(prompts), int(beams), cfg.vocab_size, int(eos)
        if not G or not all(len(p) for p in prompts):
            raise ValueError("no tokens")
        if not 1 <= W <= 32:
            raise ValueError("1 to 32 beams")
        if not -1 <= eos < V:
            raise ValueError("eos is a token or -1")
        if n_new <= 0:
            return [[] for _ in prompts]
        n, steps = G * W, n_new - 1
        if cache is None:
            longest, page = max(len(p) for p in prompts) + steps, 16
            own = -(-steps // page) + 1  # pages that a beam may write
            if cfg.window:  # those in sight, and eight, so that pages seldom run out
                own = min(own, -(-(cfg.window + 1) // page) + 1 + -(-cfg.sinks // page) + 8)
            cache = self.new_cache(longest, "e4m3", n, page, sum(-(-len(p) // page) for p in prompts) + n * own)
        if not isinstance(cache, KV8Cache) or len(cache.lengths) != n:
            raise ValueError(f"the cache must be a KV8Cache of {n} sequences")
        firsts = np.arange(0, n, W)
        if np.delete(cache.lengths, firsts).any():
            raise ValueError("only the first sequence of each prompt may hold tokens")
        read, search = 0, 0
        for g, p in zip(firsts, prompts):
            was, end = int(cache.lengths[g]), int(cache.lengths[g]) + len(p)
            if end + steps > cache.capacity:
                raise ValueError(f"KV cache full ({was}+{len(p)}+{steps} > {cache.capacity})")
            copy = bool(was % cache.page and cache._refs[cache._table[g, was // cache.page]] > 1)
            read += max(-(-end // cache.page) - int(cache._held[g]), 0) + copy
            search = search + cache.beam_pages(g, end, steps, W) + copy
        need = max(read, int(search.max()))
        if need > len(cache._free):
            raise ValueError(f"KV cache full ({need} pages for the beams, {len(cache._free)} left)")
        _, logits = self._pass([prompts[i // W] if i % W == 0 else [] for i in range(n)], cache)
        held = cache.lengths.copy()
        try:
            return self._search(logits, cache, G, W, n_new, eos, length_penalty, graph)
        except BaseException:
            # the prompts, as they were read, or nothing where a window has given pages of theirs back
            cache.adopt(cache._table, held if np.array_equal(cache.lengths, held) else 0 * held)
            raise

    def _search(self, logits, cache: KV8Cache, G: int, W: int, n_new: int, eos: int, length_penalty: float,
                graph: bool) -> list:
        """generate_beams behind its prompts' pass, `logits` of their last tokens."""
        cfg, L, s = self.cfg, self.L, self.stream
        n, V, steps, firsts = G * W, cfg.vocab_size, n_new - 1, np.arange(0, G * W, W)
        hole = cache._hole[firsts].copy()  # what a window has given back of each prompt's beams
        room, own = cache.beam_room(W, steps, 1)  # steps that there are pages for (odd: one, and then pairs)
        cache.upload(s)
        up, lengths = K.DeviceBuffer.from_array, np.where(np.arange(n) % W == 0, cache.lengths, -1).astype(np.int32)
        sums = np.where(np.arange(n) % W == 0, 0.0, -np.inf).astype(np.float32)
        # two states in turn: a step reads one and writes the other
        state = [dict(past=up(lengths), table=up(cache._table), score=up(sums), done=up(np.zeros(n, np.int32)))
                 for _ in range(2)]
        parent, mine, count = up(np.zeros(n, np.int32)), up(own), up(np.zeros(G, np.int32))
        hist = [up(np.zeros((n_new, n), np.int32)) for _ in range(2)]
        self._rows(n)
        choose = [K.LbdBeams(a["score"].ptr, a["done"].ptr, b["score"].ptr, b["done"].ptr, self.tok.ptr, parent.ptr,
                             hist[0].ptr, hist[1].ptr, count.ptr, n_new, G, W, V, eos) for a, b in (state, state[::-1])]
        work = _buf(L.lbd_beam_select_work_bytes(C.byref(choose[0])))
        q_start = up(np.arange(n + 1, dtype=np.int32))
        batches = [cache.batch(q_start.ptr, x["past"].ptr, n, 1, n, x["table"].ptr) for x in state]
        cache.room(batches[0], cfg.num_heads)

        def select(x: int, add: int):
            """The beams of state x into the other one."""
            a, b = state[x], state[1 - x]
            _check(L.lbd_beam_select(logits.ptr, V, C.byref(choose[x]), work.ptr, work.nbytes, s), "beam selection")
            order = K.LbdKv8Order(parent.ptr, b["done"].ptr, a["past"].ptr, a["table"].ptr, mine.ptr, b["past"].ptr,
                                  b["table"].ptr, G, W, cache.max_pages, add)
            _check(L.lbd_kv8_reorder(cache.pools, len(cache.layers), C.byref(order), s), "beam order")

        def step(x: int):
            self.batch = batches[x]
            self._layers(n, cache)
            self._linear(self.lm_head, self.h.ptr, n, logits.ptr)
            select(x, 1)

        def slide(x: int) -> int:
            """Pages behind the window of state x's sequences go back; the steps that there are pages for now."""
            self._sync()
            cache.adopt(state[x]["table"].to_array((n, cache.max_pages), np.int32),
                        state[x]["past"].to_array((n,), np.int32))
            for i in np.flatnonzero(cache.lengths):
                cache._hole[i] = hole[i // W]
            for i in np.flatnonzero(cache.lengths):
                cache.slide(i)
                hole[i // W] = cache._hole[i]
            room, own = cache.beam_room(W, left, 0)
            past = np.where(cache.lengths > 0, cache.lengths, -1).astype(np.int32)
            for buf, a in ((state[x]["past"], past), (state[x]["table"], cache._table), (mine, own)):
                _check(L.lb_memcpy_h2d(buf.ptr, a.ctypes.data, a.nbytes), "state upload")
            return room

        select(0, 0)
        x, left = 1, steps
        if left:  # the first step builds what later ones find (tile layouts), outside of any graph
            step(x)
            x, left, room = 1 - x, left - 1, room - 1
        ex = C.c_void_p()
        try:
            if graph and left >= 2:
                self._sync()
                _check(L.lb_stream_begin_capture(s), "begin capture")
                try:
                    step(x)
                    step(1 - x)
                finally:
                    _check(L.lb_stream_end_capture(s, C.byref(ex)), "end capture")
            since = 0
            while left:
                if not room:
                    room = slide(x)
                if ex.value and left >= 2:
                    _check(L.lb_graph_launch(ex.value, s), "graph launch")
                    took = 2
                else:
                    step(x)
                    took, x = 1, 1 - x
                left, room, since = left - took, room - took, since + took
                if eos >= 0 and since >= 32 and left:
                    since = 0
                    self._sync()
                    ended = state[x]["done"].to_array((n,), np.int32) != 0
                    if (ended | (state[x]["score"].to_array((n,), np.float32) == -np.inf)).all():
                        break
            self._sync()
        finally:
            if ex.value:
                L.lb_graph_destroy(ex.value)
        took = n_new - left
        tok, back = (h.to_array((n_new, n), np.int32)[:took] for h in hist)
        sums, ended = state[x]["score"].to_array((n,), np.float32), state[x]["done"].to_array((n,), np.int32)
        cache.adopt(state[x]["table"].to_array((n, cache.max_pages), np.int32), state[x]["past"].to_array((n,), np.int32))
        for i in np.flatnonzero(cache.lengths):
            cache._hole[i] = hole[i // W]
            cache.slide(i)
        out = []
        for g in firsts:
            found = []
            for i in range(g, g + W):
                if back[-1, i] < 0:
                    continue
                answer, at = [], i
                for t in range(took - 1, -1, -1):
                    answer.append(int(tok[t, at]))
                    at = back[t, at]
                answer.reverse()
                if ended[i]:  # it has taken eos once, and stood as it was since
                    answer = answer[:answer.index(eos) + 1]
                found.append((answer, float(sums[i])))
            out.append(sorted(found, key=lambda b: -b[1] / len(b[0]) ** length_penalty))
        return out
