"""Decoder-layer operators around the quantized projections, over torch CUDA tensors.

The reference's Qwen2-style graphs (python/mlx_worker/native_mlx/ of the reference)
run, on either side of every projection:
  * RMSNorm (models/qwen2.py:144-147,161-165; mx.fast.rms_norm),
  * RoPE on queries and keys (models/qwen2.py:91-105; mx.fast.rope, traditional=False),
  * the paged KV append and attention over the cached pages
    (attention.py:215-298 append_and_attend, cache.py:485-520 stage_layer, with the
    [pages, page_size, kv_heads, head_dim] pools of cache.py:651-700),
  * the embedding lookup (models/qwen2.py:185).
Each function here is one call into libmlxq_b200.so on the tensors' device and
current stream; misuse raises ValueError, device failures RuntimeError.
"""
from __future__ import annotations

import math
import threading
from dataclasses import dataclass

import torch

from . import _lib
from .core import Workspace

__all__ = ["rms_norm", "rope_kv_append", "paged_attention_decode", "paged_attention_prefill",
           "paged_attention_tree", "tree_masks", "kv_cache_read", "QuantizedKV",
           "quantized_embedding", "decode_advance", "PagedKVCache", "PagedBatch"]

_DT = {torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


def _code(t: torch.Tensor, what: str) -> int:
    if t.dtype not in _DT:
        raise ValueError(f"{what} must be bfloat16 or float16, got {t.dtype}")
    return _DT[t.dtype]


def _stream(dev: torch.device):
    return torch.cuda.current_stream(dev).cuda_stream


def _p(t):
    return None if t is None else t.data_ptr()


@dataclass(frozen=True)
class QuantizedKV:
    """One layer's keys or values held in 8 or 4 bits: the pool a 16-bit cache tensor
    [pages, page_size, n_kv_heads, head_dim] stands for, each head's row quantized in groups
    of group_size and laid out as quantize() does it. codes uint32
    [pages, page_size, n_kv_heads, head_dim*bits/32], scales and biases [pages, page_size, n_kv_heads, head_dim/group_size] of the
    activation dtype; a code q stands for scale * q + bias, rounded once to that dtype.
    Rows that rope_kv_append writes are quantize()'s too, bit for bit, but for groups whose
    larger end lies half way between two codes from zero (under one in a hundred).
    Takes a cache tensor's place in rope_kv_append, kv_cache_read and the paged
    attention functions (keys and values of the same width)."""
    codes: torch.Tensor
    scales: torch.Tensor
    biases: torch.Tensor
    group_size: int = 64
    bits: int = 4

    def __post_init__(self):
        if self.bits not in (4, 8):
            raise ValueError(f"a quantized cache has 4 or 8 bits, got {self.bits}")
        if self.group_size not in (32, 64, 128):
            raise ValueError(f"group_size must be 32, 64 or 128, got {self.group_size}")
        c, s, b = self.codes, self.scales, self.biases
        if c.dtype not in (torch.uint32, torch.int32) or s.dtype not in _DT or b.dtype != s.dtype:
            raise ValueError("codes must be uint32, scales and biases bfloat16 or float16")
        if c.ndim != 4 or s.shape != b.shape or s.shape[:3] != c.shape[:3] or \
                s.shape[3] * self.group_size * self.bits != c.shape[3] * 32:
            raise ValueError("codes [pages, page_size, n_kv_heads, head_dim*bits/32] and scales, "
                             "biases [..., head_dim/group_size] expected")
        if not (c.is_contiguous() and s.is_contiguous() and b.is_contiguous()):
            raise ValueError("a quantized cache's tensors must be contiguous")
        if c.device != s.device or c.device != b.device:
            raise ValueError("a quantized cache's tensors must be on one device")
        # the C ABI's fields: every call compares and passes them
        object.__setattr__(self, "_geometry", (*c.shape[:3], s.shape[3] * self.group_size,
                                               self.bits, self.group_size, _DT[s.dtype]))

    @classmethod
    def zeros(cls, num_pages: int, page_size: int, n_kv_heads: int, head_dim: int,
              group_size: int = 64, bits: int = 4, dtype=torch.bfloat16, device="cuda"):
        """An empty pool."""
        if group_size <= 0 or head_dim % group_size:
            raise ValueError(f"head_dim {head_dim} is not a multiple of group_size {group_size}")
        rows = (num_pages, page_size, n_kv_heads)
        sb = [torch.zeros(*rows, head_dim // group_size, dtype=dtype, device=device)
              for _ in range(2)]
        return cls(torch.zeros(*rows, head_dim * bits // 32, dtype=torch.int32,
                               device=device).view(torch.uint32), *sb, group_size, bits)

    @property
    def shape(self) -> tuple:
        return (*self.codes.shape[:3], self.scales.shape[3] * self.group_size)

    @property
    def dtype(self) -> torch.dtype:
        return self.scales.dtype

    @property
    def device(self) -> torch.device:
        return self.codes.device


def _kv_struct(k, v) -> _lib.KVCache:
    """The C ABI's view of one layer's pools (16-bit tensors, or QuantizedKV)."""
    if isinstance(k, QuantizedKV):
        if not isinstance(v, QuantizedKV) or v._geometry != k._geometry:
            raise ValueError("keys and values must share a quantized cache's shape and width")
        return _lib.KVCache(k.codes.data_ptr(), v.codes.data_ptr(), k.scales.data_ptr(),
                            k.biases.data_ptr(), v.scales.data_ptr(), v.biases.data_ptr(),
                            *k._geometry)
    shape, dt = k.shape, k.dtype
    if isinstance(v, QuantizedKV) or v.shape != shape or v.dtype is not dt:
        raise ValueError("k_cache and v_cache must share shape and dtype")
    if len(shape) != 4 or not k.is_contiguous() or not v.is_contiguous():
        raise ValueError("caches must be contiguous [pages, page_size, n_kv_heads, head_dim]")
    if dt not in _DT:
        raise ValueError(f"the cache must be bfloat16 or float16, got {dt}")
    return _lib.KVCache(k.data_ptr(), v.data_ptr(), None, None, None, None, *shape, 16, 0, _DT[dt])


def _on(t: torch.Tensor, *ts) -> int:
    """The index of t's CUDA device, which every other tensor has to be on."""
    i = t.get_device()
    if i < 0:
        raise ValueError(f"expected CUDA tensors, got a tensor on {t.device}")
    for u in ts:
        if u is not None and u.get_device() != i:
            raise ValueError(f"tensors are on different devices ({t.device} and {u.device})")
    return i


def _call(i: int, call):
    """call(stream) with device i current, on its current stream. (The raw handle: making
    a Stream object takes longer than a small launch.)"""
    if torch._C._cuda_getDevice() == i:
        return call(torch._C._cuda_getCurrentRawStream(i))
    with torch.cuda.device(i):
        return call(torch._C._cuda_getCurrentRawStream(i))


def _pool(c) -> torch.Tensor:
    """A tensor of a cache side, for its device."""
    return c.codes if isinstance(c, QuantizedKV) else c


def _i32(t: torch.Tensor, what: str) -> torch.Tensor:
    if t.dtype != torch.int32:
        raise ValueError(f"{what} must be int32, got {t.dtype}")
    return t.contiguous()


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
             residual: torch.Tensor | None = None, residual_out: bool = False):
    """RMSNorm of the last axis (nn.RMSNorm): round(round(h * rsqrt(mean(h^2) + eps))
    * weight) with h = x, or h = round(x + residual). With residual_out, returns
    (normed, h): the decoder block's `hidden = x + attn_out` and its norm in one
    launch (qwen2.py:161-165)."""
    dt = _code(x, "x")
    D = x.shape[-1]
    if weight.shape != (D,) or weight.dtype != x.dtype:
        raise ValueError(f"weight must be [{D}] of dtype {x.dtype}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError("residual must match x")
    if residual_out and residual is None:
        raise ValueError("residual_out needs a residual")
    x = x.contiguous()
    rows = x.numel() // D if D else 0
    out = torch.empty_like(x)
    h = torch.empty_like(x) if residual_out else None
    with torch.cuda.device(x.device):
        rc = _lib.load().mlxq_rms_norm(_p(x), _p(None if residual is None else residual.contiguous()),
                                       _p(weight.contiguous()), _p(out), _p(h), rows, D,
                                       float(eps), dt, _stream(x.device))
    _lib.check(rc, "rms_norm")
    return (out, h) if residual_out else out


def rope_kv_append(qkv: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor,
                   k_cache, v_cache, n_heads: int, n_kv_heads: int,
                   head_dim: int, base: float = 10000.0, q_norm: torch.Tensor | None = None,
                   k_norm: torch.Tensor | None = None, eps: float = 1e-6) -> torch.Tensor:
    """RoPE of the queries and keys in `qkv` [T, (n_heads + 2 n_kv_heads) * head_dim]
    (the fused q/k/v projection's output) at `positions` [T], keys and values written
    to cache rows `slots` [T] (page * page_size + offset, -1 = skip) of
    k_cache / v_cache [pages, page_size, n_kv_heads, head_dim], or quantized into a pair
    of QuantizedKV. With q_norm / k_norm [head_dim] each query / key head is RMS-normed
    first (the head norms of Qwen3-style attention, models/qwen3.py of the reference),
    in the same launch and with one rounding; angles are then, and into a QuantizedKV, reduced
    in 64 bits, where the plain form into 16-bit caches takes them in 32 (off by some 2^-23 of
    the angle, 10^-2 rad at position 10^5). A group of a QuantizedKV row that would hold a
    NaN or an infinity stands for NaN as a whole. Returns the rotated queries
    [T, n_heads, head_dim]. Two tokens of a call must not share a slot."""
    if q_norm is not None or k_norm is not None or isinstance(k_cache, QuantizedKV) or \
            isinstance(v_cache, QuantizedKV):
        return _norm_rope_append(qkv, positions, slots, k_cache, v_cache, n_heads, n_kv_heads,
                                 head_dim, base, q_norm, k_norm, eps)
    dt = _code(qkv, "qkv")
    if qkv.ndim != 2 or qkv.stride(1) != 1:
        raise ValueError("qkv must be a 2-D tensor with contiguous rows")
    T = qkv.shape[0]
    for c in (k_cache, v_cache):
        if c.dtype != qkv.dtype or c.shape[-2:] != (n_kv_heads, head_dim) or not c.is_contiguous():
            raise ValueError("caches must be contiguous [pages, page_size, n_kv_heads, head_dim] "
                             "of qkv's dtype")
    positions, slots = _i32(positions, "positions"), _i32(slots, "slots")
    if positions.shape != (T,) or slots.shape != (T,):
        raise ValueError(f"positions and slots must be [{T}]")
    q = torch.empty(T, n_heads, head_dim, dtype=qkv.dtype, device=qkv.device)
    with torch.cuda.device(qkv.device):
        rc = _lib.load().mlxq_rope_kv_append(_p(qkv), qkv.stride(0), _p(q), _p(k_cache),
                                             _p(v_cache), _p(positions), _p(slots), T, n_heads,
                                             n_kv_heads, head_dim, float(base), dt,
                                             _stream(qkv.device))
    _lib.check(rc, "rope_kv_append")
    return q


def _norm_rope_append(qkv, positions, slots, k_cache, v_cache, n_heads, n_kv_heads, head_dim,
                      base, q_norm, k_norm, eps):
    kv = _kv_struct(k_cache, v_cache)
    dt = qkv.dtype
    if qkv.dim() != 2 or qkv.stride(1) != 1 or dt is not k_cache.dtype:
        raise ValueError("qkv must be a 2-D tensor with contiguous rows, of the caches' dtype")
    if kv.n_kv_heads != n_kv_heads or kv.head_dim != head_dim:
        raise ValueError("caches must hold n_kv_heads heads of head_dim")
    T, width = qkv.shape
    if n_heads <= 0 or width < (n_heads + 2 * n_kv_heads) * head_dim:
        raise ValueError("qkv's rows must hold q, k and v")
    for w in (q_norm, k_norm):
        if w is not None and (w.dim() != 1 or w.numel() != head_dim or w.dtype is not dt or
                              not w.is_contiguous()):
            raise ValueError(f"norm weights must be contiguous [{head_dim}] of dtype {dt}")
    positions, slots = _i32(positions, "positions"), _i32(slots, "slots")
    if positions.dim() != 1 or positions.numel() != T or slots.dim() != 1 or slots.numel() != T:
        raise ValueError(f"positions and slots must be [{T}]")
    dev = _on(qkv, positions, slots, _pool(k_cache), _pool(v_cache), q_norm, k_norm)
    q = qkv.new_empty((T, n_heads, head_dim))
    # (a single row's stride is arbitrary)
    ld = qkv.stride(0) if T > 1 else (width + 7) // 8 * 8
    append = _lib.load().mlxq_norm_rope_kv_append
    rc = _call(dev, lambda st: append(
        kv, qkv.data_ptr(), ld, q.data_ptr(), None if q_norm is None else q_norm.data_ptr(),
        None if k_norm is None else k_norm.data_ptr(), eps, positions.data_ptr(),
        slots.data_ptr(), T, n_heads, base, st))
    _lib.check(rc, "rope_kv_append")
    return q


def kv_cache_read(k_cache, v_cache, slots: torch.Tensor):
    """The values cache rows `slots` [n] (page * page_size + offset) hold: keys and values
    [n, n_kv_heads, head_dim] in the cache's dtype, dequantized with one rounding from a
    QuantizedKV. Slots outside the pool (-1) give zero rows."""
    kv = _kv_struct(k_cache, v_cache)
    slots = _i32(slots, "slots")
    if slots.ndim != 1:
        raise ValueError("slots must be [n]")
    dev = _on(_pool(k_cache), _pool(v_cache), slots)
    n = slots.shape[0]
    values = k_cache.scales if kv.bits != 16 else k_cache
    k, v = (values.new_empty((n, kv.n_kv_heads, kv.head_dim)) for _ in range(2))
    rc = _call(dev, lambda st: _lib.load().mlxq_kv_cache_read(kv, _p(slots), n, _p(k), _p(v), st))
    _lib.check(rc, "kv_cache_read")
    return k, v


def _rows_attention(q, cu_q, max_q_len, k_cache, v_cache, block_table, kv_lens, max_kv_len,
                    tree_mask, scale, what):
    """mlxq_paged_attention_rows: a cache of any width, one or several rows a sequence.
    max_kv_len None: what the block table can hold."""
    kv = _kv_struct(k_cache, v_cache)
    shape = q.shape
    if len(shape) != 3 or _DT.get(q.dtype) != kv.dtype or shape[2] != kv.head_dim:
        raise ValueError("q must be [rows, n_heads, head_dim] of the cache's head_dim and dtype")
    rows, H, _ = shape
    q = q.contiguous()
    block_table, kv_lens = _i32(block_table, "block_table"), _i32(kv_lens, "kv_lens")
    if block_table.dim() != 2 or kv_lens.dim() != 1 or kv_lens.numel() != block_table.size(0):
        raise ValueError("block_table must be [B, max_blocks] and kv_lens [B]")
    B, blocks = block_table.shape
    if cu_q is not None:
        cu_q = _i32(cu_q, "cu_q")
        if cu_q.dim() != 1 or cu_q.numel() != B + 1:
            raise ValueError(f"cu_q must be [{B + 1}] (one offset per sequence, then the total)")
    elif rows != B:
        raise ValueError(f"q must have one row per sequence ({B}), got {rows}")
    if tree_mask is not None:
        if tree_mask.dtype is not torch.int64 or tree_mask.dim() != 1 or tree_mask.numel() != rows:
            raise ValueError(f"tree_mask must be int64 [{rows}]")
        tree_mask = tree_mask.contiguous()
    dev = _on(q, cu_q, _pool(k_cache), _pool(v_cache), block_table, kv_lens, tree_mask)
    out = torch.empty_like(q)
    max_q_len = int(max_q_len)
    max_kv_len = blocks * kv.page_size if max_kv_len is None else int(max_kv_len)
    L = _lib.load()

    def call(st):
        need = L.mlxq_paged_attention_rows_workspace_size(kv, B, max_q_len, max_kv_len, H)
        # per call, from the allocator: calls on other streams and in other captured graphs
        # have their own
        ws = q.new_empty(need, dtype=torch.uint8) if need else None
        return L.mlxq_paged_attention_rows(
            kv, q.data_ptr(), None if cu_q is None else cu_q.data_ptr(), rows, max_q_len,
            block_table.data_ptr(), blocks, kv_lens.data_ptr(), max_kv_len,
            None if tree_mask is None else tree_mask.data_ptr(), out.data_ptr(), B, H,
            float(scale), None if ws is None else ws.data_ptr(), need, st)

    _lib.check(_call(dev, call), what)
    return out


def paged_attention_tree(q: torch.Tensor, cu_q: torch.Tensor, max_q_len: int, k_cache, v_cache,
                         block_table: torch.Tensor, kv_lens: torch.Tensor, max_kv_len: int,
                         tree_mask: torch.Tensor, scale: float) -> torch.Tensor:
    """Trees of drafted tokens: q [total, n_heads, head_dim], sequence b's n <= 64 tokens at
    rows [cu_q[b], cu_q[b+1]), their keys and values appended as the last n of its
    kv_lens[b] <= max_kv_len cached ones (slots in row order, whatever the tokens' depths
    and positions). Every token sees the keys before those n, and of the n token j where
    bit j of its word in tree_mask [total] (int64) is set: see tree_masks. A row that sees
    nothing is zero, and so are rows behind cu_q[-1]. A value of the n new tokens that is not
    finite reaches the rows that do not see it as well. Caches of 16 bits or QuantizedKV."""
    if tree_mask is None:
        raise ValueError("paged_attention_tree needs a tree_mask")
    return _rows_attention(q, cu_q, max_q_len, k_cache, v_cache, block_table, kv_lens, max_kv_len,
                           tree_mask, scale, "paged_attention_tree")


def tree_masks(parents, device="cuda") -> torch.Tensor:
    """Ancestor masks for paged_attention_tree from one list of parents per sequence (the
    index of each token's parent, before it, in its own tree; -1 for a root): int64 [total],
    each token's own bit and its ancestors'."""
    masks = []
    for tree in parents:
        if len(tree) > 64:
            raise ValueError("a tree has at most 64 tokens")
        own = []
        for i, p in enumerate(tree):
            if not -1 <= p < i:
                raise ValueError(f"token {i}'s parent must be an earlier token or -1, got {p}")
            own.append((own[p] if p >= 0 else 0) | 1 << i)
        masks += [m - (1 << 64) if m >> 63 else m for m in own]
    return torch.tensor(masks, dtype=torch.int64, device=device)


def _cache_geometry(k_cache, v_cache, q):
    if k_cache.shape != v_cache.shape or k_cache.dtype != q.dtype or v_cache.dtype != q.dtype:
        raise ValueError("k_cache and v_cache must share shape and q's dtype")
    if k_cache.ndim != 4 or not k_cache.is_contiguous() or not v_cache.is_contiguous():
        raise ValueError("caches must be contiguous [pages, page_size, n_kv_heads, head_dim]")
    _, page, hkv, hd = k_cache.shape
    return page, hkv, hd


def paged_attention_decode(q: torch.Tensor, k_cache, v_cache,
                           block_table: torch.Tensor, kv_lens: torch.Tensor, max_kv_len: int,
                           scale: float) -> torch.Tensor:
    """One query per sequence: q [B, n_heads, head_dim] at position kv_lens[b] - 1
    attends all kv_lens[b] cached keys of sequence b (pages block_table[b]). The caches are
    16-bit tensors or a pair of QuantizedKV."""
    if isinstance(k_cache, QuantizedKV) or isinstance(v_cache, QuantizedKV):
        return _rows_attention(q, None, 1, k_cache, v_cache, block_table, kv_lens, max_kv_len,
                               None, scale, "paged_attention_decode")
    dt = _code(q, "q")
    page, hkv, hd = _cache_geometry(k_cache, v_cache, q)
    B, H, _ = q.shape
    block_table, kv_lens = _i32(block_table, "block_table"), _i32(kv_lens, "kv_lens")
    out = torch.empty_like(q)
    dev = q.device
    L = _lib.load()
    need = L.mlxq_paged_attention_workspace_size(B, hkv, max_kv_len, hd)
    with torch.cuda.device(dev):
        st = torch.cuda.current_stream(dev)
        ws = Workspace.get(dev, st, need, "attention") if need else None
        rc = L.mlxq_paged_attention_decode(_p(q.contiguous()), _p(k_cache), _p(v_cache),
                                           _p(block_table), block_table.shape[1], _p(kv_lens),
                                           int(max_kv_len), _p(out), B, H, hkv, hd, page,
                                           float(scale), dt, _p(ws),
                                           0 if ws is None else ws.numel(), st.cuda_stream)
    _lib.check(rc, "paged_attention_decode")
    return out


def paged_attention_prefill(q: torch.Tensor, cu_q: torch.Tensor, max_q_len: int,
                            k_cache, v_cache,
                            block_table: torch.Tensor, kv_lens: torch.Tensor,
                            scale: float, max_kv_len: int | None = None) -> torch.Tensor:
    """New tokens of every sequence: q [total, n_heads, head_dim], sequence b's rows
    [cu_q[b], cu_q[b+1]) at the last positions of its kv_lens[b] cached keys, causal. The
    caches are 16-bit tensors or a pair of QuantizedKV. max_kv_len is a bound on kv_lens
    (default: what the block table can hold): over a QuantizedKV it sizes the workspace and
    the work, so give it where tables are wider than the sequences."""
    if isinstance(k_cache, QuantizedKV) or isinstance(v_cache, QuantizedKV):
        return _rows_attention(q, cu_q, max_q_len, k_cache, v_cache, block_table, kv_lens,
                               max_kv_len, None, scale, "paged_attention_prefill")
    dt = _code(q, "q")
    page, hkv, hd = _cache_geometry(k_cache, v_cache, q)
    _, H, _ = q.shape
    block_table, kv_lens = _i32(block_table, "block_table"), _i32(kv_lens, "kv_lens")
    cu_q = _i32(cu_q, "cu_q")
    B = block_table.shape[0]
    if cu_q.shape != (B + 1,):
        raise ValueError(f"cu_q must be [{B + 1}] (one offset per sequence, then the total)")
    if max_kv_len is not None and not 0 <= max_kv_len <= block_table.shape[1] * page:
        raise ValueError("max_kv_len must be in [0, max_blocks * page_size]")
    out = torch.empty_like(q)
    with torch.cuda.device(q.device):
        rc = _lib.load().mlxq_paged_attention_prefill(
            _p(q.contiguous()), _p(cu_q), int(max_q_len), _p(k_cache), _p(v_cache),
            _p(block_table), block_table.shape[1], _p(kv_lens), _p(out), B, H, hkv, hd, page,
            float(scale), dt, _stream(q.device))
    _lib.check(rc, "paged_attention_prefill")
    return out


def quantized_embedding(ids: torch.Tensor, wq: torch.Tensor, scales: torch.Tensor,
                        biases: torch.Tensor, group_size: int = 64, bits: int = 4,
                        out: torch.Tensor | None = None) -> torch.Tensor:
    """Rows ids of a quantized table, dequantized (QuantizedEmbedding lookup):
    bit-identical to dequantize() of those rows; [..., dim]."""
    dt = _code(scales, "scales")
    ids = _i32(ids, "ids")
    vocab, dim = wq.shape[0], scales.shape[-1] * group_size
    if wq.ndim != 2 or wq.shape[1] * 32 // bits != dim or scales.shape != biases.shape or \
            scales.shape[0] != vocab:
        raise ValueError("wq [vocab, dim*bits/32], scales/biases [vocab, dim/group_size] expected")
    flat = ids.reshape(-1)
    if out is None:
        out = torch.empty(*ids.shape, dim, dtype=scales.dtype, device=wq.device)
    with torch.cuda.device(wq.device):
        rc = _lib.load().mlxq_quantized_embedding(_p(flat), flat.numel(), _p(wq), _p(scales),
                                                  _p(biases), _p(out), vocab, dim, group_size,
                                                  bits, dt, _stream(wq.device))
    _lib.check(rc, "quantized_embedding")
    return out


def decode_advance(positions: torch.Tensor, kv_lens: torch.Tensor, slots: torch.Tensor,
                   block_table: torch.Tensor, page_size: int) -> None:
    """In place on the device: every sequence one token further (positions += 1,
    kv_lens = positions + 1, slots = the new position's cache row)."""
    with torch.cuda.device(positions.device):
        rc = _lib.load().mlxq_decode_advance(_p(positions), _p(kv_lens), _p(slots),
                                             _p(block_table), block_table.shape[1],
                                             positions.numel(), page_size,
                                             _stream(positions.device))
    _lib.check(rc, "decode_advance")


@dataclass
class PagedBatch:
    """Where one forward step's tokens go (the reference's ForwardBatch and
    PagedBatchReservation, interfaces.py:95-109, cache.py:420-520): per new token its
    position and cache slot; per sequence its page ids, cached length after the
    append, and (prefill) the offsets of its tokens in the flat batch."""
    block_table: torch.Tensor      # [B, max_blocks] int32
    kv_lens: torch.Tensor          # [B] int32, keys cached after this step
    positions: torch.Tensor        # [T] int32
    slots: torch.Tensor            # [T] int32
    max_kv_len: int
    cu_q: torch.Tensor | None = None   # [B + 1] int32 (prefill); None = one token each
    max_q_len: int = 1


class PagedKVCache:
    """Fixed-size page pools per layer, [num_pages, page_size, n_kv_heads, head_dim]
    for keys and for values (cache.py:651-700), and a free list of page ids handed
    out to sequences in any order (the pages of a sequence need not be contiguous).
    With bits 8 or 4 the pools are QuantizedKV, quantized in groups of group_size as
    they are written."""

    def __init__(self, num_layers: int, n_kv_heads: int, head_dim: int, num_pages: int,
                 page_size: int = 16, dtype=torch.bfloat16, device="cuda", bits: int = 16,
                 group_size: int = 64):
        if bits not in (4, 8, 16):
            raise ValueError("cache bits must be 4, 8 or 16")
        if page_size not in (8, 16, 32):
            raise ValueError("page_size must be 8, 16 or 32")
        self.page_size, self.n_kv_heads, self.head_dim = page_size, n_kv_heads, head_dim
        shape = (num_pages, page_size, n_kv_heads, head_dim)
        if bits == 16:
            def pool():
                return torch.zeros(shape, dtype=dtype, device=device)
        else:
            def pool():
                return QuantizedKV.zeros(*shape, group_size, bits, dtype, device)
        self.keys = [pool() for _ in range(num_layers)]
        self.values = [pool() for _ in range(num_layers)]
        self._free = list(range(num_pages))
        self._lock = threading.Lock()

    @property
    def num_free_pages(self) -> int:
        return len(self._free)

    def allocate(self, lengths, generator=None) -> torch.Tensor:
        """Pages for sequences of the given maximum lengths: block table [B, max_blocks]
        int32 (unused entries 0). With a generator the free pages are handed out in
        a shuffled order."""
        blocks = [math.ceil(n / self.page_size) for n in lengths]
        with self._lock:
            if sum(blocks) > len(self._free):
                raise RuntimeError(f"KV cache full: {sum(blocks)} pages asked, "
                                   f"{len(self._free)} free")
            if generator is not None:
                perm = torch.randperm(len(self._free), generator=generator).tolist()
                self._free = [self._free[i] for i in perm]
            table = torch.zeros(len(lengths), max(1, max(blocks, default=1)), dtype=torch.int32)
            for b, nb in enumerate(blocks):
                for j in range(nb):
                    table[b, j] = self._free.pop()
        return table.to(self.keys[0].device)

    def release(self, block_table: torch.Tensor, lengths) -> None:
        with self._lock:
            for b, n in enumerate(lengths):
                self._free.extend(block_table[b, :math.ceil(n / self.page_size)].tolist())

    def slots(self, block_table: torch.Tensor, positions_per_seq) -> torch.Tensor:
        """Cache rows of the given positions of each sequence (host-computed), int32."""
        bt = block_table.cpu()
        out = []
        for b, poss in enumerate(positions_per_seq):
            for p in poss:
                out.append(int(bt[b, p // self.page_size]) * self.page_size + p % self.page_size)
        return torch.tensor(out, dtype=torch.int32, device=block_table.device)
