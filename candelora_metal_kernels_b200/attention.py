"""Tensor-level host API of the attention operators over the CUDA C ABI (no reference counterpart: the reference ends at
the projections). They take the projections' outputs as [tokens, heads, head_dim] CUDA tensors:

  KvCache               a paged cache: 16-bit, or int8 with a scale for each token and head
  kv_cache_write        rotates q and k, writes k and v into the cache
  kv_cache_read         cached tokens back into packed 16- or 32-bit tensors
  attention_prefill     attention of packed prompts (causal or not, grouped heads)
  attention_decode      attention of one new token a sequence over the cache

Every call is stream-ordered on the current CUDA stream and raises `Iq2Error` before anything is launched when an
argument does not fit.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import Iq2Error
from .iq2_matmul import _X_DTYPES, _bail

_KV_DTYPES = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16, torch.int8: _lib.KV_INT8}


def _call(device: torch.device, fn, *args) -> None:
    """fn(*args, stream) on `device`, which the C ABI expects to be the current one."""
    index = device.index
    stream = torch._C._cuda_getCurrentRawStream(index)  # current_stream(device).cuda_stream without the Stream object
    if index == torch._C._cuda_getDevice():
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, stream)
    if rc != _lib.IQ2_OK:
        _lib.check(rc)


def _on(op: str, device: torch.device, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != device:
            _bail(_lib.IQ2_ERR_DEVICE, f"{op} device mismatch: {name}={t.device}, expected {device}")


def _indices(op: str, name: str, t: torch.Tensor, dims: int) -> torch.Tensor:
    if t.dtype != torch.int32 or t.dim() != dims:
        _bail(_lib.IQ2_ERR_DTYPE, f"{op} expects {name} as an int32 tensor of rank {dims}, got {t.dtype} {list(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def _rows(op: str, name: str, t: torch.Tensor, heads: int | None, dim: int) -> torch.Tensor:
    """`t` as [tokens, heads, dim] with a contiguous last dimension (a copy where it is not)."""
    if t.dim() != 3 or t.shape[2] != dim or (heads is not None and t.shape[1] != heads):
        _bail(_lib.IQ2_ERR_INVALID_ARGUMENT, f"{op} expects {name} of shape [tokens, {heads if heads else 'heads'}, {dim}], "
                                             f"got {list(t.shape)}")
    return t if t.stride(2) == 1 else t.contiguous()


def _rows_struct(t: torch.Tensor) -> _lib.Rows:
    return _lib.Rows(t.data_ptr(), t.stride(0), t.stride(1))


def _out(op: str, out, shape, dtype, device) -> torch.Tensor:
    if out is None:
        return torch.empty(shape, dtype=dtype, device=device)
    if tuple(out.shape) != tuple(shape) or out.dtype != dtype or not out.is_contiguous() or out.device != device:
        _bail(_lib.IQ2_ERR_INVALID_ARGUMENT, f"{op}: out must be a contiguous {dtype} {list(shape)} tensor on {device}")
    return out


class KvCache:
    """A paged key-value cache over tensors k, v [num_pages, kv_heads, page_size, head_dim] (f16, bf16 or int8) and, for
    int8, k_scale, v_scale f32 [num_pages, kv_heads, page_size]. Token `pos` of a sequence lies in page
    block_table[sequence, pos // page_size], row pos % page_size. Holds no state besides the tensors."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None):
        op = "KvCache"
        if k.dim() != 4 or k.shape != v.shape:
            _bail(_lib.IQ2_ERR_INVALID_ARGUMENT, f"{op} expects k and v of one shape [num_pages, kv_heads, page_size, "
                                                 f"head_dim], got {list(k.shape)} and {list(v.shape)}")
        if k.device.type != "cuda":
            _bail(_lib.IQ2_ERR_DEVICE, f"{op} requires a CUDA device")
        _on(op, k.device, v=v, k_scale=k_scale, v_scale=v_scale)
        if k.dtype not in _KV_DTYPES or v.dtype != k.dtype:
            _bail(_lib.IQ2_ERR_DTYPE, f"{op} unsupported cache dtype: {k.dtype}, {v.dtype}")
        if k.dtype == torch.int8:
            for s in (k_scale, v_scale):
                if s is None or s.dtype != torch.float32 or s.shape != k.shape[:3] or not s.is_contiguous():
                    _bail(_lib.IQ2_ERR_INVALID_ARGUMENT, f"{op}: an int8 cache takes contiguous f32 scales {list(k.shape[:3])}")
        elif k_scale is not None or v_scale is not None:
            _bail(_lib.IQ2_ERR_INVALID_ARGUMENT, f"{op}: only an int8 cache takes scales")
        if not k.is_contiguous() or not v.is_contiguous():
            _bail(_lib.IQ2_ERR_INVALID_ARGUMENT, f"{op} expects contiguous layouts")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.num_pages, self.kv_heads, self.page_size, self.head_dim = k.shape
        self.dtype, self.device = k.dtype, k.device
        self._struct = _lib.KvCacheStruct(
            k.data_ptr(), v.data_ptr(), None if k_scale is None else k_scale.data_ptr(),
            None if v_scale is None else v_scale.data_ptr(), *k.shape, _KV_DTYPES[k.dtype])
        self._ptr = ctypes.addressof(self._struct)

    @classmethod
    def empty(cls, num_pages: int, kv_heads: int, page_size: int, head_dim: int, dtype: torch.dtype = torch.bfloat16,
              device="cuda") -> "KvCache":
        """A cache of zeros."""
        shape = (num_pages, kv_heads, page_size, head_dim)
        k, v = (torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
        if dtype != torch.int8:
            return cls(k, v)
        return cls(k, v, *(torch.zeros(shape[:3], dtype=torch.float32, device=device) for _ in range(2)))


def kv_cache_write(cache: KvCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, *, q: torch.Tensor | None = None,
                   q_dtype: torch.dtype | None = None, positions: torch.Tensor | None = None,
                   cos: torch.Tensor | None = None, sin: torch.Tensor | None = None, interleaved: bool = False,
                   q_out: torch.Tensor | None = None) -> torch.Tensor | None:
    """Write k, v [tokens, kv_heads, head_dim] (f32, f16 or bf16) to the cache's `slots` (int32 [tokens],
    page * page_size + row; a slot outside the cache, e.g. -1, writes nothing). With cos, sin f32
    [rows, head_dim / 2] and positions int32 [tokens], k and q are rotated first: pairs (i, i + head_dim / 2), or
    (2i, 2i + 1) with `interleaved`. q [tokens, q_heads, head_dim], of k's dtype, is returned as q_dtype (its own by
    default)."""
    op = "kv_cache_write"
    d, device = cache.head_dim, cache.device
    _on(op, device, k=k, v=v, slots=slots, q=q, positions=positions, cos=cos, sin=sin)
    k, v = _rows(op, "k", k, cache.kv_heads, d), _rows(op, "v", v, cache.kv_heads, d)
    tokens = k.shape[0]
    if k.dtype not in _X_DTYPES or v.dtype != k.dtype or (q is not None and q.dtype != k.dtype):
        _bail(_lib.IQ2_ERR_DTYPE, f"{op} expects q, k and v in one of f32, f16 and bf16, got {k.dtype} and {v.dtype}"
                                  f"{'' if q is None else f' and {q.dtype}'}")
    slots = _indices(op, "slots", slots, 1)
    args = _lib.KvTokens(k=_rows_struct(k), v=_rows_struct(v), dtype=_X_DTYPES[k.dtype], tokens=tokens,
                         slots=slots.data_ptr(), interleaved=int(interleaved))
    counts = {"v": v.shape[0], "slots": slots.shape[0]}
    if q is not None:
        q = _rows(op, "q", q, None, d)
        counts["q"] = q.shape[0]
        q_dtype = q_dtype or q.dtype
        if q_dtype not in _X_DTYPES:
            _bail(_lib.IQ2_ERR_DTYPE, f"{op} unsupported q dtype: {q_dtype}")
        q_out = _out(op, q_out, q.shape, q_dtype, device)
        args.q, args.q_heads = _rows_struct(q), q.shape[1]
        args.q_out, args.q_out_dtype = q_out.data_ptr(), _X_DTYPES[q_dtype]
    elif q_out is not None or q_dtype is not None:
        _bail(_lib.IQ2_ERR_INVALID_ARGUMENT, f"{op}: q_out and q_dtype go with q")
    if cos is not None or sin is not None or positions is not None:
        if cos is None or sin is None or positions is None:
            _bail(_lib.IQ2_ERR_INVALID_ARGUMENT, f"{op}: cos, sin and positions go together")
        for t in (cos, sin):
            if t.dtype != torch.float32 or t.dim() != 2 or t.shape != cos.shape or t.shape[1] * 2 != d or not t.is_contiguous():
                _bail(_lib.IQ2_ERR_INVALID_ARGUMENT, f"{op} expects contiguous f32 cos and sin [rows, {d // 2}], got "
                                                     f"{t.dtype} {list(t.shape)}")
        positions = _indices(op, "positions", positions, 1)
        counts["positions"] = positions.shape[0]
        args.positions, args.cos, args.sin, args.rope_len = positions.data_ptr(), cos.data_ptr(), sin.data_ptr(), cos.shape[0]
    if any(n != tokens for n in counts.values()):
        _bail(_lib.IQ2_ERR_INVALID_ARGUMENT, f"{op}: k has {tokens} tokens, the others {counts}")
    if tokens:
        _call(device, _lib.load().iq2_kv_cache_write, cache._ptr, ctypes.addressof(args))
    return q_out


def kv_cache_read(cache: KvCache, block_table: torch.Tensor, cu_seqlens: torch.Tensor, total_tokens: int, *,
                  starts: torch.Tensor | None = None, dtype: torch.dtype | None = None, k_out=None, v_out=None):
    """Packed (k, v) [total_tokens, kv_heads, head_dim] in `dtype` (the cache's own, bf16 for an int8 cache): rows
    [cu_seqlens[b], cu_seqlens[b + 1]) are the tokens starts[b], starts[b] + 1, ... (from 0 without `starts`) of the
    sequence whose pages are block_table[b] (int32 [sequences, width]). Rows of no sequence are zeros."""
    op = "kv_cache_read"
    device = cache.device
    _on(op, device, block_table=block_table, cu_seqlens=cu_seqlens, starts=starts)
    table, cu = _indices(op, "block_table", block_table, 2), _indices(op, "cu_seqlens", cu_seqlens, 1)
    seqs, width = table.shape
    starts = None if starts is None else _indices(op, "starts", starts, 1)
    if cu.shape[0] != seqs + 1 or (starts is not None and starts.shape[0] != seqs):
        _bail(_lib.IQ2_ERR_INVALID_ARGUMENT, f"{op}: block_table has {seqs} sequences, cu_seqlens {cu.shape[0]} entries")
    if dtype is None:
        dtype = torch.bfloat16 if cache.dtype == torch.int8 else cache.dtype
    if dtype not in _X_DTYPES:
        _bail(_lib.IQ2_ERR_DTYPE, f"{op} unsupported out dtype: {dtype}")
    shape = (total_tokens, cache.kv_heads, cache.head_dim)
    k_out, v_out = _out(op, k_out, shape, dtype, device), _out(op, v_out, shape, dtype, device)
    if total_tokens:
        _call(device, _lib.load().iq2_kv_cache_read, cache._ptr, table.data_ptr(), width, seqs,
              None if starts is None else starts.data_ptr(), cu.data_ptr(), total_tokens, k_out.data_ptr(),
              v_out.data_ptr(), _X_DTYPES[dtype])
    return k_out, v_out


def _aligned_rows(t: torch.Tensor) -> torch.Tensor:
    """`t`, or a copy of it where rows do not start on 16-byte boundaries of their own (whole tiles are loaded)."""
    heads, tokens = t.stride(1), t.stride(0)
    if t.data_ptr() % 16 == 0 and (t.shape[1] == 1 or (heads > 0 and heads % 8 == 0)) and \
            (t.shape[0] <= 1 or (tokens > 0 and tokens % 8 == 0)):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def attention_prefill(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens_q: torch.Tensor,
                      cu_seqlens_k: torch.Tensor | None = None, *, causal: bool = True, scale: float | None = None,
                      out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(scale q k^T) v of packed sequences: q [q_tokens, q_heads, head_dim], k, v [k_tokens, kv_heads, head_dim],
    f16 or bf16, sequence b holding the rows [cu_seqlens[b], cu_seqlens[b + 1]) (int32; cu_seqlens_k: those of q). With
    `causal`, query i of Lq sees the keys j <= i + Lk - Lq of Lk. scale: 1 / sqrt(head_dim) by default. Queries that see
    no key give zeros. Returns q's shape and dtype."""
    op = "attention_prefill"
    if q.device.type != "cuda":
        _bail(_lib.IQ2_ERR_DEVICE, f"{op} requires a CUDA device")
    cu_seqlens_k = cu_seqlens_q if cu_seqlens_k is None else cu_seqlens_k
    device = q.device
    _on(op, device, k=k, v=v, cu_seqlens_q=cu_seqlens_q, cu_seqlens_k=cu_seqlens_k)
    if q.dtype not in (torch.float16, torch.bfloat16) or k.dtype != q.dtype or v.dtype != q.dtype:
        _bail(_lib.IQ2_ERR_DTYPE, f"{op} expects q, k and v all in f16 or all in bf16, got {q.dtype}, {k.dtype}, {v.dtype}")
    q = _rows(op, "q", q, None, q.shape[-1])
    tokens, heads, d = q.shape
    k = _rows(op, "k", k, None, d)
    v = _rows(op, "v", v, k.shape[1], d)
    if v.shape[0] != k.shape[0]:
        _bail(_lib.IQ2_ERR_INVALID_ARGUMENT, f"{op}: k has {k.shape[0]} tokens, v {v.shape[0]}")
    cu_q, cu_k = _indices(op, "cu_seqlens_q", cu_seqlens_q, 1), _indices(op, "cu_seqlens_k", cu_seqlens_k, 1)
    if cu_q.shape[0] != cu_k.shape[0] or cu_q.shape[0] == 0:
        _bail(_lib.IQ2_ERR_INVALID_ARGUMENT, f"{op}: cu_seqlens_q and cu_seqlens_k have {cu_q.shape[0]} and {cu_k.shape[0]} entries")
    q, k, v = _aligned_rows(q), _aligned_rows(k), _aligned_rows(v)
    out = _out(op, out, q.shape, q.dtype, device)
    args = _lib.AttentionPrompts(_rows_struct(q), _rows_struct(k), _rows_struct(v), _X_DTYPES[q.dtype], cu_q.shape[0] - 1,
                                 tokens, k.shape[0], heads, k.shape[1], d, cu_q.data_ptr(), cu_k.data_ptr(), int(causal),
                                 _scale(op, scale), out.data_ptr())
    lib = _lib.load()
    ws, ws_len, _keep = _scratch(lib.iq2_attention_prefill_workspace_size(ctypes.addressof(args)), workspace, device)
    _call(device, lib.iq2_attention_prefill, ctypes.addressof(args), ws, ws_len)
    return out


def _scale(op: str, scale: float | None) -> float:
    if scale is None:
        return 0.0
    if not 0.0 < scale < float("inf"):
        _bail(_lib.IQ2_ERR_INVALID_ARGUMENT, f"{op}: scale is not positive")
    return scale


def _scratch(need: int, workspace, device):
    """(pointer, length, tensor to keep) of a workspace of `need` bytes: the caller's, or a new one."""
    if need == 0:
        return None, 0, None
    if workspace is None or workspace.numel() < need:
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
    return workspace.data_ptr(), workspace.numel(), workspace


def attention_decode_workspace_bytes(q: torch.Tensor, cache: KvCache, block_table: torch.Tensor) -> int:
    """Device scratch attention_decode needs for q [batch, q_heads, head_dim], whatever the lengths."""
    with torch.cuda.device(cache.device):
        return int(_lib.load().iq2_attention_decode_workspace_size(cache._ptr, q.shape[0], q.shape[1]))


def attention_decode(q: torch.Tensor, cache: KvCache, block_table: torch.Tensor, seq_lens: torch.Tensor, *,
                     scale: float | None = None, out: torch.Tensor | None = None,
                     workspace: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(scale q k^T) v of one token a sequence over its cached tokens: q [batch, q_heads, head_dim] (f32, f16 or
    bf16), block_table int32 [batch, width], seq_lens int32 [batch] (a sequence of length 0 gives zeros). Returns q's
    shape and dtype; the accumulation is in f32."""
    op = "attention_decode"
    device = cache.device
    _on(op, device, q=q, block_table=block_table, seq_lens=seq_lens)
    q = _rows(op, "q", q, None, cache.head_dim)
    batch, heads, _ = q.shape
    if q.dtype not in _X_DTYPES:
        _bail(_lib.IQ2_ERR_DTYPE, f"{op} unsupported q dtype: {q.dtype}")
    table, lens = _indices(op, "block_table", block_table, 2), _indices(op, "seq_lens", seq_lens, 1)
    if table.shape[0] != batch or lens.shape[0] != batch:
        _bail(_lib.IQ2_ERR_INVALID_ARGUMENT, f"{op}: q has a batch of {batch}, block_table {table.shape[0]}, seq_lens {lens.shape[0]}")
    out = _out(op, out, q.shape, q.dtype, device)
    args = _lib.AttentionTokens(_rows_struct(q), _X_DTYPES[q.dtype], batch, heads, table.shape[1], table.data_ptr(),
                                lens.data_ptr(), _scale(op, scale), out.data_ptr())
    lib = _lib.load()
    ws, ws_len, _keep = _scratch(lib.iq2_attention_decode_workspace_size(cache._ptr, batch, heads), workspace, device)
    _call(device, lib.iq2_attention_decode, cache._ptr, ctypes.addressof(args), ws, ws_len)
    return out
