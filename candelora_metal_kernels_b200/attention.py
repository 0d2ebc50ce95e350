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

_PREFILL_DTYPES = (torch.float16, torch.bfloat16)
_KV_DTYPES = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16, torch.int8: _lib.KV_INT8}


# These calls last a few microseconds on the GPU, so the host side counts: device indices are compared instead of device
# objects, the stream is taken without its wrapper, and arguments are packed as bytes.

def _on(index: int, fn, *args) -> int:
    """fn(*args) with GPU `index` as the current one, which the C ABI expects."""
    if index == torch._C._cuda_getDevice():
        return fn(*args)
    with torch.cuda.device(index):
        return fn(*args)


def _call(index: int, fn, *args) -> None:
    """fn(*args, stream) on GPU `index`."""
    # (current_stream(device).cuda_stream without the Stream object)
    rc = _on(index, fn, *args, torch._C._cuda_getCurrentRawStream(index))
    if rc != _lib.IQ2_OK:
        _lib.check(rc)


def _elsewhere(op: str, index: int, name: str, t: torch.Tensor):
    _bail(_lib.IQ2_ERR_DEVICE, f"{op} device mismatch: {name}={t.device}, expected cuda:{index}")


def _indices(op: str, index: int, name: str, t: torch.Tensor, dims: int) -> torch.Tensor:
    if t.get_device() != index:
        _elsewhere(op, index, name, t)
    if t.dtype != torch.int32 or t.dim() != dims:
        _bail(_lib.IQ2_ERR_DTYPE, f"{op} expects {name} as an int32 tensor of rank {dims}, got {t.dtype} {list(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def _rows(op: str, index: int, name: str, t: torch.Tensor, heads: int | None, dim: int):
    """`t` as [tokens, heads, dim] with a contiguous last dimension (a copy where it is not), its strides, its shape."""
    if t.get_device() != index:
        _elsewhere(op, index, name, t)
    shape = t.shape
    if len(shape) != 3 or shape[2] != dim or (heads is not None and shape[1] != heads):
        _bail(_lib.IQ2_ERR_INVALID_ARGUMENT, f"{op} expects {name} of shape [tokens, {heads if heads else 'heads'}, {dim}], "
                                             f"got {list(shape)}")
    strides = t.stride()
    if strides[2] != 1:
        t = t.contiguous()
        strides = t.stride()
    return t, strides, shape


def _out(op: str, index: int, out, shape, dtype, near: torch.Tensor) -> torch.Tensor:
    """`out` if it fits, or a new tensor on the device of `near`."""
    if out is None:
        if near.dtype == dtype and near.shape == shape and near.is_contiguous():
            return torch.empty_like(near)  # the cheapest way to a tensor
        return near.new_empty(shape, dtype=dtype)
    if out.shape != shape or out.dtype != dtype or not out.is_contiguous() or out.get_device() != index:
        _bail(_lib.IQ2_ERR_INVALID_ARGUMENT, f"{op}: out must be a contiguous {dtype} {list(shape)} tensor on cuda:{index}")
    return out


class KvCache:
    """A paged key-value cache over tensors k, v [num_pages, kv_heads, page_size, head_dim] (f16, bf16 or int8) and, for
    int8, k_scale, v_scale f32 [num_pages, kv_heads, page_size]. Token `pos` of a sequence lies in page
    block_table[sequence, pos // page_size], row pos % page_size. The calls take the tensors' addresses from here, so that k, v
    and the scales cannot be replaced (a cache of other tensors is another KvCache), and calls refuse ones whose memory has
    moved since. Holds no other state."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None):
        op = "KvCache"
        if k.dim() != 4 or k.shape != v.shape:
            _bail(_lib.IQ2_ERR_INVALID_ARGUMENT, f"{op} expects k and v of one shape [num_pages, kv_heads, page_size, "
                                                 f"head_dim], got {list(k.shape)} and {list(v.shape)}")
        if k.device.type != "cuda":
            _bail(_lib.IQ2_ERR_DEVICE, f"{op} requires a CUDA device")
        for name, t in (("v", v), ("k_scale", k_scale), ("v_scale", v_scale)):
            if t is not None and t.device != k.device:
                _elsewhere(op, k.get_device(), name, t)
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
        self._k, self._v, self._k_scale, self._v_scale = k, v, k_scale, v_scale
        self.num_pages, self.kv_heads, self.page_size, self.head_dim = k.shape
        self.dtype, self.device, self._index = k.dtype, k.device, k.get_device()
        self._addresses = self._now()
        self._struct = _lib.KvCacheStruct(*self._addresses, *k.shape, _KV_DTYPES[k.dtype])
        self._ptr = ctypes.addressof(self._struct)

    k = property(lambda self: self._k)
    v = property(lambda self: self._v)
    k_scale = property(lambda self: self._k_scale)
    v_scale = property(lambda self: self._v_scale)

    def _now(self) -> tuple:
        if self._k_scale is None:
            return self._k.data_ptr(), self._v.data_ptr(), None, None
        return self._k.data_ptr(), self._v.data_ptr(), self._k_scale.data_ptr(), self._v_scale.data_ptr()

    def _checked(self, op: str) -> int:
        """The address of the C struct, if the tensors still lie where they did."""
        if self._now() != self._addresses:
            _bail(_lib.IQ2_ERR_INVALID_ARGUMENT, f"{op}: the cache's tensors have moved since the KvCache was made")
        return self._ptr

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
    (2i, 2i + 1) with `interleaved`; without cos and sin, positions are not read. q [tokens, q_heads, head_dim], of k's
    dtype, is returned as q_dtype (its own by default)."""
    op = "kv_cache_write"
    d, index, kv_heads = cache.head_dim, cache._index, cache.kv_heads
    k, k_strides, (tokens, _, _) = _rows(op, index, "k", k, kv_heads, d)
    v, v_strides, v_shape = _rows(op, index, "v", v, kv_heads, d)
    slots = _indices(op, index, "slots", slots, 1)
    dtype = k.dtype
    if dtype not in _X_DTYPES or v.dtype != dtype or (q is not None and q.dtype != dtype):
        _bail(_lib.IQ2_ERR_DTYPE, f"{op} expects q, k and v in one of f32, f16 and bf16, got {dtype} and {v.dtype}"
                                  f"{'' if q is None else f' and {q.dtype}'}")
    same = v_shape[0] == tokens and slots.shape[0] == tokens
    rows_q, out_ptr, out_code, rope = (0, 0, 0, 0), 0, 0, (0, 0, 0, 0)
    if q is not None:
        q, q_strides, q_shape = _rows(op, index, "q", q, None, d)
        same = same and q_shape[0] == tokens
        q_dtype = q_dtype or dtype
        if q_dtype not in _X_DTYPES:
            _bail(_lib.IQ2_ERR_DTYPE, f"{op} unsupported q dtype: {q_dtype}")
        q_out = _out(op, index, q_out, q_shape, q_dtype, q)
        rows_q, out_ptr, out_code = (q.data_ptr(), q_strides[0], q_strides[1], q_shape[1]), q_out.data_ptr(), _X_DTYPES[q_dtype]
    elif q_out is not None or q_dtype is not None:
        _bail(_lib.IQ2_ERR_INVALID_ARGUMENT, f"{op}: q_out and q_dtype go with q")
    if cos is not None or sin is not None:
        if cos is None or sin is None or positions is None:
            _bail(_lib.IQ2_ERR_INVALID_ARGUMENT, f"{op}: cos and sin go together, and with positions")
        shape = cos.shape
        if cos.get_device() != index or sin.get_device() != index:
            _elsewhere(op, index, "cos or sin", cos if sin.get_device() == index else sin)
        if cos.dtype != torch.float32 or sin.dtype != torch.float32 or sin.shape != shape or len(shape) != 2 or \
                shape[1] * 2 != d or not cos.is_contiguous() or not sin.is_contiguous():
            _bail(_lib.IQ2_ERR_INVALID_ARGUMENT, f"{op} expects contiguous f32 cos and sin [rows, {d // 2}], got "
                                                 f"{cos.dtype} {list(shape)} and {sin.dtype} {list(sin.shape)}")
        positions = _indices(op, index, "positions", positions, 1)
        same = same and positions.shape[0] == tokens
        rope = (positions.data_ptr(), cos.data_ptr(), sin.data_ptr(), shape[0])
    if not same:
        _bail(_lib.IQ2_ERR_INVALID_ARGUMENT, f"{op}: k has {tokens} tokens, v {v.shape[0]}, slots {slots.shape[0]}"
                                             f"{'' if q is None else f', q {q.shape[0]}'}"
                                             f"{'' if positions is None else f', positions {positions.shape[0]}'}")
    if tokens:
        args = _lib.KV_TOKENS.pack(k.data_ptr(), k_strides[0], k_strides[1], v.data_ptr(), v_strides[0], v_strides[1], *rows_q[:3],
                                   _X_DTYPES[dtype], tokens, rows_q[3], slots.data_ptr(), *rope, interleaved, out_ptr, out_code)
        _call(index, _lib.load().iq2_kv_cache_write, cache._checked(op), args)
    return q_out


def kv_cache_read(cache: KvCache, block_table: torch.Tensor, cu_seqlens: torch.Tensor, total_tokens: int, *,
                  starts: torch.Tensor | None = None, dtype: torch.dtype | None = None, k_out=None, v_out=None):
    """Packed (k, v) [total_tokens, kv_heads, head_dim] in `dtype` (the cache's own, bf16 for an int8 cache): rows
    [cu_seqlens[b], cu_seqlens[b + 1]) are the tokens starts[b], starts[b] + 1, ... (from 0 without `starts`) of the
    sequence whose pages are block_table[b] (int32 [sequences, width]). Rows of no sequence are zeros."""
    op = "kv_cache_read"
    index = cache._index
    table, cu = _indices(op, index, "block_table", block_table, 2), _indices(op, index, "cu_seqlens", cu_seqlens, 1)
    seqs, width = table.shape
    starts = None if starts is None else _indices(op, index, "starts", starts, 1)
    if cu.shape[0] != seqs + 1 or (starts is not None and starts.shape[0] != seqs):
        _bail(_lib.IQ2_ERR_INVALID_ARGUMENT, f"{op}: block_table has {seqs} sequences, cu_seqlens {cu.shape[0]} entries")
    if dtype is None:
        dtype = torch.bfloat16 if cache.dtype == torch.int8 else cache.dtype
    if dtype not in _X_DTYPES:
        _bail(_lib.IQ2_ERR_DTYPE, f"{op} unsupported out dtype: {dtype}")
    shape = (total_tokens, cache.kv_heads, cache.head_dim)
    k_out = _out(op, index, k_out, shape, dtype, cache.k)
    v_out = _out(op, index, v_out, shape, dtype, k_out)
    if total_tokens:
        _call(index, _lib.load().iq2_kv_cache_read, cache._checked(op), table.data_ptr(), width, seqs,
              None if starts is None else starts.data_ptr(), cu.data_ptr(), total_tokens, k_out.data_ptr(),
              v_out.data_ptr(), _X_DTYPES[dtype])
    return k_out, v_out


def _tiles(t: torch.Tensor, strides, shape):
    """`t` and its strides, or a copy where rows do not start on 16-byte boundaries of their own (whole tiles are loaded)."""
    tokens, heads = strides[0], strides[1]
    if t.data_ptr() % 16 == 0 and (shape[1] == 1 or (heads > 0 and heads % 8 == 0)) and (shape[0] <= 1 or (tokens > 0 and tokens % 8 == 0)):
        return t, strides
    t = t.clone(memory_format=torch.contiguous_format)
    return t, t.stride()


def attention_prefill(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens_q: torch.Tensor,
                      cu_seqlens_k: torch.Tensor | None = None, *, causal: bool = True, scale: float | None = None,
                      out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(scale q k^T) v of packed sequences: q [q_tokens, q_heads, head_dim], k, v [k_tokens, kv_heads, head_dim],
    f16 or bf16, sequence b holding the rows [cu_seqlens[b], cu_seqlens[b + 1]) (int32; cu_seqlens_k: those of q). With
    `causal`, query i of Lq sees the keys j <= i + Lk - Lq of Lk. scale: 1 / sqrt(head_dim) by default. Queries that see
    no key give zeros, and rows of no sequence are zeros. Returns q's shape and dtype."""
    op = "attention_prefill"
    if not q.is_cuda:
        _bail(_lib.IQ2_ERR_DEVICE, f"{op} requires a CUDA device")
    index, dtype = q.get_device(), q.dtype
    if dtype not in _PREFILL_DTYPES or k.dtype != dtype or v.dtype != dtype:
        _bail(_lib.IQ2_ERR_DTYPE, f"{op} expects q, k and v all in f16 or all in bf16, got {dtype}, {k.dtype}, {v.dtype}")
    q, q_strides, q_shape = _rows(op, index, "q", q, None, q.shape[-1])
    tokens, heads, d = q_shape
    k, k_strides, k_shape = _rows(op, index, "k", k, None, d)
    keys, kv_heads, _ = k_shape
    v, v_strides, v_shape = _rows(op, index, "v", v, kv_heads, d)
    if v_shape[0] != keys:
        _bail(_lib.IQ2_ERR_INVALID_ARGUMENT, f"{op}: k has {keys} tokens, v {v_shape[0]}")
    cu_q = cu_k = _indices(op, index, "cu_seqlens_q", cu_seqlens_q, 1)
    if cu_seqlens_k is not None:
        cu_k = _indices(op, index, "cu_seqlens_k", cu_seqlens_k, 1)
    entries = cu_q.shape[0]
    if cu_k.shape[0] != entries or entries == 0:
        _bail(_lib.IQ2_ERR_INVALID_ARGUMENT, f"{op}: cu_seqlens_q and cu_seqlens_k have {entries} and {cu_k.shape[0]} entries")
    (q, (q0, q1, _)), (k, (k0, k1, _)), (v, (v0, v1, _)) = \
        _tiles(q, q_strides, q_shape), _tiles(k, k_strides, k_shape), _tiles(v, v_strides, v_shape)
    out = _out(op, index, out, q_shape, dtype, q)
    args = _lib.ATTENTION_PROMPTS.pack(
        q.data_ptr(), q0, q1, k.data_ptr(), k0, k1, v.data_ptr(), v0, v1,
        _X_DTYPES[dtype], entries - 1, tokens, keys, heads, kv_heads, d, cu_q.data_ptr(), cu_k.data_ptr(), causal,
        _scale(op, scale), out.data_ptr())
    lib = _lib.load()
    if workspace is None:
        workspace = _scratch(_on(index, lib.iq2_attention_prefill_workspace_size, args), q)
    _call(index, lib.iq2_attention_prefill, args, *_buffer(workspace))
    return out


def _scale(op: str, scale: float | None) -> float:
    if scale is None:
        return 0.0
    if not 0.0 < scale < float("inf"):
        _bail(_lib.IQ2_ERR_INVALID_ARGUMENT, f"{op}: scale is not positive")
    return scale


def _scratch(need: int, near: torch.Tensor):
    return near.new_empty(need, dtype=torch.uint8) if need else None


def _buffer(workspace: torch.Tensor | None):
    return (None, 0) if workspace is None else (workspace.data_ptr(), workspace.numel())


def attention_decode_workspace_bytes(q: torch.Tensor, cache: KvCache, block_table: torch.Tensor) -> int:
    """Device scratch attention_decode needs for q [batch, q_heads, head_dim], whatever the lengths."""
    return int(_on(cache._index, _lib.load().iq2_attention_decode_workspace_size, cache._ptr, q.shape[0], q.shape[1]))


def attention_decode(q: torch.Tensor, cache: KvCache, block_table: torch.Tensor, seq_lens: torch.Tensor, *,
                     scale: float | None = None, out: torch.Tensor | None = None,
                     workspace: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(scale q k^T) v of one token a sequence over its cached tokens: q [batch, q_heads, head_dim] (f32, f16 or
    bf16), block_table int32 [batch, width], seq_lens int32 [batch] (a sequence of length 0 gives zeros). Returns q's
    shape and dtype; the accumulation is in f32."""
    op = "attention_decode"
    index = cache._index
    q, strides, shape = _rows(op, index, "q", q, None, cache.head_dim)
    batch, heads, _ = shape
    dtype = q.dtype
    if dtype not in _X_DTYPES:
        _bail(_lib.IQ2_ERR_DTYPE, f"{op} unsupported q dtype: {dtype}")
    table, lens = _indices(op, index, "block_table", block_table, 2), _indices(op, index, "seq_lens", seq_lens, 1)
    tables, width = table.shape
    if tables != batch or lens.shape[0] != batch:
        _bail(_lib.IQ2_ERR_INVALID_ARGUMENT, f"{op}: q has a batch of {batch}, block_table {tables}, seq_lens {lens.shape[0]}")
    out = _out(op, index, out, shape, dtype, q)
    args = _lib.ATTENTION_TOKENS.pack(q.data_ptr(), strides[0], strides[1], _X_DTYPES[dtype], batch, heads, width,
                                      table.data_ptr(), lens.data_ptr(), _scale(op, scale), out.data_ptr())
    lib = _lib.load()
    if workspace is None:
        workspace = _scratch(attention_decode_workspace_bytes(q, cache, block_table), q)
    _call(index, lib.iq2_attention_decode, cache._checked(op), args, *_buffer(workspace))
    return out
