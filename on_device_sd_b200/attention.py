"""The attention side of a decoding step over a paged key-value cache: the cache write (with head norms and rotary
embedding in the same launch) and the attention of new tokens, single ones (draft step) or spans (verify step).

The cache tensors are the reference's, [num_blocks, block_size, kv_heads, head_dim] (demo/src/memory/paged_kv_cache.py:228),
and stay the caller's.  All calls run on the current stream of their tensors' device, never synchronise and can be
captured into CUDA graphs.  `status`, where given, is an int32 tensor of one element on the same device that the kernels
OR DEV_* bits into (include/b200moe.h); the caller zeroes and reads it.

A draft step's call is a few microseconds on the GPU, so the checks here read each attribute of a tensor once."""
from __future__ import annotations

from ctypes import byref, c_int64
from typing import Dict, Optional, Tuple, Union

import torch

from . import _lib
from ._lib import PagedAttentionArgs, StoreKvArgs, check
from .context import _DTYPE_TAG, _stream, dtype_tag

_WORKSPACE: Dict[Tuple, int] = {}
_INDEX_DTYPES = {torch.int64: 1, torch.int32: 0}


def _call(fn, args, dev: torch.device) -> None:
    """Launches on the current stream of `dev`; the library runs on the current device, so that is switched where needed."""
    if dev.index == torch.cuda.current_device():
        code = fn(byref(args), _stream(dev))
    else:
        with torch.cuda.device(dev):
            code = fn(byref(args), _stream(dev))
    if code:
        check(None, code)


def _tag(t: torch.Tensor, name: str) -> int:
    tag = _DTYPE_TAG.get(t.dtype)
    if tag is None:
        dtype_tag(t.dtype)     # raises
    if not t.is_cuda:
        raise ValueError(f"{name} must live on a CUDA device, got {t.device} (this package has no CPU path)")
    return tag


def _need(t: torch.Tensor, name: str, dev: torch.device, dtype: torch.dtype, dims: int):
    """Checks device, dtype and rank; returns the shape."""
    if t.device != dev:
        raise ValueError(f"{name} must live on {dev}, got {t.device} (this package has no CPU path)")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    shape = t.shape
    if len(shape) != dims:
        raise ValueError(f"{name} must have {dims} dimensions, got {tuple(shape)}")
    return shape


def _index(t: torch.Tensor, name: str, dev: torch.device, length: int) -> int:
    """Checks an index vector and returns 1 for int64, 0 for int32."""
    if t.device != dev:
        raise ValueError(f"{name} must live on {dev}, got {t.device} (this package has no CPU path)")
    kind = _INDEX_DTYPES.get(t.dtype)
    if kind is None:
        raise TypeError(f"{name} must be int64 or int32, got {t.dtype}")
    if t.shape != (length,) or (length > 1 and t.stride(0) != 1):
        raise ValueError(f"{name} must be contiguous of length {length}, got {tuple(t.shape)}")
    return kind


def _status_ptr(status: Optional[torch.Tensor], dev: torch.device) -> Optional[int]:
    if status is None:
        return None
    if status.device != dev or status.dtype != torch.int32 or status.numel() != 1:
        raise ValueError(f"status must be an int32 tensor of one element on {dev}")
    return status.data_ptr()


def _cache(k_cache: torch.Tensor, v_cache: torch.Tensor, dev: torch.device, dtype: torch.dtype, head_dim: int):
    """Checks the pair; returns shape and strides."""
    shape, strides = _need(k_cache, "k_cache", dev, dtype, 4), k_cache.stride()
    if _need(v_cache, "v_cache", dev, dtype, 4) != shape or v_cache.stride() != strides:
        raise ValueError("k_cache and v_cache must have the same shape and strides")
    if strides[3] != 1 or shape[3] != head_dim:
        raise ValueError(f"the caches must be [blocks, block_size, kv_heads, {head_dim}] with contiguous heads, got {tuple(shape)}")
    if shape[1] == 0:
        raise ValueError("the caches need a block size of at least one slot")
    return shape, strides


def _like(out: torch.Tensor, shape, dev: torch.device, dtype: torch.dtype):
    """Checks an output given by the caller; returns its strides."""
    strides = out.stride()
    if _need(out, "out", dev, dtype, 3) != shape or strides[2] != 1:
        raise ValueError(f"out must be {tuple(shape)} with contiguous heads, got {tuple(out.shape)}")
    return strides


def rotary_table(head_dim: int, max_position: int, base: float = 1e6, device: Optional[torch.device] = None) -> torch.Tensor:
    """The fp32 angle table [max_position, head_dim] that rope_store_kvcache takes: cos of the position's head_dim/2 angles,
    then sin.  Angles are formed in fp64, where a far position times a frequency still has all its digits."""
    inv = base ** (-torch.arange(0, head_dim, 2, dtype=torch.float64) / head_dim)
    angle = torch.arange(max_position, dtype=torch.float64)[:, None] * inv
    return torch.cat((angle.cos(), angle.sin()), dim=-1).float().to(device or "cpu")


def _store(query, key, value, positions, cos_sin, k_cache, v_cache, slot_mapping, q_norm_weight, k_norm_weight, eps, out, status):
    tag, dev, dt = _tag(key, "key"), key.device, key.dtype
    shape, ks, vs = _need(key, "key", dev, dt, 3), key.stride(), value.stride()
    if _need(value, "value", dev, dt, 3) != shape:
        raise ValueError(f"key and value must have the same shape, got {tuple(shape)} and {tuple(value.shape)}")
    T, hk, D = shape
    cshape, cs = _cache(k_cache, v_cache, dev, dt, D)
    if cshape[2] != hk:
        raise ValueError(f"the caches hold {cshape[2]} key-value heads, key and value {hk}")
    slots64 = _index(slot_mapping, "slot_mapping", dev, T)
    if ks[2] != 1 or vs[2] != 1:
        raise ValueError("heads must be contiguous")
    hq, qs, os_, q_ptr, o_ptr = 0, (0, 0), (0, 0), None, None
    if query is not None:
        qshape, qs = _need(query, "query", dev, dt, 3), query.stride()
        hq = qshape[1]
        if qshape[0] != T or qshape[2] != D or qs[2] != 1:
            raise ValueError(f"query must be [{T}, heads, {D}] with contiguous heads, got {tuple(qshape)}")
        if out is None:
            out = torch.empty(T, hq, D, dtype=dt, device=dev)
            os_ = (hq * D, D)
        else:
            os_ = _like(out, qshape, dev, dt)
        q_ptr, o_ptr = query.data_ptr(), out.data_ptr()
    pos_ptr = table_ptr = None
    pos64 = limit = 0
    if cos_sin is not None:
        limit, width = _need(cos_sin, "cos_sin", dev, torch.float32, 2)
        if width != D or not cos_sin.is_contiguous():
            raise ValueError(f"cos_sin must be a contiguous [positions, {D}], got {tuple(cos_sin.shape)}")
        pos64 = _index(positions, "positions", dev, T)
        pos_ptr, table_ptr = positions.data_ptr(), cos_sin.data_ptr()
    qw = kw = None
    if q_norm_weight is not None:
        if _need(q_norm_weight, "q_norm_weight", dev, dt, 1)[0] != D or not q_norm_weight.is_contiguous():
            raise ValueError(f"q_norm_weight must be a contiguous [{D}]")
        qw = q_norm_weight.data_ptr()
    if k_norm_weight is not None:
        if _need(k_norm_weight, "k_norm_weight", dev, dt, 1)[0] != D or not k_norm_weight.is_contiguous():
            raise ValueError(f"k_norm_weight must be a contiguous [{D}]")
        kw = k_norm_weight.data_ptr()
    _call(_lib.load().b200moe_store_kv,
          StoreKvArgs(q_ptr, key.data_ptr(), value.data_ptr(), o_ptr, k_cache.data_ptr(), v_cache.data_ptr(), pos_ptr, slot_mapping.data_ptr(),
                      table_ptr, qw, kw, None if status is None else _status_ptr(status, dev),
                      qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], os_[0], os_[1], cs[0], cs[1], cs[2],
                      T, hq, hk, D, cshape[0], cshape[1], limit, tag, pos64, slots64, eps, 0), dev)
    return out


def store_kvcache(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, slot_mapping: torch.Tensor, *,
                  status: Optional[torch.Tensor] = None) -> None:
    """key, value [T, kv_heads, D] -> rows slot_mapping[t] of the caches; slot -1 stores nothing (the reference's function of
    this name, demo/src/layers/attention.py:56-79).  The slots of one call are distinct."""
    _store(None, key, value, None, None, k_cache, v_cache, slot_mapping, None, None, 0.0, None, status)


def rope_store_kvcache(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor,
                       k_cache: torch.Tensor, v_cache: torch.Tensor, slot_mapping: torch.Tensor, *, q_norm_weight: Optional[torch.Tensor] = None,
                       k_norm_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, out: Optional[torch.Tensor] = None,
                       status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """What the reference's attention layer does between the projection and the attention, in one launch: per-head RMS norm
    of queries and keys (where weights are given), rotary embedding at `positions`, keys and values into the cache.

    query [T, heads, D], key and value [T, kv_heads, D] may be views of one projection row; cos_sin is rotary_table's.
    Returns the rotated queries [T, heads, D] (`out` when given, which may be `query` itself).  fp32 inside, each
    output rounded once."""
    if query is None or cos_sin is None or positions is None:
        raise ValueError("rope_store_kvcache needs query, positions and cos_sin (store_kvcache stores keys and values alone)")
    return _store(query, key, value, positions, cos_sin, k_cache, v_cache, slot_mapping, q_norm_weight, k_norm_weight, eps, out, status)


def _workspace_bytes(key: Tuple, dev: torch.device) -> int:
    n = c_int64(0)
    with torch.cuda.device(dev):
        check(None, _lib.load().b200moe_paged_attention_workspace(*key[:6], byref(n)))
    if len(_WORKSPACE) > 4096:
        _WORKSPACE.clear()
    _WORKSPACE[key] = n.value
    return n.value


def paged_attention(query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor, context_lens: torch.Tensor, *,
                    query_start: Optional[torch.Tensor] = None, max_query_len: Optional[int] = None, scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None, return_lse: bool = False,
                    status: Optional[torch.Tensor] = None) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Attention of new tokens over their sequences' cached keys and values (theirs included), causal within a span.

    query [T, heads, D]; block_tables int32 [B, max_blocks]; context_lens int32 [B].  Without query_start there is one token
    per sequence (T == B, the draft step); with it (int32 [B+1]) sequence b owns rows query_start[b]:query_start[b+1] and
    its last row sees all context_lens[b] keys (the verify step).  max_query_len, the longest span, picks the row tile; any
    value gives right results.  scale defaults to D ** -0.5.

    Returns out [T, heads, D] (with return_lse also the fp32 log-sum-exp [T, heads]).  A row that sees no key gives zeros
    and -inf; rows behind query_start[B] are not written (nor initialised unless `out` was given)."""
    tag, dev, dt = _tag(query, "query"), query.device, query.dtype
    shape, qs = _need(query, "query", dev, dt, 3), query.stride()
    T, hq, D = shape
    cshape, cs = _cache(k_cache, v_cache, dev, dt, D)
    blocks, page, hk, _ = cshape
    B, width = _need(block_tables, "block_tables", dev, torch.int32, 2)
    ts = block_tables.stride()
    if _need(context_lens, "context_lens", dev, torch.int32, 1)[0] != B or (B > 1 and context_lens.stride(0) != 1) or (width > 1 and ts[1] != 1):
        raise ValueError("block_tables [B, max_blocks] and context_lens [B] must be contiguous along their last dimension and agree in B")
    if qs[2] != 1:
        raise ValueError("heads must be contiguous")
    start_ptr, span = None, 1
    if query_start is not None:
        if _need(query_start, "query_start", dev, torch.int32, 1)[0] != B + 1 or query_start.stride(0) != 1:
            raise ValueError(f"query_start must be a contiguous [{B + 1}]")
        start_ptr = query_start.data_ptr()
        span = T if max_query_len is None else int(max_query_len)
        if span < 0:
            raise ValueError("max_query_len must not be negative")
    elif T != B:
        raise ValueError(f"without query_start there is one token per sequence, got {T} tokens for {B} sequences")
    if out is None:
        out = torch.empty(T, hq, D, dtype=dt, device=dev)
        os_ = (hq * D, D)
    else:
        os_ = _like(out, shape, dev, dt)
    lse = torch.empty(T, hq, dtype=torch.float32, device=dev) if return_lse else None
    # the workspace belongs to this call: calls on several streams and captured graphs do not share one
    key = (tag, hq, hk, D, span, width * page, dev.index)
    need = _WORKSPACE.get(key)
    if need is None:
        need = _workspace_bytes(key, dev)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _call(_lib.load().b200moe_paged_attention,
          PagedAttentionArgs(query.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_tables.data_ptr(), context_lens.data_ptr(), start_ptr,
                             out.data_ptr(), None if lse is None else lse.data_ptr(), None if ws is None else ws.data_ptr(),
                             None if status is None else _status_ptr(status, dev), need, qs[0], qs[1], os_[0], os_[1], cs[0], cs[1], cs[2], ts[0],
                             T, B, hq, hk, D, blocks, page, width, span, tag, D ** -0.5 if scale is None else scale, 0), dev)
    return (out, lse) if return_lse else out
