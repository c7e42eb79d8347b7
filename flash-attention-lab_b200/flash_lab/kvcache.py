"""The KV cache of a serving loop: append_kv writes new tokens, extend attends a chunk of new tokens
to it, gather_kv reads it back, and flash_lab.decode serves single tokens. No counterpart in the
reference, whose decode reads a cache that something else has filled.

A cache is [B, S_max, H_kv, D], or paged [num_blocks, page_size, H_kv, D] with block_tables
[B, max_blocks] int32, of the tokens' dtype or int8. An int8 cache holds one fp32 scale per token
and KV head in k_scale / v_scale, [B, S_max, H_kv] or [num_blocks, page_size, H_kv] with any
strides: the row x of one token and head is stored as round(x * 127 / max|x|) and max|x| / 127
(2^-100 at least; the attention kernels read a smaller or negative v_scale as that, and one above 2^127
as NaN). The attention kernels read scales along the keys of one head, so scales stored head by head
(`torch.empty(blocks, H_kv, page_size).transpose(1, 2)`) are read with wider loads.

New rows are ragged: [T, H, D] with cu_seqlens [B + 1] int32, where sequence b owns rows
cu_seqlens[b] .. cu_seqlens[b + 1] - 1, or [B, n, H, D] / [B, H, D] with the same count for every
sequence. seq_lens [B] int32 counts the keys of each sequence including its new rows, which are
its last ones. Offsets, lengths and block tables are read on the device only (no host sync), so
every call can be captured in a CUDA graph.
"""

from __future__ import annotations

import ctypes
import math

import torch

from flash_lab import _capi, ops
from flash_lab.layouts import _check_heads, _require_tensor, check_cache_inputs, ragged_rows

_DTYPE_CODE = {**ops._DECODE_DTYPE_CODE, torch.int8: _capi.FLB_INT8}
_HALF = (torch.bfloat16, torch.float16)
_ROW_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
_HEAD_DIMS = (64, 128)
_MAX_GROUP = 128   # query heads per KV head that extend takes

_APPEND_SCHEMA = ("(Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor seq_lens, "
                  "Tensor? cu_seqlens, Tensor? block_tables, Tensor(c!)? k_scale, "
                  "Tensor(d!)? v_scale, int rows_per_seq) -> ()")
_GATHER_SCHEMA = ("(Tensor k_cache, Tensor v_cache, Tensor seq_lens, Tensor cu_seqlens, "
                  "Tensor? block_tables, Tensor? k_scale, Tensor? v_scale, int total, "
                  "ScalarType dtype) -> (Tensor, Tensor)")
_EXTEND_SCHEMA = ("(Tensor q, Tensor k_cache, Tensor v_cache, Tensor seq_lens, Tensor? cu_seqlens, "
                  "Tensor? block_tables, Tensor? k_scale, Tensor? v_scale, int rows_per_seq, "
                  "bool causal, float softmax_scale) -> (Tensor, Tensor)")


# ------------------------------------------------------------------------------------------------
# Op implementations (CUDA dispatch key)
# ------------------------------------------------------------------------------------------------

def _ptr(x) -> int:
    return 0 if x is None else x.data_ptr()


def _expanded(x, dims) -> bool:
    """Whether a dimension of x, among dims, repeats the same memory."""
    return any(x.shape[i] > 1 and x.stride(i) == 0 for i in dims)


def _cache_struct(k_cache, v_cache, seq_lens, block_tables, k_scale, v_scale):
    paged = block_tables is not None
    return _capi.KVCache(
        k_cache.data_ptr(), v_cache.data_ptr(), *k_cache.stride()[:3], *v_cache.stride()[:3],
        _ptr(k_scale), _ptr(v_scale),
        *((0, 0, 0) if k_scale is None else k_scale.stride()),
        *((0, 0, 0) if v_scale is None else v_scale.stride()),
        _ptr(block_tables), block_tables.stride(0) if paged else 0,
        k_cache.shape[1] if paged else 0, k_cache.shape[0] if paged else 0,
        seq_lens.shape[0], k_cache.shape[2], k_cache.shape[3],
        block_tables.shape[1] * k_cache.shape[1] if paged else k_cache.shape[1],
        _DTYPE_CODE[k_cache.dtype])


def _rows_struct(k, v, cu_seqlens, seq_lens, rows_per_seq):
    return _capi.KVRows(k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), v.stride(0),
                        v.stride(1), _ptr(cu_seqlens), seq_lens.data_ptr(), k.shape[0],
                        rows_per_seq, _DTYPE_CODE[k.dtype])


def _append(k, v, k_cache, v_cache, seq_lens, cu_seqlens, block_tables, k_scale, v_scale,
            rows_per_seq: int):
    lib = ops._require_library()
    if ops._NATIVE is not None:
        ops._NATIVE.kv_append(k, v, k_cache, v_cache, seq_lens, cu_seqlens, block_tables, k_scale,
                              v_scale, int(rows_per_seq))
    else:
        cache = _cache_struct(k_cache, v_cache, seq_lens, block_tables, k_scale, v_scale)
        rows = _rows_struct(k, v, cu_seqlens, seq_lens, rows_per_seq)
        with ops._DeviceGuard(k.device):
            status = lib.flb_kv_append(ctypes.byref(cache), ctypes.byref(rows),
                                       ops._raw_stream(k.device))
        ops._check(status, "flb_kv_append", k.device)
        for x in (k_cache, v_cache, k_scale, v_scale):
            if x is not None and not x.is_inference():
                torch.autograd.graph.increment_version(x)


def _gather(k_cache, v_cache, seq_lens, cu_seqlens, block_tables, k_scale, v_scale, total: int,
            dtype: torch.dtype):
    lib = ops._require_library()
    if ops._NATIVE is not None:
        return ops._NATIVE.kv_gather(k_cache, v_cache, seq_lens, cu_seqlens, block_tables, k_scale,
                                     v_scale, int(total), dtype)
    shape = (total, k_cache.shape[2], k_cache.shape[3])
    k = torch.empty(shape, dtype=dtype, device=k_cache.device)
    v = torch.empty(shape, dtype=dtype, device=k_cache.device)
    cache = _cache_struct(k_cache, v_cache, seq_lens, block_tables, k_scale, v_scale)
    rows = _rows_struct(k, v, cu_seqlens, seq_lens, 0)
    with ops._DeviceGuard(k_cache.device):
        status = lib.flb_kv_gather(ctypes.byref(cache), ctypes.byref(rows),
                                   ops._raw_stream(k_cache.device))
    ops._check(status, "flb_kv_gather", k_cache.device)
    return k, v


def _extend(q, k_cache, v_cache, seq_lens, cu_seqlens, block_tables, k_scale, v_scale,
            rows_per_seq: int, causal: bool, softmax_scale: float):
    lib = ops._require_library()
    if ops._NATIVE is not None:
        o, lse = ops._NATIVE.extend(q, k_cache, v_cache, seq_lens, cu_seqlens, block_tables,
                                    k_scale, v_scale, int(rows_per_seq), bool(causal),
                                    float(softmax_scale), ops._status_ptr(q.device),
                                    ops._sm_count(q.device))
        if ops.DEBUG:
            ops._check(_capi.FLB_OK, "flb_extend_fwd", q.device)
        return o, lse
    if _expanded(q, (0, 1)):
        q = q.contiguous()
    rows, heads, head_dim = q.shape
    o = torch.empty((rows, heads, head_dim), dtype=q.dtype, device=q.device)
    lse = torch.empty((rows, heads), dtype=torch.float32, device=q.device)
    nbytes = lib.flb_extend_workspace_bytes(rows, heads, k_cache.shape[2], head_dim,
                                            ops._sm_count(q.device))
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
    cache = _cache_struct(k_cache, v_cache, seq_lens, block_tables, k_scale, v_scale)
    p = _capi.ExtendParams(
        q.data_ptr(), o.data_ptr(), lse.data_ptr(), q.stride(0), q.stride(1), o.stride(0),
        o.stride(1), _ptr(cu_seqlens), seq_lens.data_ptr(), rows, rows_per_seq, heads,
        1 if causal else 0, _DTYPE_CODE[q.dtype], float(softmax_scale), workspace.data_ptr(),
        nbytes, ops._status_ptr(q.device))
    with ops._DeviceGuard(q.device):
        status = lib.flb_extend_fwd(ctypes.byref(cache), ctypes.byref(p),
                                    ops._raw_stream(q.device))
    ops._check(status, "flb_extend_fwd", q.device)
    return o, lse


def _append_fake(k, v, k_cache, v_cache, seq_lens, cu_seqlens, block_tables, k_scale, v_scale,
                 rows_per_seq):
    return None


def _gather_fake(k_cache, v_cache, seq_lens, cu_seqlens, block_tables, k_scale, v_scale, total,
                 dtype):
    shape = (total, k_cache.shape[2], k_cache.shape[3])
    return k_cache.new_empty(shape, dtype=dtype), k_cache.new_empty(shape, dtype=dtype)


def _extend_fake(q, k_cache, v_cache, seq_lens, cu_seqlens, block_tables, k_scale, v_scale,
                 rows_per_seq, causal, softmax_scale):
    return q.new_empty(q.shape), q.new_empty(q.shape[:2], dtype=torch.float32)


if ops.HAS_EXTENSION:
    ops._define("kv_append", _APPEND_SCHEMA, _append, _append_fake)
    ops._define("kv_gather", _GATHER_SCHEMA, _gather, _gather_fake)
    ops._define("extend_sm100", _EXTEND_SCHEMA, _extend, _extend_fake)


# ------------------------------------------------------------------------------------------------
# Public entry points
# ------------------------------------------------------------------------------------------------

def _require_kernels(device: torch.device) -> None:
    if device.type != "cuda":
        raise ValueError(f"flash_lab kernels take CUDA tensors, got device {device}")
    ops._require_library()


def _check_head_dim(head_dim: int) -> None:
    if head_dim not in _HEAD_DIMS:
        raise ValueError(f"head_dim {head_dim} is not one of {_HEAD_DIMS}")


def _fast_binding():
    """The PyTorch binding when a plain eager call may use its record of checked calls: calls with
    the metadata of one that passed the checks below run without them (binding/torch_ops.cpp)."""
    return ops._NATIVE if ops._NATIVE is not None and not ops.DEBUG and ops._plain_eager() else None


def append_kv(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
              seq_lens: torch.Tensor, cu_seqlens: torch.Tensor | None = None,
              block_tables: torch.Tensor | None = None, k_scale: torch.Tensor | None = None,
              v_scale: torch.Tensor | None = None) -> None:
    """Writes new tokens' K and V into a cache, in place.

    k and v are [T, H_kv, D] with cu_seqlens, or [B, n, H_kv, D] / [B, H_kv, D]; with n new rows,
    row i of sequence b becomes key seq_lens[b] - n + i. An int8 cache is quantised as it is
    written (bf16, fp16 or fp32 rows); any other cache has the rows' dtype. Rows whose position
    lies outside the cache, whose page is not a block of the pool, or that belong to no sequence
    are skipped. Two rows that name the same cache row race.
    """
    args = (k, v, k_cache, v_cache, seq_lens, cu_seqlens, block_tables, k_scale, v_scale)
    fast = _fast_binding()
    if fast is not None and fast.append_fast(*args):
        return
    shape = check_cache_inputs(k_cache, v_cache, seq_lens, block_tables, k_scale, v_scale,
                               cu_seqlens, {"k": k, "v": v})
    for name, x in (("k_cache", k_cache), ("v_cache", v_cache), ("k_scale", k_scale),
                    ("v_scale", v_scale)):
        if x is not None and _expanded(x, range(x.dim())):
            raise ValueError(f"{name} is written and must not be expanded, got strides "
                             f"{tuple(x.stride())} for shape {tuple(x.shape)}")
    if k.shape != v.shape:
        raise ValueError(f"k and v must have the same shape, got {tuple(k.shape)} and "
                         f"{tuple(v.shape)}")
    if k.dtype != v.dtype or k.dtype not in _ROW_DTYPES or \
            not (shape.int8 or k.dtype == k_cache.dtype):
        raise TypeError(f"k and v must share the cache's dtype (any of {_ROW_DTYPES} for an "
                        f"int8 cache), got {k.dtype}, {v.dtype} and {k_cache.dtype}")
    k3, per_seq = ragged_rows("k", k, shape.batch, cu_seqlens)
    v3, _ = ragged_rows("v", v, shape.batch, cu_seqlens)
    if k3.shape[1:] != k_cache.shape[2:]:
        raise ValueError(f"k and v rows are {tuple(k3.shape[1:])} (heads, head_dim), the "
                         f"cache's {tuple(k_cache.shape[2:])}")
    _check_head_dim(shape.head_dim)
    _require_kernels(k.device)
    ops._call_op("kv_append", k3, v3, k_cache, v_cache, seq_lens, cu_seqlens, block_tables, k_scale,
                 v_scale, per_seq)
    if fast is not None:
        fast.append_known(*args)


def gather_kv(k_cache: torch.Tensor, v_cache: torch.Tensor, seq_lens: torch.Tensor,
              cu_seqlens: torch.Tensor, total: int, block_tables: torch.Tensor | None = None,
              k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
              dtype: torch.dtype | None = None):
    """Reads sequences back from a cache: (k, v), each [total, H_kv, D].

    Row cu_seqlens[b] + i is key i of sequence b, for i below cu_seqlens[b + 1] - cu_seqlens[b].
    Keys at or past seq_lens[b], rows of no sequence and pages that are not blocks of the pool
    give zeros. `total` (host int) is the number of rows to return, cu_seqlens[B] or more. An int8
    cache is read back as `dtype` (bf16 unless given); any other cache has its own dtype.
    """
    args = (k_cache, v_cache, seq_lens, cu_seqlens, total, block_tables, k_scale, v_scale, dtype)
    fast = _fast_binding() if isinstance(total, int) else None
    if fast is not None:
        done = fast.gather_fast(*args)
        if done is not None:
            return done
    shape = check_cache_inputs(k_cache, v_cache, seq_lens, block_tables, k_scale, v_scale, cu_seqlens)
    if cu_seqlens is None:
        raise TypeError("cu_seqlens must be a torch.Tensor, got NoneType")
    if not hasattr(type(total), "__index__"):
        raise TypeError(f"total must be an int, got {type(total).__name__}")
    if total < 1:
        raise ValueError(f"total must be positive, got {total}")
    out = dtype if dtype is not None else torch.bfloat16 if shape.int8 else k_cache.dtype
    if out not in _ROW_DTYPES or not (shape.int8 or out == k_cache.dtype):
        raise TypeError(f"dtype must be the cache's own (any of {_ROW_DTYPES} for an int8 "
                        f"cache), got {out} and {k_cache.dtype}")
    _check_head_dim(shape.head_dim)
    _require_kernels(k_cache.device)
    done = ops._call_op("kv_gather", k_cache, v_cache, seq_lens, cu_seqlens, block_tables, k_scale,
                        v_scale, total, out)
    if fast is not None:
        fast.gather_known(*args)
    return done


def extend(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, seq_lens: torch.Tensor,
           cu_seqlens: torch.Tensor | None = None, block_tables: torch.Tensor | None = None,
           causal: bool = True, softmax_scale: float | None = None,
           k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
           return_lse: bool = False):
    """Attention of a chunk of new tokens per sequence over a cache that already holds their K and
    V (append_kv first): chunked prefill, speculative tokens, or a batch that mixes prompt chunks
    and single tokens.

    q is [T, H, D] with cu_seqlens, or [B, n, H, D] / [B, H, D] (bf16 or fp16, H % H_kv == 0); the
    cache has q's dtype or is int8 with k_scale and v_scale. With n new rows, row i of sequence b sees
    keys 0 .. seq_lens[b] - n + i (all seq_lens[b] keys when causal is False). seq_lens values are
    clamped to [0, S_max] on the device. Paged caches take pages of 8, 16, 32 or a multiple of 64
    rows. Caches may be expanded over sequences or KV heads (a prefix that all sequences share);
    a q expanded over rows or heads is copied.

    Returns o in q's shape and dtype and, with return_lse=True, the natural-log log-sum-exp of
    each score row as fp32 in q's shape without its last dimension. Rows that see no key, or
    belong to no sequence, give zeros and -inf. One call takes at most 16384 sequences and 128
    query heads per KV head. A non-finite value in V makes the whole tile of up to 128 keys around
    it non-finite for every row that reads the tile, also for rows that the causal mask keeps from
    that key (int8 caches: only for the rows that see it); keys at or past seq_lens[b] are never
    read into a result. A call gives the same bits each time; over an int8 cache the same rows given with
    cu_seqlens and without it may be worked by different kernels and differ in their last bits.
    """
    out, lse = _extend_checked(0, q, k_cache, v_cache, seq_lens, cu_seqlens, block_tables, causal,
                               softmax_scale, k_scale, v_scale)
    return (out, lse) if return_lse else out


def _extend_checked(entry, q, k_cache, v_cache, seq_lens, cu_seqlens, block_tables, causal,
                    softmax_scale, k_scale, v_scale):
    """extend (entry 0) and decode over an int8 cache (entry 1): o and lse in q's shapes."""
    _require_tensor("q", q)
    if entry == 1 and q.dim() == 4 and q.shape[1] != 1:
        raise ValueError(f"decode takes one query token per sequence, got q {tuple(q.shape)}")
    scale = softmax_scale if softmax_scale is not None else 1.0 / math.sqrt(max(q.shape[-1], 1))
    causal = bool(causal)
    args = (q, k_cache, v_cache, seq_lens, cu_seqlens, block_tables, k_scale, v_scale, causal, scale)
    fast = _fast_binding()
    if fast is not None:
        done = fast.extend_fast(entry, *args)
        if done is not None:
            return done
    shape = check_cache_inputs(k_cache, v_cache, seq_lens, block_tables, k_scale, v_scale,
                               cu_seqlens, {"q": q})
    if q.dtype not in _HALF or not (shape.int8 or q.dtype == k_cache.dtype):
        raise TypeError(f"q must be one of {_HALF} and the cache q's dtype or int8, got "
                        f"{q.dtype} and {k_cache.dtype}")
    q3, per_seq = ragged_rows("q", q, shape.batch, cu_seqlens)
    if q3.shape[2] != shape.head_dim:
        raise ValueError(f"head_dim mismatch: q has {q3.shape[2]}, the cache has {shape.head_dim}")
    _check_heads(q3.shape[1], shape.heads_kv)
    if q3.shape[1] // shape.heads_kv > _MAX_GROUP:
        raise ValueError(f"at most {_MAX_GROUP} query heads per KV head, got "
                         f"{q3.shape[1]} and {shape.heads_kv}")
    if shape.page_size and not (shape.page_size in (8, 16, 32) or shape.page_size % 64 == 0):
        raise ValueError(f"page_size {shape.page_size} is not 8, 16, 32 or a multiple of 64")
    if _expanded(k_cache, (1,)) or _expanded(v_cache, (1,)):
        raise ValueError("caches must not be expanded along their keys")
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"softmax_scale must be positive, got {scale}")
    _check_head_dim(shape.head_dim)
    _require_kernels(q.device)
    out, lse = ops._call_op("extend_sm100", q3, k_cache, v_cache, seq_lens, cu_seqlens,
                            block_tables, k_scale, v_scale, per_seq, causal, scale)
    if q.dim() == 4:
        out, lse = out.view(q.shape), lse.view(q.shape[:3])
    if fast is not None:
        status = ops._status_ptr(q.device)
        if status:   # none: the first call of a device, under capture; recorded when it has one
            fast.extend_known(entry, *args, status, ops._sm_count(q.device))
    return out, lse


def decode_int8(q, k_cache, v_cache, seq_lens, block_tables, softmax_scale, k_scale, v_scale,
                return_lse: bool):
    """flash_lab.decode over an int8 cache: the one-row form of extend, with decode's shapes (q
    [B, 1, H, D] or [B, H, D], lse [B, H])."""
    out, lse = _extend_checked(1, q, k_cache, v_cache, seq_lens, None, block_tables, True,
                               softmax_scale, k_scale, v_scale)
    if not return_lse:
        return out
    return out, lse.flatten(1) if q.dim() == 4 else lse
