"""Operators for several continuations of one prompt: attention of queries that share cached rows, and copies of cached rows
between sequences."""
from __future__ import annotations

import ctypes as C

import numpy as np
import torch

from . import _lib

_FORMATS = {torch.float16: _lib.ACT_F16, torch.bfloat16: _lib.ACT_BF16, torch.float32: _lib.ACT_F32}


def _index(t: torch.Tensor | None, n: int, name: str, device, dtype=torch.int32) -> int | None:
    if t is None:
        return None
    if t.dtype != dtype or t.dim() != 1 or t.shape[0] != n or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {str(dtype)[6:]} tensor of {n} values on the queries' device")
    return t.data_ptr()


def prefix_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, group_first: torch.Tensor | None = None,
                     group_seq: torch.Tensor | None = None, group_len: torch.Tensor | None = None,
                     item_seq: torch.Tensor | None = None, item_begin: torch.Tensor | None = None,
                     item_end: torch.Tensor | None = None, *, scale: float | None = None, max_group: int | None = None,
                     max_prefix: int | None = None, max_own: int | None = None, skip: torch.Tensor | None = None,
                     out: torch.Tensor | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of query items [n_items, heads, dim] over a cache [n_seqs, kv_heads, rows, dim].

    Items ``group_first[g] .. group_first[g + 1] - 1`` share rows ``[0, group_len[g])`` of sequence ``group_seq[g]``; item i
    also sees rows ``[item_begin[i], item_end[i])`` of sequence ``item_seq[i]`` (by default sequence i from row 0).  The groups
    cover the items one after the other; without ``group_first`` nothing is shared, without ``item_end`` no item has rows
    of its own.  Indices are int32 tensors on the device, read when the kernels run.  ``skip`` (uint8) marks items that get
    zeros, as those that see no row do.  The ``max_*`` are upper bounds of what the tensors hold and only plan the work, but
    ``max_group``: no group may have more items.  ``status`` (int32, one value) becomes non-zero when an index is outside the
    cache.  The queries may be rows of a wider matrix; all else is contiguous.  Runs on the current stream."""
    if q.dim() != 3 or k.dim() != 4 or k.shape != v.shape or k.shape[3] != q.shape[2]:
        raise ValueError("queries are [items, heads, dim], keys and values [sequences, kv_heads, rows, dim]")
    dev = q.device
    if dev.type != "cuda" or k.device != dev or v.device != dev:
        raise ValueError("queries, keys and values must be on one CUDA device")
    if q.dtype not in _FORMATS or k.dtype not in _FORMATS or k.dtype != v.dtype:
        raise ValueError("prefix attention works on float16, bfloat16 and float32")
    n, heads, dim = q.shape
    seqs, kv, rows, _ = k.shape
    if not k.is_contiguous() or not v.is_contiguous():
        raise ValueError("keys and values must be contiguous")
    if q.stride(2) != 1 or (heads > 1 and q.stride(1) != dim):
        raise ValueError("an item's heads must be consecutive")
    if out is None:
        out = torch.empty((n, heads, dim), dtype=q.dtype, device=dev)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != dev or not out.is_contiguous():
        raise ValueError("out must be a contiguous tensor like the queries")
    if n == 0:
        return out
    groups = 0
    if group_first is not None:
        groups = group_first.shape[0] - 1 if group_first.dim() == 1 else -1
        if groups < 1 or group_seq is None or group_len is None:
            raise ValueError("groups need group_first, group_seq and group_len")
    for name, most in (("max_group", max_group), ("max_prefix", max_prefix), ("max_own", max_own)):
        if most is not None and most < 0:
            raise ValueError(f"{name} must not be negative")
    a = _lib.PrefixAttentionArgs(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
        _index(group_first, groups + 1, "group_first", dev), _index(group_seq, groups, "group_seq", dev) if groups else None,
        _index(group_len, groups, "group_len", dev) if groups else None, _index(item_seq, n, "item_seq", dev),
        _index(item_begin, n, "item_begin", dev), _index(item_end, n, "item_end", dev),
        _index(skip, n, "skip", dev, torch.uint8), _index(status, 1, "status", dev),
        None, 0, q.stride(0) if n > 1 else 0, groups, n, heads, kv, dim, seqs, rows,
        max_group or 0, max_prefix or 0, max_own or 0, dim ** -0.5 if scale is None else scale, _FORMATS[q.dtype], _FORMATS[k.dtype], 0)
    lib = _lib.load()
    ref = C.byref(a)
    if dev.index != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return _attend(lib, a, ref, dev, out)
    return _attend(lib, a, ref, dev, out)


def _attend(lib, a, ref, dev, out):
    need = lib.arcb_prefix_attention_scratch_bytes(ref)
    if need < 0:
        _lib.check(need)
    if need:
        # from the current stream's pool: free for the next call on it when this one's kernels are done
        scratch = torch.empty(need, dtype=torch.uint8, device=dev)
        a.d_scratch, a.scratch_bytes = scratch.data_ptr(), need
    _lib.check(lib.arcb_op_prefix_attention(ref, torch.cuda.current_stream(dev).cuda_stream))
    return out


def copy_cache_rows(cache: torch.Tensor, copies) -> None:
    """Copies rows between the sequences of ``cache`` [..., n_seqs, heads, rows, dim], in place: (src, dst, begin, end) takes rows
    ``[begin, end)`` of every plane and head of sequence ``src`` to the same rows of ``dst``.  ``copies``: any number of them, as
    a list or an integer array [n, 4] on the host.  All rows are read before any is written, so sequences may change places; no
    sequence may be written twice.  Runs on the current stream; ``copies`` may be changed after the call."""
    if cache.dim() < 4 or not cache.is_contiguous() or cache.device.type != "cuda":
        raise ValueError("the cache must be a contiguous CUDA tensor [..., n_seqs, heads, rows, dim]")
    m = np.asarray(copies)
    if m.size == 0:
        return
    if m.ndim != 2 or m.shape[1] != 4 or m.dtype.kind not in "iu":
        raise ValueError("copies are (src, dst, begin, end) in whole numbers")
    if m.dtype != np.int32:
        if m.min() < -1 or m.max() > 0x7fffffff:
            raise ValueError("a copy names a sequence or rows outside the cache")
        m = m.astype(np.int32)
    m = np.ascontiguousarray(m)
    seqs, heads, rows, dim = cache.shape[-4:]
    if cache.numel() == 0:
        raise ValueError("the cache is empty")
    planes = cache.numel() // (seqs * heads * rows * dim)
    lib = _lib.load()
    dev = cache.device
    args = (cache.data_ptr(), planes, seqs, heads, rows, dim * cache.element_size(), m.ctypes.data, len(m))
    if dev.index != torch.cuda.current_device():
        with torch.cuda.device(dev):
            _lib.check(lib.arcb_op_cache_copy(*args, torch.cuda.current_stream(dev).cuda_stream))
    else:
        _lib.check(lib.arcb_op_cache_copy(*args, torch.cuda.current_stream(dev).cuda_stream))
