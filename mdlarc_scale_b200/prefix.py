"""Operators for several continuations of one prompt: attention of queries that share cached rows, and copies of cached rows
between sequences."""
from __future__ import annotations

import struct

import numpy as np
import torch

from . import _lib

_FORMATS = {torch.float16: _lib.ACT_F16, torch.bfloat16: _lib.ACT_BF16, torch.float32: _lib.ACT_F32}


_I32, _U8 = torch.int32, torch.uint8
# The fields of _lib.PrefixAttentionArgs: packing them takes a sixth of filling the ctypes structure, which a call's time shows.
_ARGS = struct.Struct("@13P2q10if3i")
_SCRATCH, _SCRATCH_AT = struct.Struct("@Pq"), _lib.PrefixAttentionArgs.d_scratch.offset
_raw_stream = torch._C._cuda_getCurrentRawStream      # the current stream's handle; torch.cuda.current_stream() takes 2 us
_current_device = torch._C._cuda_getDevice             # of a process that has CUDA tensors: nothing is left to initialise


def _refuse_gradient():
    raise ValueError("there is no gradient of this operator: detach() what requires one, or call it under torch.no_grad()")


def _refuse_index(name: str, n: int):
    raise ValueError(f"{name} must be a contiguous int32 tensor (skip: uint8) of {n} values on the queries' device")


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
    zeros, as those that see no row do.  The ``max_*`` are upper bounds of what the tensors hold (None: as many as there can be) and
    only plan the work, but ``max_group``: no group may have more items.  ``status`` (int32, one value) becomes non-zero when an index is outside the
    cache.  Keys that an item sees are finite where half queries meet a bfloat16 cache (a query is a sum of two pieces there,
    which an infinity would turn into no number); what no item sees may hold anything.  The queries may be rows of a wider
    matrix; all else is contiguous.  Has no gradient, and refuses tensors that require one where it would be recorded.  Runs on the
    current stream."""
    if (q.requires_grad or k.requires_grad or v.requires_grad or (out is not None and out.requires_grad)) and torch.is_grad_enabled():
        _refuse_gradient()
    if q.dim() != 3 or k.dim() != 4 or k.shape != v.shape:
        raise ValueError("queries are [items, heads, dim], keys and values [sequences, kv_heads, rows, dim]")
    n, heads, dim = q.shape
    seqs, kv, rows, kv_dim = k.shape
    if kv_dim != dim:
        raise ValueError("queries and keys must have heads of the same size")
    dev = q.get_device()
    if dev < 0 or k.get_device() != dev or v.get_device() != dev:
        raise ValueError("queries, keys and values must be on one CUDA device")
    act, form = _FORMATS.get(q.dtype), _FORMATS.get(k.dtype)
    if act is None or form is None or k.dtype != v.dtype:
        raise ValueError("prefix attention works on float16, bfloat16 and float32")
    if not k.is_contiguous() or not v.is_contiguous():
        raise ValueError("keys and values must be contiguous")
    pitch = 0
    if not q.is_contiguous():
        if q.stride(2) != 1 or (heads > 1 and q.stride(1) != dim):
            raise ValueError("an item's heads must be consecutive")
        pitch = q.stride(0) if n > 1 else 0
        if pitch == 0 and n > 1:
            raise ValueError("every item has queries of its own (broadcast ones: contiguous())")
    if out is None:
        out = q.new_empty((n, heads, dim)) if pitch else torch.empty_like(q)
    elif out.shape != q.shape or out.dtype != q.dtype or out.get_device() != dev or not out.is_contiguous():
        raise ValueError("out must be a contiguous tensor like the queries")
    if n == 0:
        return out

    def index(t, size, name, dtype=_I32):
        if t is None:
            return 0
        if t.dtype is not dtype or t.numel() != size or t.get_device() != dev or not t.is_contiguous():
            _refuse_index(name, size)
        return t.data_ptr()

    groups = first = seq = length = 0
    if group_first is not None:
        groups = group_first.numel() - 1
        if groups < 1 or group_seq is None or group_len is None:
            raise ValueError("groups need group_first, group_seq and group_len")
        first, seq, length = index(group_first, groups + 1, "group_first"), index(group_seq, groups, "group_seq"), index(group_len, groups, "group_len")
    # to the library 0 is a bound that is not known; one of no rows plans for as few as there can be
    max_group, max_prefix, max_own = max_group or 0, 0 if max_prefix is None else max_prefix or 1, 0 if max_own is None else max_own or 1
    if max_group < 0 or max_prefix < 0 or max_own < 0:
        raise ValueError("max_group, max_prefix and max_own must not be negative")
    fields = (
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), first, seq, length, index(item_seq, n, "item_seq"), index(item_begin, n, "item_begin"),
        index(item_end, n, "item_end"), index(skip, n, "skip", _U8), index(status, 1, "status"), 0, 0, pitch, groups, n, heads, kv, dim, seqs, rows,
        max_group, max_prefix, max_own, dim ** -0.5 if scale is None else scale, act, form, 0)
    try:
        a = _ARGS.pack(*fields)
    except (struct.error, OverflowError):
        raise ValueError("scale, max_group, max_prefix and max_own must be numbers of 32 bits") from None
    if dev != _current_device():
        with torch.cuda.device(dev):
            _attend(a, out, dev)
    else:
        _attend(a, out, dev)
    return out


def _attend(a: bytes, out: torch.Tensor, dev: int) -> None:
    lib = _lib.load()
    need = lib.arcb_prefix_attention_scratch_bytes(a)
    if need > 0:
        # from the current stream's pool: free for the next call on it when this one's kernels are done
        scratch = torch.empty(need, dtype=_U8, device=out.device)
        a = a[:_SCRATCH_AT] + _SCRATCH.pack(scratch.data_ptr(), need) + a[_SCRATCH_AT + _SCRATCH.size:]
    code = need if need < 0 else lib.arcb_op_prefix_attention(a, _raw_stream(dev))
    if code:
        _lib.check(code)


def copy_cache_rows(cache: torch.Tensor, copies) -> None:
    """Copies rows between the sequences of ``cache`` [..., n_seqs, heads, rows, dim], in place: (src, dst, begin, end) takes rows
    ``[begin, end)`` of every plane and head of sequence ``src`` to the same rows of ``dst``.  ``copies``: any number of them, as
    a list or an integer array [n, 4] on the host.  All rows are read before any is written, so sequences may change places; no
    sequence may be written twice.  Has no gradient, and refuses a cache that requires one where it would be recorded.  Runs on the
    current stream; ``copies`` may be changed after the call."""
    if cache.requires_grad and torch.is_grad_enabled():
        _refuse_gradient()
    dev = cache.get_device()
    if cache.dim() < 4 or dev < 0 or not cache.is_contiguous():
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
    total = cache.numel()
    if total == 0:
        raise ValueError("the cache is empty")
    args = (cache.data_ptr(), total // (seqs * heads * rows * dim), seqs, heads, rows, dim * cache.element_size(), m.ctypes.data, len(m), _raw_stream(dev))
    lib = _lib.load()
    if dev != _current_device():
        with torch.cuda.device(dev):
            code = lib.arcb_op_cache_copy(*args)
    else:
        code = lib.arcb_op_cache_copy(*args)
    if code:
        _lib.check(code)
