"""Decode attention of a batch whose sequences share leading pages.

``SharedPrefixPlan`` takes what ``DecodePlan`` takes and computes the same
attention, but the pages that several sequences start with are attended to
once for all of them: per KV head, the group's queries are one matrix against
the prefix.  The other pages go through the decode kernel, and both parts
meet by their softmax statistics.
"""
from __future__ import annotations

import ctypes
import operator

import numpy as np

from . import _native
from .layout import Layout, validate_metadata
from .rotary import _cuda_device, _dtype_code, _int32
from .runtime import _check_limits

__all__ = ["SharedPrefixPlan", "find_prefixes", "inspect_prefix_plan"]


def _native_plan(layout, table, lengths, prefixes, max_lengths, code, device_index, find=-1):
    lib = _native.load()
    c_layout = _native.Layout(layout.batch, layout.query_heads, layout.kv_heads, layout.head_dim,
                              layout.page_size, layout.physical_pages)
    table = np.ascontiguousarray(table, dtype=np.int32)
    lengths = np.ascontiguousarray(lengths, dtype=np.int32)
    if max_lengths is not None:
        max_lengths = np.ascontiguousarray(max_lengths, dtype=np.int32)
    count, arrays = find, [None, None, None]
    if prefixes is not None:
        prefixes = list(prefixes)
        members = [np.asarray(m) for m, _ in prefixes]
        pages = [p for _, p in prefixes]
        try:
            if any(isinstance(p, bool) for p in pages):
                raise TypeError
            pages = np.asarray([operator.index(p) for p in pages], dtype=np.int64)
            if any(m.ndim != 1 or (m.size and m.dtype.kind not in "iu") for m in members):
                raise TypeError
        except TypeError:
            raise TypeError("prefixes must be pairs (sequence indices, pages)") from None
        sizes = [m.size for m in members]
        if any(((m < 0) | (m >= layout.batch)).any() for m in members):
            raise ValueError("prefix group names a sequence outside the batch")
        if ((pages < 1) | (pages > table.shape[1])).any():
            raise ValueError("a prefix must have 1 .. table width pages")
        count = len(sizes)
        arrays = [np.concatenate(([0], np.cumsum(sizes))).astype(np.int32),
                  np.concatenate(members or [np.empty(0)]).astype(np.int32), pages.astype(np.int32)]
    handle = ctypes.c_void_p()
    status = lib.pd_prefix_plan_create(
        ctypes.byref(c_layout), table.ctypes.data, table.shape[1], lengths.ctypes.data,
        None if max_lengths is None else max_lengths.ctypes.data, count,
        *(None if x is None else x.ctypes.data for x in arrays), code, device_index, ctypes.byref(handle))
    _native.check(status, "prefix plan")
    return handle


def _groups(lib, handle, batch):
    """(pd_prefix_info, [(sequence indices, pages)])."""
    info = _native.PrefixInfo()
    _native.check(lib.pd_prefix_plan_get_info(handle, ctypes.byref(info)))
    group, pages = np.empty(batch, dtype=np.int32), np.empty(max(info.groups, 1), dtype=np.int32)
    _native.check(lib.pd_prefix_plan_copy_groups(handle, group.ctypes.data, pages.ctypes.data))
    return info, [(np.flatnonzero(group == g), int(pages[g])) for g in range(info.groups)]


def _named_dtype_code(dtype):
    """The library's code of "float16" or torch.float16, .. (torch need not be there)."""
    code = {"float16": _native.PD_FLOAT16, "float32": _native.PD_FLOAT32}.get(str(dtype).removeprefix("torch."))
    if code is None:
        raise TypeError("dtype must be float16 or float32")
    return code


def _check_max_lengths(max_lengths, layout, table, lengths):
    max_lengths = np.asarray(max_lengths)
    if max_lengths.shape != lengths.shape or max_lengths.dtype.kind not in "iu":
        raise ValueError("max_lengths must be integers of shape [batch]")
    if (max_lengths < lengths).any() or (max_lengths > table.shape[1] * layout.page_size).any():
        raise ValueError("max_lengths must lie between lengths and the page table capacity")
    return max_lengths


def find_prefixes(layout: Layout, table, lengths, *, dtype="float16"):
    """The groups of sequences that start with the same pages, [(sequence indices, pages)].

    Each group is all sequences with some leading pages in common, chosen so that the page reads
    that sharing saves are the most.  No GPU needed; a plan uses them by itself only where they
    save enough.
    """
    _check_limits(layout, 256, "serial")
    table, lengths = validate_metadata(layout, table, lengths)
    lib = _native.load()
    code = _named_dtype_code(dtype)
    handle = _native_plan(layout, table, lengths, None, None, code, -1, find=-2)
    try:
        return _groups(lib, handle, layout.batch)[1]
    finally:
        lib.pd_prefix_plan_destroy(handle)


def inspect_prefix_plan(layout: Layout, table, lengths, *, prefixes=None, dtype="float16", max_lengths=None):
    """A host-only plan's (info, groups, work items) as pd_prefix_plan_copy_items lays them out (no GPU needed)."""
    _check_limits(layout, 256, "serial")
    table, lengths = validate_metadata(layout, table, lengths)
    if max_lengths is not None:
        max_lengths = _check_max_lengths(max_lengths, layout, table, lengths)
    lib = _native.load()
    code = _named_dtype_code(dtype)
    handle = _native_plan(layout, table, lengths, prefixes, max_lengths, code, -1)
    try:
        info, groups = _groups(lib, handle, layout.batch)
        items = np.empty((info.items, info.item_words), dtype=np.int32)
        _native.check(lib.pd_prefix_plan_copy_items(handle, items.ctypes.data))
    finally:
        lib.pd_prefix_plan_destroy(handle)
    return {name: getattr(info, name) for name, _ in info._fields_}, groups, items


class SharedPrefixPlan:
    """A decode plan that computes shared leading pages once.

    ``layout``, ``table`` and ``lengths`` as for ``DecodePlan``.  ``prefixes``
    lists the groups as (sequence indices, pages): each sequence in at most one
    group, whose first ``pages`` pages are the same and whole in all of them;
    None takes those of ``find_prefixes`` that make a call shorter by the plan's
    estimate (the decode kernel reads the copies of a short prefix from L2 in less time), []
    shares nothing.  ``max_lengths`` makes a dynamic plan (``run_dynamic``).  ``run``
    returns the plan's own [batch, query_heads, head_dim] output in ``dtype``
    (the inputs' type; sums are FP32), which the next run overwrites.  Launch a
    plan from one stream at a time.
    """

    def __init__(self, layout: Layout, table, lengths, *, prefixes=None, dtype=None, device="cuda",
                 max_lengths=None):
        import torch
        dtype = torch.float16 if dtype is None else dtype
        self._code = _dtype_code(dtype, "q/k/v")
        _check_limits(layout, 256, "serial")
        table, lengths = validate_metadata(layout, table, lengths)
        if max_lengths is not None:
            max_lengths = _check_max_lengths(max_lengths, layout, table, lengths)
        self.layout, self.dtype, self.max_lengths = layout, dtype, max_lengths
        self.device = _cuda_device(device)
        self._lib = _native.load()
        self._width = table.shape[1]
        self._handle = _native_plan(layout, table, lengths, prefixes, max_lengths, self._code, self.device.index)
        self.info, self.prefixes = _groups(self._lib, self._handle, layout.batch)
        self._buffer = torch.empty(int(self._lib.pd_prefix_plan_device_bytes(self._handle)), dtype=torch.uint8,
                                   device=self.device)
        _native.check(self._lib.pd_prefix_plan_bind(
            self._handle, self._buffer.data_ptr(), self._buffer.numel(),
            torch.cuda.current_stream(self.device).cuda_stream), "bind")
        self._q_shape = (layout.batch, layout.query_heads, layout.head_dim)
        self._k_shape = (layout.physical_pages, layout.page_size, layout.kv_heads, layout.head_dim)
        self._out = torch.empty(self._q_shape, dtype=dtype, device=self.device)
        self._index = self.device.index

    def __del__(self):
        handle = getattr(self, "_handle", None)
        if handle:
            self._lib.pd_prefix_plan_destroy(handle)
            self._handle = None

    @property
    def device_bytes(self):
        """Device bytes the plan holds: metadata and workspace."""
        return int(self._buffer.numel())

    def _check(self, q, k, v, out):
        index, dtype = self._index, self.dtype
        if q.shape != self._q_shape or k.shape != self._k_shape or v.shape != self._k_shape:
            raise ValueError("input shape does not match plan")
        if q.dtype != dtype or k.dtype != dtype or v.dtype != dtype:
            raise TypeError("q/k/v must have the plan's dtype")
        for tensor in (q, k, v):
            if tensor.get_device() != index or not tensor.is_contiguous():
                raise ValueError("inputs must be contiguous on the plan device")
            if tensor.requires_grad:
                raise ValueError("inference only: detach tensors requiring gradients")
        if out is None:
            return self._out
        if out.shape != self._q_shape or out.dtype != dtype or out.get_device() != index or not out.is_contiguous():
            raise ValueError("out must be a contiguous [B,Hq,D] tensor of the plan's dtype on the plan device")
        return out

    def run(self, q, k, v, out=None):
        """Decode one step; returns the plan's borrowed output, or writes into ``out`` and returns it."""
        out = self._check(q, k, v, out)
        status = self._lib.pd_prefix_decode(self._handle, q.data_ptr(), k.data_ptr(), v.data_ptr(), self._code,
                                            out.data_ptr(), _native.stream_of(self._index))
        if status:
            _native.check(status, "decode")
        return out

    def run_dynamic(self, q, k, v, table, lengths, out=None):
        """Decode with live metadata in device memory (plans built with ``max_lengths``).

        As ``DecodePlan.run_dynamic``: the live table and lengths count.  A
        sequence whose live table no longer starts with the plan's shared
        pages, or whose live length ends inside them (0: not in use), is
        computed on its own there: right, but slow, so build a new plan when
        prefixes change.
        """
        if self.max_lengths is None:
            raise ValueError("run_dynamic needs a plan built with max_lengths")
        out = self._check(q, k, v, out)
        index, batch = self._index, self.layout.batch
        table_at = _int32(table, (batch, self._width), "table", index)
        lengths_at = _int32(lengths, (batch,), "lengths", index)
        status = self._lib.pd_prefix_decode_dynamic(
            self._handle, q.data_ptr(), k.data_ptr(), v.data_ptr(), self._code, table_at, lengths_at, out.data_ptr(),
            _native.stream_of(index))
        if status:
            _native.check(status, "decode")
        return out

    def read_errors(self):
        """Return and clear the device error word (synchronises the current stream)."""
        import torch
        word = ctypes.c_uint32(0)
        _native.check(self._lib.pd_prefix_plan_read_errors(
            self._handle, ctypes.byref(word), torch.cuda.current_stream(self.device).cuda_stream))
        return int(word.value)
