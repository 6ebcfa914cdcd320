"""Query and key heads on their way to the decode, and the append into the paged cache.

``HeadRotation`` norms each query and key head (RMS, optional) and rotates it
by its position in one pass; ``CacheAppend`` does the same while it writes a
step's (or a prompt's) keys and values into the paged cache that ``DecodePlan``
reads, through the live page table and lengths that ``run_dynamic`` takes.
Inference only.  Neither call allocates when its outputs are given, nor
synchronises, so both can be captured in a CUDA graph.
"""
from __future__ import annotations

import ctypes

from . import _native
from .layout import Layout

__all__ = ["CacheAppend", "HeadRotation", "rotation_table"]


def rotation_table(max_positions, rotary_dim, *, base=10000.0, device="cuda"):
    """cos | sin of every position, FP32 [max_positions, rotary_dim]: pair i turns by
    position * base^(-2i / rotary_dim).  Angles are formed in FP64, so that far positions
    keep FP32 accuracy."""
    import torch
    if rotary_dim < 2 or rotary_dim % 2 or max_positions < 1:
        raise ValueError("rotary_dim must be even and positive, max_positions positive")
    freq = float(base) ** (-torch.arange(0, rotary_dim, 2, device=device, dtype=torch.float64) / rotary_dim)
    angle = torch.arange(max_positions, device=device, dtype=torch.float64)[:, None] * freq
    return torch.cat((angle.cos(), angle.sin()), 1).float()


def _dtype_code(dtype, what):
    import torch
    if dtype == torch.float16:
        return _native.PD_FLOAT16
    if dtype == torch.float32:
        return _native.PD_FLOAT32
    raise TypeError(f"{what} must be float16 or float32")


def _cuda_device(device):
    import torch
    device = torch.device(device)
    if device.type != "cuda":
        raise ValueError("a CUDA device is required")
    return torch.device("cuda", torch.cuda.current_device()) if device.index is None else device


def _refuse_rows(x, name, shape, dtype, index):
    """Raise for the first thing that is wrong with heads x."""
    if tuple(x.shape) != shape:
        raise ValueError(f"{name} must have shape {list(shape)}")
    if x.dtype != dtype:
        raise TypeError("q/k/v, their outputs and the caches must share float16 or float32 dtype")
    if x.get_device() != index or x.stride(2) != 1:
        raise ValueError(f"{name} must be on the device, its last dim contiguous")
    raise ValueError("inference only: detach tensors requiring gradients")


def _heads(x, out, name, shape, dtype, index):
    """Check x (and out) [tokens, heads, head_dim]; their pd_heads as bytes, each call's own (threads
    may share the object; packing takes a fifth of the time of a ctypes structure)."""
    strides = x.stride()
    if x.shape != shape or x.dtype != dtype or x.get_device() != index or strides[2] != 1 or x.requires_grad:
        _refuse_rows(x, name, shape, dtype, index)
    if out is None:
        return _native.pack_heads(x.data_ptr(), strides[0], strides[1], 0, 0, 0, shape[1])
    into = strides
    if out is not x:
        into = out.stride()
        if out.shape != shape or out.dtype != dtype or out.get_device() != index or into[2] != 1 or out.requires_grad:
            _refuse_rows(out, f"{name}_out", shape, dtype, index)
    return _native.pack_heads(x.data_ptr(), strides[0], strides[1], out.data_ptr(), into[0], into[1], shape[1])


def _int32(t, shape, name, index):
    import torch
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.shape != shape or \
            t.get_device() != index or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 CUDA tensor of shape {list(shape)} on the device")
    return t.data_ptr()


class HeadRotation:
    """RMS norm and position rotation of query and key heads.

    ``table`` is FP32 [max_positions, rotary_dim], cos then sin of each
    position's rotary_dim / 2 angles (``rotation_table`` makes the usual one);
    rotary_dim is a multiple of 16 up to head_dim, elements past it are not
    rotated, and None rotates nothing.  Pairs are (i, i + rotary_dim / 2), or
    with ``interleaved`` (2i, 2i + 1).  ``q_weight`` / ``k_weight`` [head_dim]
    norm the queries / keys before the rotation (None: no norm); they are kept
    in FP32.  Everything is computed in FP32 and rounded once.  Threads and streams
    may share an object: a call keeps nothing on it but the error word's flags.
    """

    def __init__(self, head_dim, table=None, *, interleaved=False, q_weight=None, k_weight=None, eps=1e-6,
                 device="cuda"):
        import torch
        if head_dim not in (64, 128):
            raise ValueError("head_dim must be 64 or 128")
        if not (0 <= eps < float("inf")):
            raise ValueError("eps must be finite and not negative")
        self.device = _cuda_device(device)
        self.head_dim, self.interleaved, self.eps = head_dim, bool(interleaved), float(eps)
        self.rotary_dim = self.max_positions = 0
        if table is not None:
            if table.ndim != 2 or table.shape[0] < 1 or table.shape[1] % 16 or not 16 <= table.shape[1] <= head_dim:
                raise ValueError("table must have shape [positions, rotary_dim], rotary_dim a multiple of 16 up to "
                                 "head_dim")
            if table.dtype != torch.float32:
                raise TypeError("the rotation table must be float32")
            if table.device != self.device or not table.is_contiguous() or table.data_ptr() % 16:
                raise ValueError("the rotation table must be contiguous and 16-byte aligned on the device")
            self.max_positions, self.rotary_dim = table.shape
        weights = []
        for w in (q_weight, k_weight):
            if w is not None:
                if tuple(w.shape) != (head_dim,):
                    raise ValueError("norm weights must have shape [head_dim]")
                w = w.detach().to(device=self.device, dtype=torch.float32, copy=True).contiguous()
            weights.append(w)
        self.table, (self.q_weight, self.k_weight) = table, weights
        self._lib = _native.load()
        self._error = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._error_at, self._index = self._error.data_ptr(), self.device.index
        self._spec = _native.Rotation(head_dim, self.rotary_dim, int(self.interleaved), self.eps, self.max_positions,
                                      *(None if t is None else t.data_ptr() for t in (table, *weights)))
        self._spec_at = ctypes.addressof(self._spec)
        torch.cuda.current_stream(self.device).synchronize()    # a call may come on any stream

    def run(self, q, k, positions, *, q_out=None, k_out=None):
        """Returns (q_out, k_out): q [N, Hq, D] and k [N, Hkv, D] normed and rotated.

        ``positions`` is int32 [N] on the device.  q and k may have any token
        and head stride (parts of a packed projection); either may be None.
        Outputs default to new tensors; an output may be its input (in place).
        A position outside the table gives zero rows and flags
        PD_DEVERR_POSITION (``read_errors``).
        """
        import torch
        first = q if q is not None else k
        if first is None:
            raise ValueError("q or k is needed")
        if first.ndim != 3:
            raise ValueError("heads must have shape [tokens, heads, head_dim]")
        dtype, index, tokens = first.dtype, self._index, first.shape[0]
        code = _dtype_code(dtype, "q/k")
        outs, descriptions = [], []
        for name, x, out in (("q", q, q_out), ("k", k, k_out)):
            rows = None
            if x is None:
                if out is not None:
                    raise ValueError(f"{name}_out without {name}")
            else:
                if x.ndim != 3:
                    raise ValueError("heads must have shape [tokens, heads, head_dim]")
                if out is None:
                    out = torch.empty(x.shape, dtype=dtype, device=self.device)
                rows = _heads(x, out, name, (tokens, x.shape[1], self.head_dim), dtype, index)
            outs.append(out)
            descriptions.append(rows)
        status = self._lib.pd_rotate_heads(
            self._spec_at, *descriptions, tokens, _int32(positions, (tokens,), "positions", index), code,
            self._error_at, index, _native.stream_of(index))
        if status:
            _native.check(status, "rotate")
        return tuple(outs)

    def read_errors(self):
        """Return and clear the device error word (synchronises the current stream)."""
        word = int(self._error.item())
        if word:
            self._error.zero_()
        return word


class CacheAppend:
    """Appends new tokens' keys and values to a paged cache.

    ``rotation`` (a ``HeadRotation``) norms and rotates keys, and queries given
    beside them, at their position in the sequence; None copies keys as they are.
    Shared by threads and streams as a ``HeadRotation`` is.
    """

    def __init__(self, layout: Layout, rotation=None, *, device="cuda"):
        import torch
        if layout.head_dim not in (64, 128):
            raise ValueError("head_dim must be 64 or 128")
        if layout.page_size not in (16, 32):
            raise ValueError("page_size must be 16 or 32")
        if layout.batch > 65535 or layout.query_heads > 65535:
            raise ValueError("batch/head count exceeds CUDA grid limits")
        self.device = _cuda_device(device)
        if rotation is not None and (rotation.head_dim != layout.head_dim or rotation.device != self.device):
            raise ValueError("rotation must have the layout's head_dim and be on the same device")
        self.layout, self.rotation = layout, rotation
        self._lib = _native.load()
        self._error = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._error_at, self._index = self._error.data_ptr(), self.device.index
        self._layout = _native.Layout(layout.batch, layout.query_heads, layout.kv_heads, layout.head_dim,
                                      layout.page_size, layout.physical_pages)
        self._cache_shape = (layout.physical_pages, layout.page_size, layout.kv_heads, layout.head_dim)
        self._layout_at = ctypes.addressof(self._layout)
        self._spec_at = None if rotation is None else rotation._spec_at
        torch.cuda.current_stream(self.device).synchronize()

    def run(self, k, v, k_cache, v_cache, table, lengths, *, q=None, indptr=None, q_out=None):
        """Write k, v [N, Hkv, D] into the caches; returns q's output (None without q).

        ``lengths`` int32 [B] already count the new tokens and ``table`` int32
        [B, W] already names their pages: both are what ``run_dynamic`` takes
        next.  With ``indptr`` int32 [B + 1] tokens indptr[b] .. indptr[b+1] - 1
        are the last ones of sequence b (indptr[0] is 0, tokens from indptr[B] on are padding);
        without it token b is the last one of sequence b, and a sequence of
        length 0 is not in use.  q [N, Hq, D] is normed and rotated into
        ``q_out`` (default: a new tensor; q itself: in place).  Padding and
        skipped tokens write no cache row and leave zero query rows; skipped
        tokens flag PD_DEVERR_LENGTH, PD_DEVERR_POSITION or PD_DEVERR_BAD_PAGE
        (``read_errors``).  All device inputs are read when the kernel runs.
        """
        import torch
        layout, index = self.layout, self._index
        if k.ndim != 3:
            raise ValueError("heads must have shape [tokens, heads, head_dim]")
        dtype, tokens, dim = k.dtype, k.shape[0], layout.head_dim
        code = _dtype_code(dtype, "k/v")
        q_rows = None
        if q is not None:
            if q_out is None:
                q_out = torch.empty((tokens, layout.query_heads, dim), dtype=dtype, device=self.device)
            q_rows = _heads(q, q_out, "q", (tokens, layout.query_heads, dim), dtype, index)
        elif q_out is not None:
            raise ValueError("q_out without q")
        shape = (tokens, layout.kv_heads, dim)
        k_rows, v_rows = _heads(k, None, "k", shape, dtype, index), _heads(v, None, "v", shape, dtype, index)
        for cache in (k_cache, v_cache):
            if cache.shape != self._cache_shape or cache.dtype != dtype or cache.get_device() != index or \
                    not cache.is_contiguous() or cache.requires_grad:
                self._refuse_cache(cache, dtype, index)
        if indptr is None:
            if tokens != layout.batch:
                raise ValueError("without indptr there is one token per sequence")
            indptr_at = None
        else:
            indptr_at = _int32(indptr, (layout.batch + 1,), "indptr", index)
        if not isinstance(table, torch.Tensor) or table.ndim != 2 or table.shape[1] < 1:
            raise ValueError("table must be a contiguous int32 CUDA tensor of shape [batch, width] on the device")
        width = table.shape[1]
        status = self._lib.pd_cache_append(
            self._layout_at, self._spec_at, q_rows, k_rows, v_rows, tokens, k_cache.data_ptr(),
            v_cache.data_ptr(), code, _int32(table, (layout.batch, width), "table", index), width,
            _int32(lengths, (layout.batch,), "lengths", index), indptr_at, self._error_at, index,
            _native.stream_of(index))
        if status:
            _native.check(status, "append")
        return q_out

    def _refuse_cache(self, cache, dtype, index):
        if tuple(cache.shape) != self._cache_shape:
            raise ValueError("cache shape does not match the layout")
        if cache.dtype != dtype:
            raise TypeError("q/k/v, their outputs and the caches must share float16 or float32 dtype")
        if cache.get_device() != index or not cache.is_contiguous():
            raise ValueError("caches must be contiguous on the device")
        raise ValueError("inference only: detach tensors requiring gradients")

    read_errors = HeadRotation.read_errors
