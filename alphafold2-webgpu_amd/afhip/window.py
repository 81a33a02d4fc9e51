"""Attention over a window of keys and the first few ("sinks"): prompts,
pieces of them and single tokens against a cache, and the way back.

Over afhip_window_*, for the layers over one sequence's tokens whose queries
and keys HeadRotary (rotary.py) turns. Attention (attention.py) is the
Evoformer's, with its projections, gate and pair bias; this is the bare
product, with grouped heads, lengths and gradients. No counterpart in the
reference.
"""
from __future__ import annotations

import ctypes
import math

from . import _lib
from .device import device, open_device
from .heads import (FORMS, address, check_device, check_heads, check_ints, current_device, current_stream, form,
                    packed_like, strides)

_DT = {"f32": _lib.F32, "f16": _lib.F16}


class WindowAttention:
    """Queries [batch][queries][query_heads][head_dim] against keys and values [batch][keys][key_heads][head_dim]
    (views with contiguous channels, the other strides multiples of 16 bytes; a cache, for instance).

    The queries are the last of their sequence: query i has position p = key_length - query_length + i and sees key
    j where j < key_length, j <= p + right, and j >= p - left or j < sinks; None has no end on that side. Query head
    h reads key head h // (query_heads / key_heads). scale is 1 / sqrt(head_dim) where none is given."""

    def __init__(self, query_heads: int, key_heads: int, head_dim: int, *, left: int | None = None,
                 right: int | None = 0, sinks: int = 0, dtype: str = "f32", scale: float | None = None):
        import torch

        open_device()
        if dtype not in _DT:
            raise _lib.RangeError(f"unknown dtype {dtype!r}")
        self.query_heads, self.key_heads, self.head_dim = query_heads, key_heads, head_dim
        self.left, self.right, self.sinks = -1 if left is None else left, -1 if right is None else right, sinks
        if head_dim <= 0:
            raise _lib.RangeError("attention dimensions must be positive")
        self.dtype, self.scale = dtype, 1.0 / math.sqrt(head_dim) if scale is None else scale
        probe = self._desc(1, 1, 1)  # refuses what no call can have
        _lib.call("afhip_window_workspace_size", ctypes.byref(probe), ctypes.byref(ctypes.c_size_t()))
        self._torch_dtype = torch.float32 if dtype == "f32" else torch.float16
        self._torch_device = device()
        self._device = self._torch_device.index
        self._forms = {}

    def _desc(self, batch: int, queries: int, keys: int, **tensors) -> _lib.WindowDesc:
        desc = _lib.WindowDesc(batch, queries, keys, self.query_heads, self.key_heads, self.head_dim, self.left,
                               self.right, self.sinks, _DT[self.dtype], self.scale)
        for name, tensor in tensors.items():
            if tensor is not None:
                setattr(desc, name, strides(tensor))
        return desc

    def _checked(self, q, k, v, query_lengths, key_lengths) -> tuple:
        check_heads("q", q, self._torch_dtype, (None, None, self.query_heads, self.head_dim), self._device)
        batch, queries = q.shape[:2]
        check_heads("k", k, self._torch_dtype, (batch, None, self.key_heads, self.head_dim), self._device)
        check_heads("v", v, self._torch_dtype, k.shape, self._device)
        check_ints("query_lengths", query_lengths, (batch,), self._device)
        check_ints("key_lengths", key_lengths, (batch,), self._device)
        return batch, queries, k.shape[1]

    def _remember(self, key, value):
        if len(self._forms) >= FORMS:
            self._forms.clear()
        self._forms[key] = value
        return value

    def __call__(self, q, k, v, *, query_lengths=None, key_lengths=None, out=None, return_lse: bool = False):
        """out [batch][queries][query_heads][head_dim], and with return_lse each row's log-sum-exp of its scaled
        scores, f32 [batch][query_heads][queries] (what backward needs). query_lengths, key_lengths: int32 [batch]
        (all). Rows that see nothing, or lie past their length, give zeros and -inf; keys past the length are not
        read."""
        import torch

        if current_device() != self._device:
            with torch.cuda.device(self._device):
                return self(q, k, v, query_lengths=query_lengths, key_lengths=key_lengths, out=out,
                            return_lse=return_lse)
        key = (form(q), form(k), form(v), form(query_lengths), form(key_lengths), form(out))
        found = self._forms.get(key)
        if found is None:
            batch, queries, keys = self._checked(q, k, v, query_lengths, key_lengths)
            if out is not None:
                check_heads("out", out, self._torch_dtype, q.shape, self._device, True)
            desc = self._desc(batch, queries, keys, q=q, k=k, v=v, out=out)
            size = ctypes.c_size_t()
            _lib.call("afhip_window_workspace_size", ctypes.byref(desc), ctypes.byref(size))
            found = self._remember(key, (ctypes.pointer(desc), size.value, (batch, self.query_heads, queries)))
        desc, bytes_, rows = found
        if out is None:
            out = packed_like(q)
        lse = torch.empty(rows, dtype=torch.float32, device=self._torch_device) if return_lse else None
        # From the caching allocator at each call: calls on several streams, and captured ones, share nothing.
        workspace = torch.empty(bytes_, dtype=torch.uint8, device=self._torch_device) if bytes_ else None
        _lib.call("afhip_window_run", desc, q.data_ptr(), k.data_ptr(), v.data_ptr(), address(query_lengths),
                  address(key_lengths), out.data_ptr(), address(lse), address(workspace), bytes_,
                  current_stream(self._device))
        return (out, lse) if return_lse else out

    def backward(self, q, k, v, out, lse, dout, *, query_lengths=None, key_lengths=None) -> tuple:
        """(dq, dk, dv) from a call's inputs, its out and lse, and the gradient of out; those of k and v summed over
        the query heads that read them. Zeros past the lengths. The same bits at every call."""
        import torch

        if current_device() != self._device:
            with torch.cuda.device(self._device):
                return self.backward(q, k, v, out, lse, dout, query_lengths=query_lengths, key_lengths=key_lengths)
        key = ("backward", form(q), form(k), form(v), form(out), form(lse), form(dout), form(query_lengths),
               form(key_lengths))
        found = self._forms.get(key)
        if found is None:
            batch, queries, keys = self._checked(q, k, v, query_lengths, key_lengths)
            check_heads("out", out, self._torch_dtype, q.shape, self._device)
            check_heads("dout", dout, self._torch_dtype, q.shape, self._device)
            check_device("lse", lse, self._device)
            if (lse.dtype != torch.float32 or tuple(lse.shape) != (batch, self.query_heads, queries)
                    or not lse.is_contiguous()):
                raise _lib.RangeError(f"lse must be contiguous f32 of shape {(batch, self.query_heads, queries)}")
            desc = self._desc(batch, queries, keys, q=q, k=k, v=v, out=out)
            size = ctypes.c_size_t()
            _lib.call("afhip_window_backward_workspace_size", ctypes.byref(desc), ctypes.byref(size))
            found = self._remember(key, (ctypes.pointer(desc), ctypes.pointer(strides(dout)), size.value))
        desc, dout_strides, bytes_ = found
        dq, dk, dv = packed_like(q), packed_like(k), packed_like(v)
        workspace = torch.empty(max(bytes_, 1), dtype=torch.uint8, device=self._torch_device)
        _lib.call("afhip_window_backward", desc, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                  lse.data_ptr(), dout.data_ptr(), dout_strides, address(query_lengths), address(key_lengths),
                  dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), workspace.data_ptr(), bytes_,
                  current_stream(self._device))
        return dq, dk, dv
