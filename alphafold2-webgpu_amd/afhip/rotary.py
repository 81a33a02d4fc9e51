"""The norm of each query and key head, the rotation by its position and the
write into a cache, in one pass; and the way back.

What comes before WindowAttention (window.py) in a layer over one sequence's
tokens, over afhip_rotary_*. No counterpart in the reference, whose attention
has neither positions nor a cache.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np

from . import _lib
from .device import device, open_device
from .heads import (FORMS, address, check_device, check_heads, check_ints, current_device, current_stream, form,
                    packed_like, strides)

_DT = {"f32": _lib.F32, "f16": _lib.F16}
_LAYOUTS = {"half": _lib.ROTARY_HALF, "interleaved": _lib.ROTARY_INTERLEAVED}
_NORMS = {None: _lib.HEAD_NORM_NONE, "rms": _lib.HEAD_NORM_RMS, "layer": _lib.HEAD_NORM_LAYER}


def frequencies(rotary_dim: int, *, base: float = 10000.0, scaling: str | None = None, factor: float = 1.0,
                trained_length: int = 2048, fast: float = 32.0, slow: float = 1.0) -> np.ndarray:
    """The angle of one position for each of rotary_dim / 2 pairs, f64:
    base^(-2j / rotary_dim), changed for contexts `factor` times as long:

      "linear"  all of them over `factor` (positions interpolated)
      "ntk"     a larger base, so that the slowest pair turns `factor` times slower and the fastest as before
      "yarn"    over `factor` for pairs that turn fewer than `slow` times within trained_length, unchanged
                from `fast` turns on, in between by the logarithm of the turns (rotation_scale beside it:
                yarn_scale(factor))
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise _lib.RangeError("rotary_dim must be even and positive")
    if not (base > 0 and factor > 0):
        raise _lib.RangeError("base and factor must be positive")
    if scaling == "ntk" and rotary_dim > 2:
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    f = base ** -(np.arange(0, rotary_dim, 2, dtype=np.float64) / rotary_dim)
    if scaling in (None, "ntk"):
        return f
    if scaling == "linear":
        return f / factor
    if scaling != "yarn":
        raise _lib.RangeError(f"unknown scaling {scaling!r}")
    if not fast > slow > 0:
        raise _lib.RangeError("fast must be larger than slow, and slow positive")
    turns = trained_length * f / (2 * math.pi)
    keep = np.clip((np.log(turns) - math.log(slow)) / (math.log(fast) - math.log(slow)), 0, 1)
    return f * keep + f / factor * (1 - keep)


def yarn_scale(factor: float) -> float:
    """rotation_scale for frequencies(scaling="yarn"): the square root of the scores' factor."""
    return 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0


class HeadRotary:
    """Norms and turns q [batch][tokens][query_heads][head_dim] and k [..][key_heads][..], views of one
    projection for instance (channels contiguous, the other strides multiples of 16 bytes). The first
    rotary_dim channels turn, by `frequencies` (f64 [rotary_dim / 2]; from `base` where none are given)."""

    def __init__(self, query_heads: int, key_heads: int, head_dim: int, *, rotary_dim: int | None = None,
                 layout: str = "half", norm: str | None = None, dtype: str = "f32", base: float = 10000.0,
                 frequencies=None, rotation_scale: float = 1.0, epsilon: float = 1e-5):
        import torch

        open_device()
        if dtype not in _DT:
            raise _lib.RangeError(f"unknown dtype {dtype!r}")
        if layout not in _LAYOUTS:
            raise _lib.RangeError(f"unknown rotary layout {layout!r}")
        if norm not in _NORMS:
            raise _lib.RangeError(f"unknown head norm {norm!r}")
        self.query_heads, self.key_heads, self.head_dim = query_heads, key_heads, head_dim
        self.rotary_dim = head_dim if rotary_dim is None else rotary_dim
        self.layout, self.norm, self.dtype = layout, norm, dtype
        self.rotation_scale, self.epsilon = rotation_scale, epsilon
        probe = self._desc(1, 1, 0)  # refuses what no call can have
        _lib.call("afhip_rotary_backward_workspace_size", ctypes.byref(probe), ctypes.byref(ctypes.c_size_t()))
        if frequencies is None:
            frequencies = globals()["frequencies"](self.rotary_dim, base=base) if self.rotary_dim else np.zeros(0)
        f = torch.as_tensor(frequencies, dtype=torch.float64).reshape(-1)
        if f.numel() != self.rotary_dim // 2:
            raise _lib.RangeError(f"frequencies has {f.numel()} values; expected {self.rotary_dim // 2}")
        self.frequencies = f.to(device()).contiguous()
        self._torch_dtype = torch.float32 if dtype == "f32" else torch.float16
        self._torch_device = device()
        self._device = self._torch_device.index
        self._forms = {}
        self.query_scale = self.key_scale = self.query_offset = self.key_offset = None

    def prepare(self, query_scale=None, key_scale=None, query_offset=None, key_offset=None) -> None:
        """The norm's vectors, f32 [head_dim]: scales for "rms", scales and offsets for "layer". Device tensors
        are kept as they are (a training step that changes them in place needs no new call)."""
        import torch

        given = {"query_scale": query_scale, "key_scale": key_scale, "query_offset": query_offset,
                 "key_offset": key_offset}
        for name, value in given.items():
            wanted = self.norm is not None and (name.endswith("scale") or self.norm == "layer")
            if (value is not None) != wanted:
                raise _lib.RangeError(f"{name} is {'needed' if wanted else 'not taken'} with norm {self.norm!r}")
            if value is None:
                continue
            if not isinstance(value, torch.Tensor):
                value = torch.from_numpy(np.ascontiguousarray(value, np.float32))
            if not value.is_cuda:
                value = value.to(device())
            check_device(name, value, self._device)
            if value.dtype != torch.float32 or value.numel() != self.head_dim or not value.is_contiguous():
                raise _lib.RangeError(f"{name} must be contiguous f32 of {self.head_dim} values")
            given[name] = value
        self.query_scale, self.key_scale = given["query_scale"], given["key_scale"]
        self.query_offset, self.key_offset = given["query_offset"], given["key_offset"]

    def _desc(self, batch: int, tokens: int, capacity: int, **tensors) -> _lib.RotaryDesc:
        desc = _lib.RotaryDesc(batch, tokens, self.query_heads, self.key_heads, self.head_dim, self.rotary_dim,
                               _LAYOUTS[self.layout], _NORMS[self.norm], _DT[self.dtype], capacity, self.epsilon,
                               self.rotation_scale)
        for name, tensor in tensors.items():
            if tensor is not None:
                setattr(desc, name, strides(tensor))
        return desc

    def _ready(self) -> None:
        if self.norm is not None and self.query_scale is None:
            raise _lib.RangeError("prepare() has not been given the norm's vectors")

    def _checked(self, q, k, past, lengths, positions) -> tuple:
        if q.dim() != 4:
            raise _lib.RangeError(f"q has shape {tuple(q.shape)}; expected [batch, tokens, heads, channels]")
        batch, tokens = q.shape[:2]
        check_heads("q", q, self._torch_dtype, (None, None, self.query_heads, self.head_dim), self._device)
        check_heads("k", k, self._torch_dtype, (batch, tokens, self.key_heads, self.head_dim), self._device)
        check_ints("past", past, (batch,), self._device)
        check_ints("lengths", lengths, (batch,), self._device)
        check_ints("positions", positions, (batch, tokens), self._device)
        return batch, tokens

    def __call__(self, q, k, v=None, *, past=None, lengths=None, positions=None, q_out=None, k_out=None,
                 k_cache=None, v_cache=None):
        """(q, k) normed and turned, or (q, k_cache, v_cache) where caches [batch][capacity][key_heads][head_dim]
        are given: token i of a sequence goes to row past + i (not written where the cache has no such row).

        past, lengths: int32 [batch], what a sequence has behind it (0) and how many of these tokens it has
        (all); positions: int32 [batch][tokens] (past + i). Tokens past the length give zeros, and write nothing
        into a cache. q_out may be q, and k_out k."""
        import torch

        if current_device() != self._device:
            with torch.cuda.device(self._device):
                return self(q, k, v, past=past, lengths=lengths, positions=positions, q_out=q_out, k_out=k_out,
                            k_cache=k_cache, v_cache=v_cache)
        self._ready()
        key = (form(q), form(k), form(v), form(past), form(lengths), form(positions), form(q_out), form(k_out),
               form(k_cache), form(v_cache))
        desc = self._forms.get(key)
        if desc is None:
            desc = self._form(q, k, v, past, lengths, positions, q_out, k_out, k_cache, v_cache)
            if len(self._forms) >= FORMS:
                self._forms.clear()
            self._forms[key] = desc
        if q_out is None:
            q_out = packed_like(q)
        if k_cache is None and k_out is None:
            k_out = packed_like(k)
        _lib.call("afhip_rotary_run", desc, q.data_ptr(), k.data_ptr(), address(v), address(past), address(lengths),
                  address(positions), self.frequencies.data_ptr(), address(self.query_scale),
                  address(self.query_offset), address(self.key_scale), address(self.key_offset), q_out.data_ptr(),
                  (k_out if k_cache is None else k_cache).data_ptr(), address(v_cache),
                  current_stream(self._device))
        return (q_out, k_out) if k_cache is None else (q_out, k_cache, v_cache)

    def _form(self, q, k, v, past, lengths, positions, q_out, k_out, k_cache, v_cache):
        """Checks one form of a call and describes it."""
        batch, tokens = self._checked(q, k, past, lengths, positions)
        if q_out is not None:
            check_heads("q_out", q_out, self._torch_dtype, q.shape, self._device, True)
        capacity = 0
        if k_cache is None:
            if v is not None or v_cache is not None:
                raise _lib.RangeError("v is taken with k_cache and v_cache")
            if k_out is not None:
                check_heads("k_out", k_out, self._torch_dtype, k.shape, self._device, True)
        else:
            if k_out is not None:
                raise _lib.RangeError("k_out is not taken with k_cache")
            if (v is None) != (v_cache is None):
                raise _lib.RangeError("v and v_cache go together")
            check_heads("k_cache", k_cache, self._torch_dtype, (batch, None, self.key_heads, self.head_dim),
                        self._device, True)
            capacity = k_cache.shape[1]
            if capacity < 1:
                raise _lib.RangeError("k_cache holds no tokens")
            if v is not None:
                check_heads("v", v, self._torch_dtype, k.shape, self._device)
                check_heads("v_cache", v_cache, self._torch_dtype, k_cache.shape, self._device, True)
        return ctypes.pointer(self._desc(batch, tokens, capacity, q=q, k=k, v=v, q_out=q_out,
                                         k_out=k_out if k_cache is None else k_cache, v_out=v_cache))

    def backward(self, q, k, dq_out, dk_out, *, past=None, lengths=None, positions=None) -> dict:
        """The gradients, from those of a call without a cache: "dq" and "dk", and with a norm "dquery_scale" and
        "dkey_scale", with "layer" "dquery_offset" and "dkey_offset" too (f32 [head_dim])."""
        import torch

        if current_device() != self._device:
            with torch.cuda.device(self._device):
                return self.backward(q, k, dq_out, dk_out, past=past, lengths=lengths, positions=positions)
        self._ready()
        key = ("backward", form(q), form(k), form(dq_out), form(dk_out), form(past), form(lengths), form(positions))
        found = self._forms.get(key)
        if found is None:
            batch, tokens = self._checked(q, k, past, lengths, positions)
            check_heads("dq_out", dq_out, self._torch_dtype, q.shape, self._device)
            check_heads("dk_out", dk_out, self._torch_dtype, k.shape, self._device)
            desc = self._desc(batch, tokens, 0, q=q, k=k, q_out=dq_out, k_out=dk_out)
            size = ctypes.c_size_t()
            _lib.call("afhip_rotary_backward_workspace_size", ctypes.byref(desc), ctypes.byref(size))
            if len(self._forms) >= FORMS:
                self._forms.clear()
            found = self._forms[key] = (ctypes.pointer(desc), size.value)
        desc, bytes_ = found
        out = {"dq": packed_like(q), "dk": packed_like(k)}
        if self.norm is not None:
            out["dquery_scale"] = torch.empty_like(self.query_scale)
            out["dkey_scale"] = torch.empty_like(self.key_scale)
            if self.norm == "layer":
                out["dquery_offset"] = torch.empty_like(self.query_scale)
                out["dkey_offset"] = torch.empty_like(self.key_scale)
        # From the caching allocator at each call: calls on several streams, and captured ones, share nothing.
        workspace = torch.empty(max(bytes_, 1), dtype=torch.uint8, device=self._torch_device)
        _lib.call("afhip_rotary_backward", desc, q.data_ptr(), k.data_ptr(), address(past), address(lengths),
                  address(positions), self.frequencies.data_ptr(), address(self.query_scale),
                  address(self.key_scale), dq_out.data_ptr(), dk_out.data_ptr(), out["dq"].data_ptr(),
                  out["dk"].data_ptr(), address(out.get("dquery_scale")), address(out.get("dquery_offset")),
                  address(out.get("dkey_scale")), address(out.get("dkey_offset")), workspace.data_ptr(), bytes_,
                  current_stream(self._device))
        return out
