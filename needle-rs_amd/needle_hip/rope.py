"""Rotary positions over the C ABI (nh_rope_* in include/needle_hip.h).  No
counterpart in the reference as an operator."""
from __future__ import annotations

import ctypes as C

import numpy as np
import torch

import needle_hip as nh

from .kvcache import _TYPES, _like, _on

_LAYOUTS = {"half": 0, "interleaved": 1}  # NH_ROPE_HALF, NH_ROPE_INTERLEAVED
# NH_ROPE_LINEAR .., and the turns (low, high) where none are given
_SCALINGS = {"linear": (1, None), "base": (2, None), "parts": (3, (1.0, 32.0)), "bands": (4, (1.0, 4.0))}


def _row_stride(t: torch.Tensor, rows: int, dim: int, index: int, dtype, what: str) -> int:
    """The row stride of [rows][heads][dim]; a row lies in one piece."""
    shape = t.shape
    if len(shape) != 3 or shape[0] != rows or shape[2] != dim:
        raise ValueError(f"{what} is [{rows}][heads][{dim}], not {list(shape)}")
    if t.dtype is not dtype or t.get_device() != index:
        raise ValueError(f"{what} is of q's type, f32, f16 or bf16, on the plan's device")
    heads = shape[1]
    ld, of_head, of_dim = t.stride()
    if (of_dim != 1 and dim > 1) or (of_head != dim and heads > 1):
        raise ValueError(f"a row of {what} is not contiguous")
    return ld if rows > 1 else heads * dim


class Rope:
    """A plan of rotary positions (nh_rope): the first `dim` dims of a head turn
    in pairs, (i, i + dim / 2) in layout "half", neighbours in "interleaved".
    scaling, for contexts `factor` times longer than the model's own `original`
    length: ("linear", factor), ("base", factor), ("parts", factor, original[,
    low, high]) or ("bands", factor, original[, low, high]) (NH_ROPE_LINEAR ..
    in the header)."""

    def __init__(self, dim: int, theta: float = 10000.0, layout: str = "half", scaling=None):
        lib = nh.load_library()
        kind, rest = 0, (1.0, 1.0, 1.0, 2.0)
        if scaling is not None:
            name, *given = scaling
            if name not in _SCALINGS:
                raise ValueError(f"no such scaling: {name}")
            kind, turns = _SCALINGS[name]
            if len(given) not in ((1,) if turns is None else (2, 4)):
                raise ValueError(f"{name}: a factor" + ("" if turns is None else ", the original length and, if not the usual, two numbers of turns"))
            rest = (*given, 1.0, 1.0, 2.0) if turns is None else (*given, *turns) if len(given) == 2 else tuple(given)
        f, amplitude = np.zeros(max(int(dim) // 2, 1)), C.c_double()
        nh._check(lib.nh_rope_freqs(int(dim), float(theta), kind, *(float(x) for x in rest), nh._hptr(f), C.byref(amplitude)))
        self._make(f, amplitude.value, layout)

    @classmethod
    def from_freqs(cls, freqs, amplitude: float = 1.0, layout: str = "half") -> "Rope":
        """A plan of given frequencies, radians a position, one a pair."""
        self = cls.__new__(cls)
        self._make(np.ascontiguousarray(freqs, np.float64).reshape(-1).copy(), float(amplitude), layout)
        return self

    def _make(self, freqs, amplitude, layout):
        lib = nh.load_library()
        self.h = None
        if layout not in _LAYOUTS:
            raise ValueError(f"no such layout: {layout}")
        if torch.cuda.is_available():
            nh.init()
        h = C.c_void_p()
        nh._check(lib.nh_rope_new(nh._hptr(freqs), freqs.size, amplitude, _LAYOUTS[layout], C.byref(h)))
        self.h = h
        self.freqs, self.amplitude, self.layout, self.dim = freqs, amplitude, layout, 2 * freqs.size
        self.device = torch.device("cuda", torch.cuda.current_device())
        self._index = self.device.index

    def _positions(self, positions: torch.Tensor, rows: int):
        if positions.dtype is not torch.int32 or positions.shape != (rows,) or not positions.is_contiguous() or \
                positions.get_device() != self._index:
            raise ValueError(f"positions: contiguous int32 [{rows}] on {self.device}")
        return positions.data_ptr()

    def apply(self, positions: torch.Tensor, q: torch.Tensor, k: torch.Tensor | None = None, out=None,
              transposed: bool = False, stream=None):
        """q [rows][heads][dim] (and k [rows][kv_heads][dim], in the same launch)
        turned to the rows' positions (int32 [rows]).  Rows may be views of a
        wider matrix's columns.  out: a tensor, with k a pair of them (None:
        new ones); q itself and k itself turn in place.  transposed: gradients of
        the outputs to the inputs' (the same angles backwards).  Returns q's
        rows, with k the pair.  The call records no gradients: rows that would
        need them are refused (a torch.autograd.Function calls apply forwards and
        transposed backwards; detach() or torch.no_grad() otherwise)."""
        if len(q.shape) != 3:
            raise ValueError(f"q is [rows][heads][dim], not {list(q.shape)}")
        rows, heads, dim = q.shape
        dtype, index = q.dtype, self._index
        if dtype not in _TYPES:
            raise ValueError("q is f32, f16 or bf16")
        if (q.requires_grad or (k is not None and k.requires_grad)) and torch.is_grad_enabled():
            raise ValueError("apply records no gradients: detach q and k, or turn their gradients with transposed=True")
        pos = self._positions(positions, rows)
        ldq = _row_stride(q, rows, dim, index, dtype, "q")
        ldk = kv_heads = 0
        if k is not None:
            ldk = _row_stride(k, rows, dim, index, dtype, "k")
            kv_heads = k.shape[1]
        if out is None:
            with _on(stream):
                out = qo = _like(q)
                ldqo = heads * dim
                if k is not None:
                    ko = _like(k)
                    ldko, out = kv_heads * dim, (qo, ko)
        else:
            if k is None:
                qo = out
            else:
                qo, ko = out
                if ko.shape != k.shape:
                    raise ValueError("k and its out differ in shape")
                ldko = _row_stride(ko, rows, dim, index, dtype, "out")
            if qo.shape != q.shape:
                raise ValueError("q and its out differ in shape")
            ldqo = _row_stride(qo, rows, dim, index, dtype, "out")
        if k is None:
            args = (None, 0, 0, None, 0)
        else:
            args = (k.data_ptr(), ldk, kv_heads, ko.data_ptr(), ldko)
        nh._check(nh._lib.nh_rope_apply(self.h, pos, rows, dim, q.data_ptr(), ldq, heads, qo.data_ptr(), ldqo, *args, _TYPES[dtype],
                                        1 if transposed else 0, nh._stream(stream)))
        return out

    def __del__(self):
        if getattr(self, "h", None) and nh is not None and nh._lib is not None:
            nh._lib.nh_rope_free(self.h)
        self.h = None
