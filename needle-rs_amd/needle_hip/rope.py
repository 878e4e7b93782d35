"""Rotary positions over the C ABI (nh_rope_* in include/needle_hip.h).  No
counterpart in the reference as an operator."""
from __future__ import annotations

import ctypes as C

import numpy as np
import torch

import needle_hip as nh

from .kvcache import _TYPES, _on

_LAYOUTS = {"half": 0, "interleaved": 1}  # NH_ROPE_HALF, NH_ROPE_INTERLEAVED
# NH_ROPE_LINEAR .., and the turns (low, high) where none are given
_SCALINGS = {"linear": (1, None), "base": (2, None), "parts": (3, (1.0, 32.0)), "bands": (4, (1.0, 4.0))}


def _row_stride(t: torch.Tensor, rows: int, dim, index: int, what: str) -> int:
    """The row stride of [rows][heads][dim]; a row lies in one piece."""
    if len(t.shape) != 3 or t.shape[0] != rows or (dim is not None and t.shape[2] != dim):
        raise ValueError(f"{what} is [{rows}][heads][{'dim' if dim is None else dim}], not {list(t.shape)}")
    if t.get_device() != index or t.dtype not in _TYPES:
        raise ValueError(f"{what} is f32, f16 or bf16 on the plan's device")
    _, heads, dim = t.shape
    ld, of_head, of_dim = t.stride()
    if (dim > 1 and of_dim != 1) or (heads > 1 and of_head != dim):
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
        if positions.dtype != torch.int32 or positions.shape != (rows,) or not positions.is_contiguous() or \
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
        rows, with k the pair."""
        rows = q.shape[0]
        pos = self._positions(positions, rows)
        given = (q,) if k is None else (q, k)
        outs = (None,) * len(given) if out is None else (out,) if k is None else tuple(out)
        if len(outs) != len(given):
            raise ValueError("one out for each of q and k")
        args, made = [], []
        dim = q.shape[2] if len(q.shape) == 3 else None
        with _on(stream):
            for x, y, what in zip(given, outs, ("q", "k")):
                ld = _row_stride(x, rows, dim, self._index, what)
                if x.dtype != q.dtype:
                    raise ValueError("q and k differ in type")
                if y is None:
                    y = torch.empty(x.shape, dtype=x.dtype, device=self.device)
                elif y.dtype != x.dtype or y.shape != x.shape:
                    raise ValueError(f"{what} and its out differ in type or shape")
                made.append(y)
                args += (x.data_ptr(), ld, x.shape[1], y.data_ptr(), _row_stride(y, rows, dim, self._index, "out"))
        if k is None:
            args += (None, 0, 0, None, 0)
        nh._check(nh._lib.nh_rope_apply(self.h, pos, rows, dim, *args, _TYPES[q.dtype], int(bool(transposed)),
                                        nh._stream(stream)))
        return made[0] if k is None else tuple(made)

    def __del__(self):
        if getattr(self, "h", None) and nh is not None and nh._lib is not None:
            nh._lib.nh_rope_free(self.h)
        self.h = None
