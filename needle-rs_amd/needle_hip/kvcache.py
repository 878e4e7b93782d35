"""What the paged key/value caches share over the C ABI (nh_kv4_* and nh_kv8_*
in include/needle_hip.h): sequences, batches, reading, attention.  No
counterpart in the reference."""
from __future__ import annotations

import array
import contextlib
import ctypes as C
import types

import torch

import needle_hip as nh

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}  # NH_F32, NH_F16, NH_BF16


def _ints(v):
    """(the numbers as C ints, their address, their count); the array keeps them alive."""
    try:
        a = array.array("i", v)
    except (OverflowError, TypeError) as e:
        raise ValueError(f"not a list of 32-bit numbers: {e}") from None
    at, n = a.buffer_info()
    return a, at, n


_here = contextlib.nullcontext()


def _on(stream):
    """Allocations of the call come from the memory of the stream that uses them."""
    return torch.cuda.stream(stream) if stream is not None else _here


def _like(t):
    """A new contiguous tensor like t."""
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def _ptr(t):
    return t.data_ptr() if t is not None else None


class PagedCache:
    """A paged cache of keys and values, shared by many sequences.  A step:
    `extend` names its sequences and their new rows; then, for every layer,
    `append` stores the rows' keys and values and `attend` attends with their
    queries.  For serving: no call records gradients.  The formats: KvCache4,
    KvCache8."""

    _CALLS = ("free", "bytes", "free_pages", "seq_new", "seq_len", "seq_free", "seq_truncate", "seq_fork", "seq_copy",
              "extend", "rows", "append", "read", "debug_kernel", "attend_ws_bytes", "attend")

    def _make(self, prefix: str, layers: int, kv_heads: int, qk_dim: int, v_dim: int, pages: int, page: int, args):
        """The handle of nh_<prefix>_new(*args), and its entry points."""
        lib = nh.load_library()
        self.h = None
        self._c = types.SimpleNamespace(**{f: getattr(lib, f"nh_{prefix}_{f}") for f in self._CALLS})
        if torch.cuda.is_available():
            nh.init()
        h = C.c_void_p()
        nh._check(getattr(lib, f"nh_{prefix}_new")(*args, C.byref(h)))
        self.h = h
        self.layers, self.kv_heads, self.qk_dim, self.v_dim = int(layers), int(kv_heads), int(qk_dim), int(v_dim)
        self.page, self.pages = int(page), int(pages)
        self.device = torch.device("cuda", torch.cuda.current_device())
        self._index = self.device.index
        self._like = {}
        self._batch(0)

    def _batch(self, rows: int):
        """Another batch, of so many rows."""
        self._rows = rows
        self._ws_bytes = {}  # of attend, by what it depends on beside the batch

    def _empty(self, shape, dtype):
        """torch.empty on the cache's device, a microsecond sooner: like a tensor that is there."""
        t = self._like.get(dtype)
        if t is None:
            t = self._like[dtype] = torch.empty(0, dtype=dtype, device=self.device)
        return t.new_empty(shape)

    # ---- sequences
    def new_seq(self) -> int:
        """An empty sequence's id."""
        return nh._check(self._c.seq_new(self.h))

    def length(self, seq: int) -> int:
        return nh._check(self._c.seq_len(self.h, int(seq)))

    def free(self, seq: int):
        """Gives back the pages that no branch shares."""
        nh._check(self._c.seq_free(self.h, int(seq)))
        self._batch(self.rows)  # (it may be over)

    def truncate(self, seq: int, length: int):
        """Forgets positions `length` and on."""
        nh._check(self._c.seq_truncate(self.h, int(seq), int(length)))
        self._batch(self.rows)

    def fork(self, seq: int, n: int = 1) -> list:
        """n branches that share the sequence's pages until they are written."""
        out = (C.c_int * max(int(n), 1))()
        nh._check(self._c.seq_fork(self.h, int(seq), int(n), C.addressof(out)))
        self._batch(self.rows)
        return out[:n]

    def copy(self, seq: int, stream=None) -> int:
        """A branch with pages of its own."""
        made = nh._check(self._c.seq_copy(self.h, int(seq), nh._stream(stream)))
        self._batch(self.rows)
        return made

    @property
    def free_pages(self) -> int:
        return nh._check(self._c.free_pages(self.h))

    def bytes(self) -> int:
        n = self._c.bytes(self.h)
        nh._check(-1 if n < 0 else 0)
        return n

    # ---- rows
    def extend(self, seqs, rows, stream=None):
        """rows[i] more positions for each sequence; they become the batch."""
        s, ps, n = _ints(seqs)
        r, pr, m = _ints(rows)
        if n != m:
            raise ValueError("one number of rows for each sequence")
        nh._check(self._c.extend(self.h, ps, pr, n, nh._stream(stream)))
        self._batch(sum(r))

    @property
    def rows(self) -> int:
        """The batch's rows."""
        return nh._check(self._c.rows(self.h))

    def _rows_of(self, t: torch.Tensor, heads: int, dim: int, what: str) -> int:
        """The row stride of [rows][heads][dim]; a row lies in one piece."""
        n = self._rows
        if t.shape != (n, heads, dim):
            raise ValueError(f"{what} is [{n}][{heads}][{dim}], not {list(t.shape)}")
        if t.get_device() != self._index or t.dtype not in _TYPES:
            raise ValueError(f"{what} is f32, f16 or bf16 on {self.device}")
        ld, of_head, of_dim = t.stride()
        if (dim > 1 and of_dim != 1) or (heads > 1 and of_head != dim):
            raise ValueError(f"a row of {what} is not contiguous")
        return ld if n > 1 else heads * dim

    def read(self, layer, seqs, starts, rows, dtype=torch.float32, stream=None):
        """The values held: rows[i] positions from starts[i] of seqs[i], as (k
        [rows][kv_heads][qk_dim], v [rows][kv_heads][v_dim]); with layer None of
        every layer, [layers] in front."""
        s, ps, count = _ints(seqs)
        p, pp, m = _ints(starts)
        r, pr, m2 = _ints(rows)
        if not count == m == m2:
            raise ValueError("one start and one number of rows for each sequence")
        if dtype not in _TYPES:
            raise ValueError("f32, f16 or bf16")
        if layer is not None and int(layer) < 0:
            raise ValueError("no such layer")
        n = max(sum(r), 0)  # (a negative number among them is refused below)
        shape = (n, self.kv_heads) if layer is not None else (self.layers, n, self.kv_heads)
        with _on(stream):
            k = self._empty((*shape, self.qk_dim), dtype)
            v = torch.empty_like(k) if self.v_dim == self.qk_dim else self._empty((*shape, self.v_dim), dtype)
        nh._check(self._c.read(self.h, -1 if layer is None else int(layer), ps, pp, pr, count, k.data_ptr(),
                                      v.data_ptr(), _TYPES[dtype], nh._stream(stream)))
        return k, v

    def attend(self, layer: int, q: torch.Tensor, scale: float | None = None, sink: int = 0, ring: int = 0,
               out: torch.Tensor | None = None, lse: torch.Tensor | None = None, stream=None) -> torch.Tensor:
        """Attention of the batch's queries [rows][heads][qk_dim] over their
        sequences, each up to its own position; with a ring > 0 over the first
        `sink` positions and its last `ring`.  Returns [rows][heads][v_dim] of
        q's type (`out`, if given); lse (f32 [rows][heads]) takes the logs of
        the summed exponentials.  scale: 1 / sqrt(qk_dim) unless given."""
        heads = q.shape[1] if len(q.shape) == 3 else 0
        ldq = self._rows_of(q, heads, self.qk_dim, "q")
        with _on(stream):
            if out is None:
                out, ldo = q.new_empty((self._rows, heads, self.v_dim)), heads * self.v_dim
            else:
                ldo = self._rows_of(out, heads, self.v_dim, "out")
                if out.dtype != q.dtype:
                    raise ValueError("q and out differ in type")
            if lse is not None and (lse.dtype != torch.float32 or lse.shape != (q.shape[0], heads) or
                                    not lse.is_contiguous() or lse.get_device() != self._index):
                raise ValueError("lse is a contiguous f32 [rows][heads]")
            n = self._ws_bytes.get((heads, sink, ring))
            if n is None:
                n = self._c.attend_ws_bytes(self.h, heads, int(sink), int(ring))
                if n < 0:
                    nh._check(int(n))
                self._ws_bytes[heads, sink, ring] = n
            ws = self._empty((n,), torch.uint8) if n else None
        nh._check(self._c.attend(self.h, int(layer), q.data_ptr(), ldq, heads,
                                        float(self.qk_dim ** -0.5 if scale is None else scale), int(sink), int(ring),
                                        out.data_ptr(), ldo, _ptr(lse), _TYPES[q.dtype], _ptr(ws), n, nh._stream(stream)))
        return out

    def debug_kernel(self, kernel: int):
        """Attention by one of its kernels (nh_kv4_debug_kernel, nh_kv8_debug_kernel); tests only."""
        nh._check(self._c.debug_kernel(self.h, int(kernel)))
        self._ws_bytes = {}

    def __del__(self):
        if getattr(self, "h", None) and nh is not None and nh._lib is not None:
            self._c.free(self.h)
        self.h = None
