"""The 4-bit key/value cache and the check of drafted tokens over the C ABI
(nh_kv4_* and nh_verify_drafts in include/needle_hip.h).  Neither has a
counterpart in the reference."""
from __future__ import annotations

import array
import contextlib
import ctypes as C

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


def _ptr(t):
    return t.data_ptr() if t is not None else None


class KvCache4:
    """A paged cache of keys and values in 4 bits, shared by many sequences
    (nh_kv4).  A step: `extend` names its sequences and their new rows; then,
    for every layer, `append` stores the rows' keys and values and `attend`
    attends with their queries."""

    def __init__(self, layers: int, kv_heads: int, qk_dim: int, v_dim: int, pages: int, seqs: int, cap: int,
                 group: int = 32, page: int = 64):
        lib = nh.load_library()
        self.h = None
        if torch.cuda.is_available():
            nh.init()
        h = C.c_void_p()
        nh._check(lib.nh_kv4_new(int(layers), int(kv_heads), int(qk_dim), int(v_dim), int(group), int(page), int(pages),
                                 int(seqs), int(cap), C.byref(h)))
        self.h = h
        self.layers, self.kv_heads, self.qk_dim, self.v_dim = int(layers), int(kv_heads), int(qk_dim), int(v_dim)
        self.group, self.page, self.pages = int(group), int(page), int(pages)
        self.device = torch.device("cuda", torch.cuda.current_device())
        self._index = self.device.index
        self._rows = 0  # the batch's

    # ---- sequences
    def new_seq(self) -> int:
        """An empty sequence's id."""
        return nh._check(nh._lib.nh_kv4_seq_new(self.h))

    def length(self, seq: int) -> int:
        return nh._check(nh._lib.nh_kv4_seq_len(self.h, int(seq)))

    def free(self, seq: int):
        """Gives back the pages that no branch shares."""
        nh._check(nh._lib.nh_kv4_seq_free(self.h, int(seq)))
        self._rows = self.rows  # (the batch may be over)

    def truncate(self, seq: int, length: int):
        """Forgets positions `length` and on."""
        nh._check(nh._lib.nh_kv4_seq_truncate(self.h, int(seq), int(length)))
        self._rows = self.rows

    def fork(self, seq: int, n: int = 1) -> list:
        """n branches that share the sequence's pages until they are written."""
        out = (C.c_int * max(int(n), 1))()
        nh._check(nh._lib.nh_kv4_seq_fork(self.h, int(seq), int(n), C.addressof(out)))
        self._rows = self.rows
        return out[:n]

    def copy(self, seq: int, stream=None) -> int:
        """A branch with pages of its own."""
        made = nh._check(nh._lib.nh_kv4_seq_copy(self.h, int(seq), nh._stream(stream)))
        self._rows = self.rows
        return made

    def compact(self, seqs, ranges, stream=None):
        """Sequence seqs[i] keeps the positions of ranges[i], ascending (begin,
        end) pairs, closed up."""
        if len(ranges) != len(seqs):
            raise ValueError("one list of ranges for each sequence")
        if any(len(pair) != 2 for r in ranges for pair in r):
            raise ValueError("a range is a (begin, end) pair")
        s, ps, n = _ints(seqs)
        counts, pc, _ = _ints([len(r) for r in ranges])
        flat, pf, _ = _ints([x for r in ranges for pair in r for x in pair])
        nh._check(nh._lib.nh_kv4_seq_compact(self.h, ps, n, pc, pf, nh._stream(stream)))
        self._rows = self.rows

    @property
    def free_pages(self) -> int:
        return nh._check(nh._lib.nh_kv4_free_pages(self.h))

    def bytes(self) -> int:
        n = nh._lib.nh_kv4_bytes(self.h)
        nh._check(-1 if n < 0 else 0)
        return n

    # ---- rows
    def extend(self, seqs, rows, stream=None):
        """rows[i] more positions for each sequence; they become the batch."""
        s, ps, n = _ints(seqs)
        r, pr, m = _ints(rows)
        if n != m:
            raise ValueError("one number of rows for each sequence")
        nh._check(nh._lib.nh_kv4_extend(self.h, ps, pr, n, nh._stream(stream)))
        self._rows = sum(r)

    @property
    def rows(self) -> int:
        """The batch's rows."""
        return nh._check(nh._lib.nh_kv4_rows(self.h))

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

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, stream=None):
        """The batch's keys [rows][kv_heads][qk_dim] and values [rows][kv_heads][v_dim]
        into one layer; rows may be a view of a wider matrix's columns."""
        ldk = self._rows_of(k, self.kv_heads, self.qk_dim, "k")
        ldv = self._rows_of(v, self.kv_heads, self.v_dim, "v")
        if k.dtype != v.dtype:
            raise ValueError("k and v differ in type")
        nh._check(nh._lib.nh_kv4_append(self.h, int(layer), k.data_ptr(), v.data_ptr(), ldk, ldv, _TYPES[k.dtype],
                                        nh._stream(stream)))

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
        n = sum(x for x in r if x > 0)
        shape = (n, self.kv_heads) if layer is not None else (self.layers, n, self.kv_heads)
        with _on(stream):
            k = torch.empty((*shape, self.qk_dim), dtype=dtype, device=self.device)
            v = torch.empty((*shape, self.v_dim), dtype=dtype, device=self.device)
        nh._check(nh._lib.nh_kv4_read(self.h, -1 if layer is None else int(layer), ps, pp, pr, count, k.data_ptr(),
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
                out, ldo = torch.empty((self._rows, heads, self.v_dim), dtype=q.dtype, device=self.device), heads * self.v_dim
            else:
                ldo = self._rows_of(out, heads, self.v_dim, "out")
                if out.dtype != q.dtype:
                    raise ValueError("q and out differ in type")
            if lse is not None and (lse.dtype != torch.float32 or lse.shape != (q.shape[0], heads) or
                                    not lse.is_contiguous() or lse.get_device() != self._index):
                raise ValueError("lse is a contiguous f32 [rows][heads]")
            n = nh._lib.nh_kv4_attend_ws_bytes(self.h, heads, int(sink), int(ring))
            if n < 0:
                nh._check(int(n))
            ws = torch.empty(n, dtype=torch.uint8, device=self.device) if n else None
        nh._check(nh._lib.nh_kv4_attend(self.h, int(layer), q.data_ptr(), ldq, heads,
                                        float(self.qk_dim ** -0.5 if scale is None else scale), int(sink), int(ring),
                                        out.data_ptr(), ldo, _ptr(lse), _TYPES[q.dtype], _ptr(ws), n, nh._stream(stream)))
        return out

    def debug_kernel(self, kernel: int):
        """Attention by one of its kernels (nh_kv4_debug_kernel); tests only."""
        nh._check(nh._lib.nh_kv4_debug_kernel(self.h, int(kernel)))

    def __del__(self):
        if getattr(self, "h", None) and nh is not None and nh._lib is not None:
            nh._lib.nh_kv4_free(self.h)
        self.h = None


def _row_stride(t, index, what):
    """Elements from one row of [batch][rows][vocab] to the next."""
    if t.dtype not in _TYPES or t.get_device() != index or index < 0:
        raise ValueError(f"{what}: f32, f16 or bf16 on the logits' device")
    b, r, v = t.shape
    sb, sr, sv = t.stride()
    ld = sr if r > 1 else sb if b > 1 else v
    if v > 1 and sv != 1 or b > 1 and sb != ld * r:
        raise ValueError(f"the rows of {what} do not follow each other")
    if ld < v and b * r:
        # (one row expanded to many holds fewer elements than rows of v would)
        raise ValueError(f"the rows of {what} repeat or overlap: make them contiguous")
    return max(ld, v)


def _plain(t, dtype, shape, index, what):
    if t.dtype != dtype or t.shape != shape or not t.is_contiguous() or t.get_device() != index:
        raise ValueError(f"{what}: contiguous {dtype} {list(shape)} on the logits' device")


class _DraftCheck:
    """One check of drafts, its arguments looked over and its outputs and
    workspace there; `run` queues it on the current stream.  What can be refused
    is refused here, so that a session is fed after it."""

    def __init__(self, logits, drafts, u=None, probs=None, counts=None, temperature=1.0):
        if not nh._ready:
            nh.init()
        if len(logits.shape) != 3 or len(drafts.shape) != 2:
            raise ValueError("logits are [batch][n + 1][vocab], drafts [batch][n]")
        batch, rows, vocab = logits.shape
        n, index = rows - 1, logits.get_device()
        ldl, ldp = _row_stride(logits, index, "logits"), 0
        _plain(drafts, torch.int32, (batch, n), index, "drafts")
        if u is not None:
            _plain(u, torch.float32, (batch, n + 1), index, "u")
        if counts is not None:
            _plain(counts, torch.int32, (batch,), index, "counts")
        if probs is not None:
            if probs.shape != (batch, n, vocab):
                raise ValueError("probs are [batch][n][vocab]")
            ldp = _row_stride(probs, index, "probs") if batch * n else vocab
        if index != torch.cuda.current_device():
            raise ValueError("the tensors are on another device than the current one")
        temperature = C.c_float(float(temperature)).value  # (as the entry takes it)
        if not 0.0 <= temperature < float("inf") or temperature > 0.0 and u is None:
            raise nh.NeedleHipError(-1, "a temperature is 0 (greedy), or positive with uniforms")
        ws_bytes = nh._lib.nh_verify_drafts_ws_bytes(batch, n, vocab)
        if ws_bytes < 0:
            nh._check(int(ws_bytes))
        self.accepted = torch.empty(batch, dtype=torch.int32, device=logits.device)
        self.tokens = torch.empty((batch, n + 1), dtype=torch.int32, device=logits.device)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=logits.device) if ws_bytes else None
        self._held = (logits, drafts, counts, probs, u, ws)
        self._args = (logits.data_ptr(), _TYPES[logits.dtype], ldl, _ptr(drafts), _ptr(counts), _ptr(probs),
                      _TYPES[probs.dtype] if probs is not None else 0, ldp, _ptr(u), temperature, batch, n, vocab,
                      self.accepted.data_ptr(), self.tokens.data_ptr(), _ptr(ws), ws_bytes)

    def run(self):
        nh._check(nh._lib.nh_verify_drafts(*self._args, nh._stream()))
        return self.accepted, self.tokens


def verify_drafts(logits: torch.Tensor, drafts: torch.Tensor, u: torch.Tensor | None = None,
                  probs: torch.Tensor | None = None, counts: torch.Tensor | None = None, temperature: float = 1.0,
                  stream=None):
    """Drafted tokens [batch][n] (int32) against the target's logits [batch][n +
    1][vocab] from uniforms u [batch][n + 1] (nh_verify_drafts): (accepted
    [batch], tokens [batch][n + 1]: the kept drafts, the next token, then -1),
    int32.  probs [batch][n][vocab]: the drafter's probabilities (None: it has
    none); counts [batch]: drafts of each sequence (None: n); temperature 0:
    greedy.  Rows of logits and probs may be padded (a view of wider rows), not
    repeated (an expanded row)."""
    with _on(stream):
        return _DraftCheck(logits, drafts, u, probs, counts, temperature).run()
