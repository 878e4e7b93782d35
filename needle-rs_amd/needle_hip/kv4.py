"""The 4-bit key/value cache and the check of drafted tokens over the C ABI
(nh_kv4_* and nh_verify_drafts in include/needle_hip.h).  Neither has a
counterpart in the reference."""
from __future__ import annotations

import ctypes as C

import torch

import needle_hip as nh

from .kvcache import _TYPES, PagedCache, _ints, _on, _ptr


class KvCache4(PagedCache):
    """A paged cache of keys and values in 4 bits, shared by many sequences
    (nh_kv4).  A step: `extend` names its sequences and their new rows; then,
    for every layer, `append` stores the rows' keys and values and `attend`
    attends with their queries."""

    def __init__(self, layers: int, kv_heads: int, qk_dim: int, v_dim: int, pages: int, seqs: int, cap: int,
                 group: int = 32, page: int = 64):
        self._make("kv4", layers, kv_heads, qk_dim, v_dim, pages, page,
                   (int(layers), int(kv_heads), int(qk_dim), int(v_dim), int(group), int(page), int(pages), int(seqs), int(cap)))
        self.group = int(group)

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
        self._batch(self.rows)

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, stream=None):
        """The batch's keys [rows][kv_heads][qk_dim] and values [rows][kv_heads][v_dim]
        into one layer; rows may be a view of a wider matrix's columns."""
        ldk = self._rows_of(k, self.kv_heads, self.qk_dim, "k")
        ldv = self._rows_of(v, self.kv_heads, self.v_dim, "v")
        if k.dtype != v.dtype:
            raise ValueError("k and v differ in type")
        nh._check(nh._lib.nh_kv4_append(self.h, int(layer), k.data_ptr(), v.data_ptr(), ldk, ldv, _TYPES[k.dtype],
                                        nh._stream(stream)))


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
