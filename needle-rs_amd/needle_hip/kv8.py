"""The 8-bit key/value cache over the C ABI (nh_kv8_* in include/needle_hip.h).
No counterpart in the reference."""
from __future__ import annotations

import torch

import needle_hip as nh

from .kvcache import _TYPES, PagedCache, _ints, _like, _on
from .rope import Rope


class KvCache8(PagedCache):
    """A paged cache of keys and values in 8 bits, a step for each block of 16
    positions and head, shared by many sequences (nh_kv8).  A step: `extend`
    names its sequences and their new rows; then, for every layer, `append`
    stores the rows' keys and values (with a Rope, turns keys and queries on the
    way) and `attend` attends with their queries.  `ask` instead of `extend`:
    rows of queries alone, each of which sees its whole sequence (a decoder's
    rows and their encoder's states)."""

    _CALLS = PagedCache._CALLS + ("ask", "end_batch")

    def __init__(self, layers: int, kv_heads: int, qk_dim: int, v_dim: int, pages: int, seqs: int, cap: int, page: int = 64):
        self._make("kv8", layers, kv_heads, qk_dim, v_dim, pages, page,
                   (int(layers), int(kv_heads), int(qk_dim), int(v_dim), int(page), int(pages), int(seqs), int(cap)))

    def _changed(self, call, args, stream):
        """A call that may end the batch: the device is told (before it, end_batch checks for a capture alone)."""
        st = nh._stream(stream)
        nh._check(self._c.end_batch(self.h, st))
        made = call(*args)
        nh._check(self._c.end_batch(self.h, st))
        return made

    def free(self, seq: int, stream=None):
        """Gives back the pages that no branch shares.  free, truncate and fork do device work only where an
        append was captured, whose replays then store nothing until the next extend."""
        self._changed(super().free, (seq,), stream)

    def truncate(self, seq: int, length: int, stream=None):
        """Forgets positions `length` and on.  Rows that are kept beside them in a block of 16 stay as they
        are held: a step that a forgotten row has doubled is not halved again."""
        self._changed(super().truncate, (seq, length), stream)

    def fork(self, seq: int, n: int = 1, stream=None) -> list:
        """n branches that share the sequence's pages until they are written."""
        return self._changed(super().fork, (seq, n), stream)

    def ask(self, seqs, rows, stream=None):
        """rows[i] query rows for each sequence; they become the batch, and no
        position is added."""
        s, ps, n = _ints(seqs)
        r, pr, m = _ints(rows)
        if n != m:
            raise ValueError("one number of rows for each sequence")
        nh._check(self._c.ask(self.h, ps, pr, n, nh._stream(stream)))
        self._batch(sum(r))

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, rope: Rope | None = None,
               positions: torch.Tensor | None = None, q: torch.Tensor | None = None, out: torch.Tensor | None = None,
               stream=None):
        """The batch's keys [rows][kv_heads][qk_dim] and values [rows][kv_heads][v_dim]
        into one layer; rows may be a view of a wider matrix's columns.  rope: keys
        are turned first, to their positions in their sequences or to `positions`
        (int32 [rows]); q [rows][heads][qk_dim] is turned with them, in the same
        launch, into `out` (q itself: in place; None: a new tensor), which is
        returned."""
        ldk = self._rows_of(k, self.kv_heads, self.qk_dim, "k")
        ldv = self._rows_of(v, self.kv_heads, self.v_dim, "v")
        t = k.dtype
        if t != v.dtype:
            raise ValueError("k and v differ in type")
        if rope is None:
            if positions is not None or q is not None or out is not None:
                raise ValueError("positions and queries go with a rope")
            nh._check(self._c.append(self.h, int(layer), k.data_ptr(), v.data_ptr(), ldk, ldv, _TYPES[t], None, None, None, 0,
                                     0, None, 0, nh._stream(stream)))
            return None
        pos = rope._positions(positions, self._rows) if positions is not None else None
        heads = ldq = ldo = 0
        pq = po = None
        if q is not None:
            heads = q.shape[1] if len(q.shape) == 3 else 0
            ldq = self._rows_of(q, heads, self.qk_dim, "q")
            if q.dtype != t:
                raise ValueError("q and k differ in type")
            if out is None:
                with _on(stream):
                    out = _like(q)
                ldo = heads * self.qk_dim
            else:
                ldo = self._rows_of(out, heads, self.qk_dim, "out")
                if out.dtype != t:
                    raise ValueError("q and out differ in type")
            pq, po = q.data_ptr(), out.data_ptr()
        elif out is not None:
            raise ValueError("an out goes with queries")
        nh._check(self._c.append(self.h, int(layer), k.data_ptr(), v.data_ptr(), ldk, ldv, _TYPES[t], rope.h, pos, pq, ldq,
                                 heads, po, ldo, nh._stream(stream)))
        return out
