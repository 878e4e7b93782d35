"""The 8-bit cache's format and its attention by plain numpy, for the tests."""
import copy

import numpy as np

from kv4_ref import half_step

F32 = np.float32
BLOCK = 16


class Side:
    """The keys (or values) of one sequence in one layer: whole numbers, steps, marked rows."""

    def __init__(self, heads, dim):
        self.heads, self.dim = heads, dim
        self.codes = np.zeros((0, heads, dim), np.float64)
        self.bad = np.zeros((0, heads), bool)
        self.steps = np.zeros((0, heads), F32)

    def store(self, x):
        """Rows x [n][heads][dim] of one call, a block at a time by the 32-bit rule."""
        x = np.asarray(x, F32)
        at = len(self.codes)
        self.codes = np.concatenate([self.codes, np.zeros(x.shape)])
        self.bad = np.concatenate([self.bad, ~np.isfinite(x).all(-1)])
        self.steps = np.concatenate([self.steps, np.zeros((-(-len(self.codes) // BLOCK) - len(self.steps), self.heads), F32)])
        while len(x):
            b, slot = divmod(at, BLOCK)
            n = min(BLOCK - slot, len(x))
            for h in range(self.heads):
                rows = np.where(self.bad[at:at + n, h, None], F32(0), x[:n, h])
                need = np.abs(rows).max() * F32(1 / 127)
                need = F32(0) if need < 2.0 ** -120 else need
                step = self.steps[b, h] if slot else F32(0)
                if step > 0:
                    halvings = 0
                    while step < need:
                        step, halvings = step * F32(2), halvings + 1
                    before = self.codes[at - slot:at, h]
                    before[:] = np.rint(before * 2.0 ** -halvings)
                else:
                    step = need
                with np.errstate(all="ignore"):
                    inv = F32(1) / step if step > 0 else F32(0)
                    self.codes[at:at + n, h] = np.clip(np.rint(rows * inv), -127, 127)
                self.steps[b, h] = step
            at += n
            x = x[n:]

    def cut(self, n):
        self.codes, self.bad, self.steps = self.codes[:n], self.bad[:n], self.steps[:-(-n // BLOCK)]

    def held(self):
        """The values held, f64, NaN where a row was marked."""
        y = self.codes * np.repeat(self.steps, BLOCK, 0)[:len(self.codes), :, None].astype(np.float64)
        y[self.bad] = np.nan
        return y

    def held32(self):
        with np.errstate(invalid="ignore"):
            return (self.codes.astype(F32) * np.repeat(self.steps, BLOCK, 0)[:len(self.codes), :, None]) * \
                np.where(self.bad, F32(np.nan), F32(1))[..., None]

    def fork(self):
        return copy.deepcopy(self)


def quantize(x, cuts=()):
    """The values that rows x [n][heads][dim] are held as, stored in calls cut at `cuts`; f32."""
    s = Side(x.shape[1], x.shape[2])
    last = 0
    for c in (*cuts, len(x)):
        if c > last:
            s.store(x[last:c])
        last = c
    return s.held32()


def seen_by(rows, n, sink=0, ring=0, ask=False):
    """[rows][n]: which keys a row sees."""
    i = np.full(rows, n - 1)[:, None] if ask else np.arange(n - rows, n)[:, None]
    j = np.arange(n)[None]
    seen = j <= i
    if ring:
        seen = seen & ((j < sink) | (j > i - ring))
    return seen


def attend(q, k, v, scale, sink=0, ring=0, ask=False):
    """q [rows][heads][dk], k [len][kv][dk], v [len][kv][dv] as held: (o, lse), f64; no key: 0, -inf."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    rows, heads, _ = q.shape
    n, kv, _ = k.shape
    seen = seen_by(rows, n, sink, ring, ask)
    o = np.zeros((rows, heads, v.shape[-1]))
    lse = np.full((rows, heads), -np.inf)
    for h in range(heads):
        g = h // (heads // kv)
        s = np.where(seen, (q[:, h] @ np.nan_to_num(k[:, g]).T) * scale, -np.inf)
        s = np.where(seen & (np.isnan(k[:, g]).any(-1) | np.isnan(v[:, g]).any(-1)), np.nan, s)
        for r in range(rows):
            at = np.flatnonzero(seen[r])
            if not len(at):
                continue
            m = np.max(s[r, at])
            p = np.exp(s[r, at] - m)
            o[r, h] = p @ v[at, g] / p.sum()
            lse[r, h] = m + np.log(p.sum())
    return o, lse


def attend_bound(q, k, v, o, scale, dtype, many=False):
    """How far an output may be from the exact one, by arithmetic.

    The output's rounding.  The scores: an f16 MFMA cuts its products off at
    2^-20 of the largest (d of them, and 16 roundings of sums), an f32 query's
    whole numbers are off by 2^-24 of the row's largest each (the products are
    exact, their sum is rounded twice); a score off by e changes a weight by e,
    numerator and denominator alike: 2 delta.  A key of few rows enters as code + 128, so
    the largest product is up to 255 / 127 of a code's: 4.016 delta.  The weights: 11 bits (22 in f32 and f16
    calls of few rows), f16 values of many rows 11 bits of their own; 32
    products of an MFMA cut off at 2^-20 of its largest, the largest of all
    MFMAs adding up to at most 1; a rounding a key in the running sums."""
    q, k, v = (np.nan_to_num(np.asarray(a, np.float64)) for a in (q, k, v))
    d, kmax = q.shape[-1], np.abs(k).max() if k.size else 0.0
    qmax, qsum = (np.abs(q).max(), np.abs(q).sum(-1).max()) if q.size else (0.0, 0.0)
    if dtype == "f32":
        delta = abs(scale) * kmax * (d * 2.0 ** -23 * qmax + 8 * 2.0 ** -24 * qsum)
    else:
        delta = abs(scale) * kmax * (d * 2.0 ** -20 * qmax + 16 * 2.0 ** -24 * qsum)
    vmax = np.abs(v).max() if v.size else 0.0
    weight = 2.0 ** -11 * (2 if many else 1) if dtype == "bf16" or many else 2.0 ** -21
    rounding = half_step(dtype) * np.abs(o) * 1.01 + (2.0 ** -24 if dtype == "f16" else 0.0)
    return rounding + vmax * (weight + 2.0 ** -15 + 4.016 * delta + 4 * (len(k) + 64) * 2.0 ** -24) + 1e-30
