"""The 4-bit cache's format, its attention and the check of drafts by plain
numpy in 64 bits (codes by the format's 32-bit rule), for the tests."""
import numpy as np

F32 = np.float32
THIRD = np.frombuffer(np.uint32(0x3D888889).tobytes(), F32)[0]  # f32(1/15)


def quantize(x, group):
    """x f32 [..., d] (finite, or a group with NaN / infinity): the values held, f64."""
    x = np.asarray(x, F32)
    out = np.empty(x.shape, np.float64)
    for a in range(0, x.shape[-1], group):
        y = x[..., a:a + group]
        bad = ~np.isfinite(y).all(-1)
        with np.errstate(all="ignore"):
            y = np.where(np.isnan(y), F32(0), np.clip(y, F32(-65504), F32(65504)))
            mn, mx = y.min(-1), y.max(-1)
            low = mn.astype(np.float16)
            step = ((mx - mn) * THIRD).astype(np.float16)
            inv = np.where(step > 0, F32(1) / np.where(step > 0, step.astype(F32), F32(1)), F32(0))
            c = np.clip(np.rint((y - low.astype(F32)[..., None]) * inv[..., None]), 0, 15)
        out[..., a:a + group] = low.astype(np.float64)[..., None] + step.astype(np.float64)[..., None] * c
        out[..., a:a + group][bad] = np.nan
    return out


def attend(q, k, v, scale, sink=0, ring=0):
    """q [rows][heads][dk] of the last rows, k [len][kv][dk], v [len][kv][dv]: (o, lse), f64."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    rows, heads, _ = q.shape
    n, kv, _ = k.shape
    o = np.zeros((rows, heads, v.shape[-1]))
    lse = np.zeros((rows, heads))
    i = np.arange(n - rows, n)[:, None]
    j = np.arange(n)[None]
    seen = j <= i
    if ring:
        seen = seen & ((j < sink) | (j > i - ring))
    for h in range(heads):
        g = h // (heads // kv)
        for r in range(rows):
            at = np.flatnonzero(seen[r])
            s = (k[at, g] @ q[r, h]) * scale
            m = s.max()
            p = np.exp(s - m)
            o[r, h] = p @ v[at, g] / p.sum()
            lse[r, h] = m + np.log(p.sum())
    return o, lse


def half_step(dtype):
    return {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[dtype]


def attend_bound(q, k, v, o, scale, dtype):
    """How far an output may be from the exact one, by arithmetic.

    The output's rounding; the weights' (11 bits, f32 calls 22: half a step of
    each on step x code, which spans at most twice the largest |v|); the
    scores', d products summed in f32 (d + 16 roundings of at most scale
    sum |q||k|), which change a weight by that much, and numerator and
    denominator alike; exp and the running sums, a rounding a key."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    size = np.abs(q).sum(-1).max() * np.abs(k).max() * abs(scale)
    delta = (q.shape[-1] + 16) * 2.0 ** -24 * size
    vmax = np.abs(v).max() if v.size else 0.0
    weight = 2.0 ** -21 if dtype == "f32" else 2.0 ** -11
    return half_step(dtype) * np.abs(o) + vmax * (weight + 4 * delta + 4 * (len(k) + 64) * 2.0 ** -24) + 1e-30


def verify(logits, drafts, u, probs=None, counts=None, temperature=1.0):
    """(accepted, tokens) of the check of drafts, logits f32 [b][n + 1][v], in 64 bits."""
    b, rows, vocab = logits.shape
    n = rows - 1
    accepted = np.zeros(b, np.int32)
    tokens = np.full((b, rows), -1, np.int32)

    def best(x):
        if np.isnan(x[0]):
            return 0
        y = np.where(np.isnan(x), -np.inf, x)
        return int(y.argmax())

    def weights(x):
        x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
        m = x.max()
        if m == -np.inf:
            return np.zeros(vocab)
        with np.errstate(invalid="ignore"):
            w = np.where(x == m, 1.0, np.where(np.isinf(x), 0.0, np.exp((x - m) / temperature)))
        return w / w.sum()

    for s in range(b):
        cnt = n if counts is None else int(np.clip(counts[s], 0, n))
        kept = 0
        for i in range(cnt):
            x = int(drafts[s, i])
            if not 0 <= x < vocab:
                break
            if temperature == 0:
                if x != best(logits[s, i]):
                    break
            else:
                qx = 1.0 if probs is None else float(probs[s, i, x])
                if not float(u[s, i]) * qx < weights(logits[s, i])[x]:
                    break
            kept += 1
        row = logits[s, kept]
        if temperature == 0:
            pick = best(row)
        else:
            p = weights(row)
            w = p
            if kept < cnt:
                if probs is None:
                    w = p.copy()
                    if 0 <= drafts[s, kept] < vocab:
                        w[drafts[s, kept]] = 0.0
                else:
                    d = p - probs[s, kept].astype(np.float64)
                    w = np.where(d > 0, d, 0.0)
                if not w.sum() > 0:
                    w = p
            if not w.sum() > 0:
                pick = best(row)
            else:
                c = np.cumsum(w)
                over = np.flatnonzero(c > float(u[s, n]) * c[-1])
                last = int(np.flatnonzero(w > 0)[-1])
                pick = min(int(over[0]), last) if over.size else last
        accepted[s] = kept
        tokens[s, :kept] = drafts[s, :kept]
        tokens[s, kept] = pick
    return accepted, tokens
