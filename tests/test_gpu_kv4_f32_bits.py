"""f32 attention over the 4-bit cache holds 22 bits of queries and of weights: its distance from the 64-bit result beside
that of a plain evaluation in f32's 24 bits."""
import numpy as np
import pytest

import kv4_ref as ref
from test_gpu_kv4 import filled, plain, rows_of

pytestmark = pytest.mark.gpu


def attend32(q, k, v, scale):
    """The last row's attention in f32, one product and one sum after the other: q [heads][dk], k [n][kv][dk], v .."""
    q, k, v, scale = q.astype(np.float32), k.astype(np.float32), v.astype(np.float32), np.float32(scale)
    heads, kv = q.shape[0], k.shape[1]
    out = np.zeros((heads, v.shape[-1]), np.float32)
    for h in range(heads):
        g = h // (heads // kv)
        s = np.cumsum(k[:, g] * q[h], axis=1, dtype=np.float32)[:, -1] * scale
        p = np.exp(s - s.max())
        out[h] = np.cumsum(p[:, None] * v[:, g], axis=0, dtype=np.float32)[-1] / np.cumsum(p, dtype=np.float32)[-1]
    return out


@pytest.mark.parametrize("qk,v,group,n", [(48, 64, 32, 300), (128, 128, 32, 1000), (128, 128, 64, 90), (256, 256, 64, 200)])
def test_f32_calls_hold_22_bits(nh, qk, v, group, n):
    """At most four times the plain f32 evaluation's distance: a rounding to 22 bits is four of 24 (a part of a query
    or a weight left out is past it several hundred times)."""
    rng = np.random.default_rng(qk + n)
    c, ids, ks, vs = filled(nh, rng, [n], 2, qk, v, group, 32, "f32", last=[1])
    q = rows_of(rng, 1, 12, qk, "f32")
    o = plain(c.attend(0, q.cuda())).astype(np.float64)[0]
    k, w = ref.quantize(plain(ks[0][0]), group), ref.quantize(plain(vs[0][0]), group)
    want, _ = ref.attend(plain(q), k, w, qk ** -0.5)
    off, off32 = np.linalg.norm(o - want[0]), np.linalg.norm(attend32(plain(q)[0], k, w, qk ** -0.5) - want[0])
    assert off <= 4.0 * off32, (off / off32, off / np.linalg.norm(want))
