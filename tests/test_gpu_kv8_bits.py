"""How many bits attention over the 8-bit cache carries: scores whose products are exact, values that cancel, so that
neither the matrix instructions' cuts nor the output's own size hide a weight's rounding.

Queries are -1, 0 and 1: a product is a code (or a code + 128), and a sum of 256 of them has 17 bits, which no
instruction cuts off.  Values are +-c by the key's parity: what is left of them is small beside their size, which is
what a weight's error is multiplied by.  Each bound is checked to tell: the formula itself with a weight (a score) of
fewer bits is outside of it."""
import numpy as np
import pytest
import torch

import kv8_ref as ref
from kv4_ref import half_step
from test_gpu_kv8 import T, plain, rows_of

pytestmark = pytest.mark.gpu

DIMS = [(64, 64), (48, 64), (45, 51), (128, 128), (192, 128), (256, 256)]


def cut(x, bits):
    """x rounded to so many bits."""
    m, e = np.frexp(x)
    return np.ldexp(np.rint(m * 2.0 ** bits) * 2.0 ** -bits, e)


def case(qk, v, n, dtype, spread):
    """(q, k, v, scale): 2 kv heads, 33 rows of 4 heads; scores of standard deviation `spread`."""
    rng = np.random.default_rng(qk * 31 + n)
    q = torch.from_numpy(rng.integers(-1, 2, (33, 4, qk)).astype(np.float32)).to(T[dtype])
    k = torch.from_numpy(rng.standard_normal((n, 2, qk)).astype(np.float32)).to(T[dtype])
    size = 1.0 + rng.integers(0, 100, (1, 2, v)) / 16
    w = torch.from_numpy((np.where(np.arange(n) % 2, -1.0, 1.0)[:, None, None] * size).astype(np.float32)).to(T[dtype])
    return q, k, w, float(np.float32(spread / (0.82 * qk ** 0.5)))


def weights(q, hk, scale, g, h):
    s = (plain(q)[:, h].astype(np.float64) @ hk[:, g].astype(np.float64).T) * scale
    return s, np.exp(s - s.max(-1, keepdims=True))


def bound(o, hv, n, dtype, kernel):
    """The output's rounding, and of the values' size: a weight's, 2^-22 for two f16 parts, each off by half a step,
    2^-11 of itself (2^-11: bf16 and many rows, one part; with two keys both weights can be off by that, one up and
    one down, and their values' signs differ: 2^-11 of the size, not half of it); its score, in units of a factor
    2, rounded at 8 to 16 (2^-21), the exponential's last bit; an MFMA's cut at 2^-20 of its largest product, two
    parts; n / 16 roundings of sums."""
    many = kernel == 2 and dtype != "f32"
    bits = 2.0 ** -11 if dtype == "bf16" or many else 2.0 ** -22
    size = np.abs(hv).max()
    least = 2.0 ** -25 if dtype == "f16" else 0.0
    return half_step(dtype) * np.abs(o) * 1.01 + least + size * (bits + 2.0 ** -20 + 2.0 ** -22 + 2.0 ** -19 + n / 16 * 2.0 ** -24)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [2, 24, 300])
@pytest.mark.parametrize("qk,v", DIMS)
def test_weights_keep_their_bits(nh, qk, v, n, dtype):
    q, k, w, scale = case(qk, v, n, dtype, 2.0 ** -4)
    hk, hv = ref.quantize(plain(k)), ref.quantize(plain(w))
    o, l = ref.attend(plain(q), hk, hv, scale, ask=True)
    c = nh.KvCache8(1, 2, qk, v, pages=5, seqs=1, cap=n)
    s = c.new_seq()
    c.extend([s], [n])
    c.append(0, k.cuda(), w.cuda())
    c.ask([s], [33])
    for kernel in (1, 2):
        limit = bound(o, hv, n, dtype, kernel)
        coarse = kernel == 2 and dtype != "f32" or dtype == "bf16"
        if n < 100 or not coarse:
            off = np.zeros_like(o)
            for h in range(4):
                _, p = weights(q, hk, scale, h // 2, h)
                step = np.abs(hv[0, h // 2]).max() / 127
                off[:, h] = (cut(p * step, 8 if coarse else 11) / step) @ hv[:, h // 2] / p.sum(-1, keepdims=True) - o[:, h]
            assert (np.abs(off) > limit).any(), "the bound tells fewer bits"
        c.debug_kernel(kernel)
        lse = torch.empty(33, 4, dtype=torch.float32, device="cuda")
        got = plain(c.attend(0, q.cuda(), scale=scale, lse=lse)).astype(np.float64)
        assert (np.abs(got - o) <= limit).all(), (kernel, (np.abs(got - o) / limit).max())
        # a score as above, and f32 roundings of a logarithm of at most 2 log2(300)
        assert np.abs(plain(lse) - l).max() <= 2.0 ** -20 + 2.0 ** -19 + n / 16 * 2.0 ** -24, kernel


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("qk,v", DIMS)
def test_scores_keep_their_bits(nh, qk, v, dtype):
    """Scores up to 30: the logs of their sums."""
    n = 300
    q, k, w, scale = case(qk, v, n, dtype, 8.0)
    hk, hv = ref.quantize(plain(k)), ref.quantize(plain(w))
    _, l = ref.attend(plain(q), hk, hv, scale, ask=True)
    top, off = 0.0, np.zeros_like(l)
    for h in range(4):
        s, _ = weights(q, hk, scale, h // 2, h)
        top = max(top, np.abs(s).max())
        off[:, h] = np.log(np.exp(cut(s, 14)).sum(-1)) - l[:, h]
    # four f32 roundings of a score's factors and of its sum with the reference, in units of a factor 2 (and 15 more),
    # of the logarithm, and of the sum of weights
    limit = 5 * 2.0 ** -24 * (2 * top * 1.4427 + 15) + 2.0 ** -20
    assert (np.abs(off) > limit).any(), "the bound tells fewer bits"
    c = nh.KvCache8(1, 2, qk, v, pages=5, seqs=1, cap=n)
    s = c.new_seq()
    c.extend([s], [n])
    c.append(0, k.cuda(), w.cuda())
    c.ask([s], [33])
    for kernel in (1, 2):
        c.debug_kernel(kernel)
        lse = torch.empty(33, 4, dtype=torch.float32, device="cuda")
        c.attend(0, q.cuda(), scale=scale, lse=lse)
        assert np.abs(plain(lse) - l).max() <= limit, kernel


@pytest.mark.parametrize("qk,v", [(128, 128), (192, 128), (256, 256), (45, 51)])
@pytest.mark.parametrize("n", [20, 700, 6000])
def test_f32_attention_beside_a_plain_f32_evaluation_at_other_dims(nh, qk, v, n):
    """The error's norm against 64 bits, of the outputs and of lse: of the size of a plain f32 evaluation's."""
    rng = np.random.default_rng(n + qk)
    k, w, q = rows_of(rng, n, 2, qk, "f32"), rows_of(rng, n, 2, v, "f32"), rows_of(rng, 2, 4, qk, "f32")
    hk, hv = ref.quantize(plain(k)), ref.quantize(plain(w))
    scale = qk ** -0.5
    want, l = ref.attend(plain(q), hk, hv, scale, ask=True)
    c = nh.KvCache8(1, 2, qk, v, pages=24, seqs=1, cap=n, page=256)
    s = c.new_seq()
    c.extend([s], [n])
    c.append(0, k.cuda(), w.cuda())
    c.ask([s], [2])
    lse = torch.empty(2, 4, dtype=torch.float32, device="cuda")
    got = plain(c.attend(0, q.cuda(), lse=lse))
    a, b = (torch.from_numpy(np.repeat(x, 2, 1)).transpose(0, 1) for x in (hk, hv))
    t = torch.matmul(q.transpose(0, 1), a.transpose(1, 2)) * scale
    top = t.amax(-1, keepdim=True)
    p = torch.exp(t - top)
    other = plain((torch.matmul(p, b) / p.sum(-1, keepdim=True)).transpose(0, 1))
    other_l = plain((top + p.sum(-1, keepdim=True).log())[..., 0].T)
    for x, y, z in ((got, other, want), (plain(lse), other_l, l)):
        size = np.linalg.norm(z)
        mine, plain32 = (np.linalg.norm(r - z) / size for r in (x, y))
        # f32 sums of n keys: both within a few of the other; an MFMA's cut at 2^-20 of a product, over many, 2^-21
        assert mine <= 4 * plain32 + 2.0 ** -21, (n, mine, plain32)
