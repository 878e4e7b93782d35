"""Plans of rotary positions, and what they refuse, before any device work (no
GPU needed: the last check is nh_init's)."""
import ctypes as C

import numpy as np
import pytest

import needle_hip as nh
import rope_ref as ref

EINVAL, ESTATE = -1, -5
KINDS = {"plain": 0, "linear": 1, "base": 2, "parts": 3, "bands": 4}


def freqs(dim=64, theta=10000.0, scaling=0, factor=8.0, original=8192.0, low=1.0, high=32.0, out=True):
    lib = nh.load_library()
    f, a = np.zeros(128), C.c_double()
    rc = lib.nh_rope_freqs(dim, theta, scaling, factor, original, low, high, f.ctypes.data_as(C.c_void_p) if out else None,
                           C.byref(a))
    return rc if rc else (f[:dim // 2], a.value)


@pytest.mark.parametrize("dim", [2, 4, 48, 64, 96, 128, 256])
@pytest.mark.parametrize("theta", [10000.0, 500000.0, 1.5])
@pytest.mark.parametrize("scaling", [("plain",), ("linear", 4.0), ("base", 8.0), ("parts", 16.0, 4096.0, 1.0, 32.0),
                                     ("parts", 4.0, 8192.0, 0.5, 20.0), ("bands", 8.0, 8192.0, 1.0, 4.0), ("bands", 1.0, 100.0, 1.0, 4.0)])
def test_frequencies(dim, theta, scaling):
    kind, *args = scaling
    named = dict(zip(("factor", "original", "low", "high"), args))
    got, amplitude = freqs(dim, theta, KINDS[kind], **named)
    want, a = ref.frequencies(dim, theta, scaling)
    # (a power, a logarithm and a few products in 64 bits: a few of their roundings)
    assert np.allclose(got, want, rtol=1e-13, atol=0)
    assert abs(amplitude - a) < 1e-14
    assert (np.diff(got) < 0).all() or dim == 2


def test_scalings_ends():
    """base: the quickest pair keeps its frequency, the slowest is slowed by the factor; bands and parts: both as their ends say."""
    plain, _ = freqs()
    base, _ = freqs(scaling=2)
    assert base[0] == plain[0] and abs(base[-1] * 8 / plain[-1] - 1) < 1e-12
    for kind in (3, 4):
        f, _ = freqs(scaling=kind, high=32.0 if kind == 3 else 4.0)
        assert f[0] == plain[0] and abs(f[-1] * 8 / plain[-1] - 1) < 1e-12


@pytest.mark.parametrize("over", [dict(dim=0), dict(dim=3), dict(dim=258), dict(dim=-2), dict(theta=1.0), dict(theta=float("nan")),
                                  dict(theta=float("inf")), dict(scaling=-1), dict(scaling=5), dict(scaling=1, factor=0.5),
                                  dict(scaling=1, factor=float("nan")), dict(scaling=3, original=0.0),
                                  dict(scaling=4, original=float("inf")), dict(scaling=4, low=0.0), dict(scaling=3, low=32.0),
                                  dict(scaling=4, high=float("nan")), dict(out=False)])
def test_frequencies_refused(over):
    assert freqs(**over) == EINVAL
    assert nh.load_library().nh_last_error()


def new(f=(1.0, 0.1), pairs=None, amplitude=1.0, layout=0):
    lib = nh.load_library()
    f = np.array(f, np.float64)
    h = C.c_void_p()
    rc = lib.nh_rope_new(f.ctypes.data_as(C.c_void_p), len(f) if pairs is None else pairs, amplitude, layout, C.byref(h))
    if h.value:
        lib.nh_rope_free(h)
    return rc


@pytest.mark.parametrize("over", [dict(pairs=0), dict(pairs=129), dict(f=(float("nan"),)), dict(f=(float("inf"),)),
                                  dict(f=(2e6,)), dict(amplitude=float("nan")), dict(amplitude=float("inf")), dict(layout=2),
                                  dict(layout=-1)])
def test_plans_refused(over):
    assert new(**over) == EINVAL


def test_null_handles_and_before_init():
    lib = nh.load_library()
    one = np.zeros(4, np.int32)
    p = one.ctypes.data_as(C.c_void_p)
    assert lib.nh_rope_new(p, 1, 1.0, 0, None) == EINVAL
    assert lib.nh_rope_new(None, 1, 1.0, 0, C.byref(C.c_void_p())) == EINVAL
    assert lib.nh_rope_free(None) == 0
    assert lib.nh_rope_apply(None, p, 1, 2, p, 2, 1, p, 2, None, 0, 0, None, 0, 0, 0, None) == EINVAL
    if not nh._ready:
        assert new() == ESTATE


@pytest.mark.parametrize("scaling", [("else", 2.0), ("linear",), ("linear", 2.0, 3.0), ("parts", 2.0), ("bands", 2.0, 3.0, 4.0)])
def test_python_scalings_refused(scaling):
    with pytest.raises(ValueError):
        nh.Rope(64, scaling=scaling)


def test_python_layout_refused():
    with pytest.raises(ValueError):
        nh.Rope(64, layout="thirds")
