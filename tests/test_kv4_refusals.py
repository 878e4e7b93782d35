"""Arguments that the 4-bit cache and the check of drafts refuse, before any
device work (no GPU needed: the last check is nh_init's)."""
import ctypes as C

import numpy as np
import pytest
import torch

import needle_hip as nh

GOOD = dict(layers=2, kv_heads=2, qk_dim=48, v_dim=64, group=32, page=32, pages=8, seqs=3, cap=100)
EINVAL, ESTATE = -1, -5


def new(**over):
    lib = nh.load_library()
    h = C.c_void_p()
    a = {**GOOD, **over}
    rc = lib.nh_kv4_new(*[a[k] for k in GOOD], C.byref(h))
    if h.value:
        lib.nh_kv4_free(h)
    return rc


@pytest.mark.parametrize("over", [dict(layers=0), dict(layers=5000), dict(kv_heads=0), dict(kv_heads=2000), dict(qk_dim=0),
                                  dict(qk_dim=257), dict(v_dim=0), dict(v_dim=300), dict(group=16), dict(group=128),
                                  dict(page=16), dict(page=33), dict(page=512), dict(pages=0), dict(pages=-1),
                                  dict(pages=1 << 29), dict(seqs=0), dict(seqs=70000), dict(cap=0), dict(cap=-5),
                                  dict(cap=(1 << 30) + 1), dict(seqs=65536, cap=1 << 30),
                                  dict(layers=4096, kv_heads=1024, pages=1 << 28)])
def test_shapes(over):
    assert new(**over) == EINVAL
    assert nh.load_library().nh_last_error()


def test_null_handles():
    lib = nh.load_library()
    one = np.zeros(4, np.int32)
    p = one.ctypes.data_as(C.c_void_p)
    assert lib.nh_kv4_new(*GOOD.values(), None) == EINVAL
    assert lib.nh_kv4_free(None) == 0
    assert lib.nh_kv4_bytes(None) == EINVAL
    assert lib.nh_kv4_free_pages(None) == EINVAL
    assert lib.nh_kv4_rows(None) == EINVAL
    assert lib.nh_kv4_seq_new(None) == EINVAL
    assert lib.nh_kv4_seq_len(None, 0) == EINVAL
    assert lib.nh_kv4_seq_free(None, 0) == EINVAL
    assert lib.nh_kv4_seq_truncate(None, 0, 0) == EINVAL
    assert lib.nh_kv4_seq_fork(None, 0, 1, p) == EINVAL
    assert lib.nh_kv4_seq_copy(None, 0, None) == EINVAL
    assert lib.nh_kv4_seq_compact(None, p, 1, p, p, None) == EINVAL
    assert lib.nh_kv4_extend(None, p, p, 1, None) == EINVAL
    assert lib.nh_kv4_append(None, 0, p, p, 1, 1, 0, None) == EINVAL
    assert lib.nh_kv4_read(None, 0, p, p, p, 1, p, p, 0, None) == EINVAL
    assert lib.nh_kv4_attend_ws_bytes(None, 2, 0, 0) == EINVAL
    assert lib.nh_kv4_attend(None, 0, p, 1, 1, 1.0, 0, 0, p, 1, None, 0, None, 0, None) == EINVAL


def test_before_init():
    if nh._ready:
        pytest.skip("this process has initialised a device")
    lib = nh.load_library()
    assert new() == ESTATE
    assert verify() == ESTATE
    with pytest.raises(nh.NeedleHipError):
        nh.KvCache4(1, 1, 64, 64, pages=4, seqs=1, cap=64) if not torch.cuda.is_available() else nh._check(-5)
    assert b"nh_init" in lib.nh_last_error() or torch.cuda.is_available()


def verify(type=0, ldl=100, probs=True, probs_type=0, ldp=100, temperature=1.0, batch=2, n=3, vocab=100):
    # (every check that can refuse comes before the pointers are used)
    lib = nh.load_library()
    one = np.zeros(4, np.int32)
    p = one.ctypes.data_as(C.c_void_p)
    return lib.nh_verify_drafts(p, type, ldl, p, None, p if probs else None, probs_type, ldp, p, temperature, batch, n, vocab,
                                p, p, None, 0, None)


@pytest.mark.parametrize("over", [dict(type=3), dict(type=-1), dict(ldl=99), dict(probs_type=7), dict(ldp=50),
                                  dict(temperature=-0.1), dict(temperature=float("nan")), dict(temperature=float("inf")),
                                  dict(batch=-1), dict(n=-1), dict(n=1025), dict(vocab=0), dict(vocab=-3),
                                  dict(batch=1 << 24, n=1)])
def test_verify_arguments(over):
    assert verify(**over) == EINVAL


@pytest.mark.parametrize("sizes", [(-1, 1, 10), (1, -1, 10), (1, 2000, 10), (1, 1, 0), (1 << 25, 0, 5)])
def test_verify_workspace_sizes(sizes):
    assert nh.load_library().nh_verify_drafts_ws_bytes(*sizes) == EINVAL


def test_verify_workspace_grows():
    f = nh.load_library().nh_verify_drafts_ws_bytes
    assert f(0, 0, 5) >= 0 and f(4, 3, 1000) >= f(1, 3, 1000) > 0
