"""Arguments that the 8-bit cache refuses, before any device work (no GPU needed:
the last check is nh_init's)."""
import ctypes as C

import numpy as np
import pytest
import torch

import needle_hip as nh

GOOD = dict(layers=2, kv_heads=2, qk_dim=48, v_dim=64, page=64, pages=8, seqs=3, cap=100)
EINVAL, ESTATE = -1, -5


def new(**over):
    lib = nh.load_library()
    h = C.c_void_p()
    a = {**GOOD, **over}
    rc = lib.nh_kv8_new(*[a[k] for k in GOOD], C.byref(h))
    if h.value:
        lib.nh_kv8_free(h)
    return rc


@pytest.mark.parametrize("over", [dict(layers=0), dict(layers=5000), dict(kv_heads=0), dict(kv_heads=2000), dict(qk_dim=0),
                                  dict(qk_dim=257), dict(v_dim=0), dict(v_dim=300), dict(page=32), dict(page=65),
                                  dict(page=512), dict(page=0), dict(page=-64), dict(pages=0), dict(pages=-1),
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
    assert lib.nh_kv8_new(*GOOD.values(), None) == EINVAL
    assert lib.nh_kv8_free(None) == 0
    assert lib.nh_kv8_bytes(None) == EINVAL
    assert lib.nh_kv8_free_pages(None) == EINVAL
    assert lib.nh_kv8_rows(None) == EINVAL
    assert lib.nh_kv8_seq_new(None) == EINVAL
    assert lib.nh_kv8_seq_len(None, 0) == EINVAL
    assert lib.nh_kv8_seq_free(None, 0) == EINVAL
    assert lib.nh_kv8_seq_truncate(None, 0, 0) == EINVAL
    assert lib.nh_kv8_seq_fork(None, 0, 1, p) == EINVAL
    assert lib.nh_kv8_seq_copy(None, 0, None) == EINVAL
    assert lib.nh_kv8_extend(None, p, p, 1, None) == EINVAL
    assert lib.nh_kv8_ask(None, p, p, 1, None) == EINVAL
    assert lib.nh_kv8_append(None, 0, p, p, 1, 1, 0, None, None, None, 0, 0, None, 0, None) == EINVAL
    assert lib.nh_kv8_read(None, 0, p, p, p, 1, p, p, 0, None) == EINVAL
    assert lib.nh_kv8_debug_kernel(None, 0) == EINVAL
    assert lib.nh_kv8_attend_ws_bytes(None, 2, 0, 0) == EINVAL
    assert lib.nh_kv8_attend(None, 0, p, 1, 1, 1.0, 0, 0, p, 1, None, 0, None, 0, None) == EINVAL


def test_before_init():
    if nh._ready:
        pytest.skip("this process has initialised a device")
    assert new() == ESTATE
    with pytest.raises(nh.NeedleHipError):
        nh.KvCache8(1, 1, 64, 64, pages=4, seqs=1, cap=64) if not torch.cuda.is_available() else nh._check(-5)
