"""The call that ends a batch of the 8-bit cache on the device: a null handle (no GPU needed)."""
import needle_hip as nh


def test_null_handle():
    assert nh.load_library().nh_kv8_end_batch(None, None) == -1
