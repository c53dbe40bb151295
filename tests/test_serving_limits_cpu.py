"""CPU tests of the serving operators' limits at the C ABI: what is refused before a device is touched."""
import ctypes

import pytest

from dirktensor_b200 import _lib

FAKE = 1 << 20  # 16-byte aligned, never dereferenced: every case is refused, or fails where no device is


def cache(**kw):
    f = dict(k=FAKE, v=2 * FAKE, k_scale=3 * FAKE, v_scale=4 * FAKE, num_pages=8, page_size=64, kv_heads=4, format=0)
    f.update(kw)
    return ctypes.byref(_lib.dt_kv_cache(*(f[n] for n, _ in _lib.dt_kv_cache._fields_)))


@pytest.mark.parametrize("prefix_len", [(1 << 30) + 1, (1 << 31) - 640, (1 << 31) - 1])
def test_a_prefix_past_2_to_the_30_tokens_is_refused(prefix_len):
    """The kernel looks three tiles of 128 keys ahead of its last one with 32-bit positions."""
    L = _lib.lib()
    size = L.dt_prefix_attn_workspace_bytes(1, 1, 4, 4, 0, 64, 0, prefix_len)
    status = L.dt_prefix_attn_fwd(cache(), 5 * FAKE, 512, 512, 0, 6 * FAKE, None, None, 7 * FAKE, prefix_len, None, 0, 0,
                                  None, None, 1, 1, 4, 0.1, 8 * FAKE, size, None)
    assert status == 1 and b"2^30" in L.dt_last_error(), L.dt_last_error()
