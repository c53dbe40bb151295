"""CPU tests of the serving operators' limits at the C ABI: what is refused before a device is touched.  A call that
passes the check in question is refused by a later one, so that none reaches a device, whether or not there is one."""
import ctypes

import pytest

from dirktensor_b200 import _lib

FAKE = 1 << 20  # 16-byte aligned, never dereferenced: every case is refused


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


@pytest.mark.parametrize("prefix_len", [0, 100])
def test_an_output_that_overlaps_its_queries_is_refused(prefix_len):
    """One item's rows would be written while another's queries are still read.  In place is fine."""
    L = _lib.lib()

    def overlaps(delta, B=2, T=3, H=4, qb=None, qt=512, f32=0):
        q = 64 * FAKE
        qb = T * qt if qb is None else qb
        # a prefix, or few items of many keys, need a workspace, and get none
        assert L.dt_prefix_attn_workspace_bytes(B, T, H, 4, f32, 64, 4096, prefix_len) > 0
        status = L.dt_prefix_attn_fwd(cache(), q, qb, qt, f32, q + delta, None, None, 7 * FAKE, prefix_len, 9 * FAKE, 4096, 4096,
                                      10 * FAKE, None, B, T, H, 0.1, None, 0, None)
        assert status == 1 and (b"overlap" in L.dt_last_error()) != (b"workspace" in L.dt_last_error())
        return b"overlap" in L.dt_last_error()

    row = 4 * 128 * 2  # of one token
    assert not overlaps(0) and not overlaps(0, f32=1)                       # in place
    assert overlaps(16) and overlaps(-16) and overlaps(row) and overlaps(-row) and overlaps(5 * row) and overlaps(-5 * row)
    assert not overlaps(6 * row) and not overlaps(-6 * row)                 # before and behind
    assert overlaps(0, qt=1024) and overlaps(0, qb=4 * 512)                 # the same start, other rows
    assert not overlaps(0, B=1, qb=16) and not overlaps(0, T=1, qt=16, qb=512) and not overlaps(0, B=1, T=1, qb=0, qt=0)
    # queries of a fused projection, the output between its rows
    assert not overlaps(row, B=1, T=2, qt=3 * 512) and overlaps(row + 16, B=1, T=2, qt=3 * 512)
    assert overlaps(0, qb=0, qt=0) and overlaps(-16, qb=0, qt=0) and not overlaps(row, qb=0, qt=0)  # one query for all
    assert overlaps(2 * row, B=2, T=2, qb=1 << 20, qt=512) is False and overlaps(2 << 20, B=3, T=2, qb=1 << 20, qt=512)


def test_append_into_a_cache_whose_arrays_overlap_is_refused():
    """K and V of a token would be written to one place at once.  Reading such a cache is fine."""
    L = _lib.lib()
    codes, scales = 8 * 4 * 64 * 128, 8 * 4 * 64 * 4  # bytes of cache()'s arrays

    def refused(**kw):
        status = L.dt_kv_cache_append(cache(**kw), 5 * FAKE, 512, 512, 6 * FAKE, 512, 512, 0, 7 * FAKE, 4, 4, None, None, 1 << 20,
                                      1 << 20, None)
        assert status == 1 and (b"overlap" in L.dt_last_error()) != (b"too large" in L.dt_last_error())
        return b"overlap" in L.dt_last_error()

    assert not refused()
    assert refused(v=FAKE) and refused(v_scale=3 * FAKE) and refused(v=FAKE + codes - 16) and refused(k=2 * FAKE + codes - 16)
    assert not refused(v=FAKE + codes) and not refused(v_scale=3 * FAKE + scales) and refused(v_scale=3 * FAKE + scales - 16)
    assert refused(k_scale=FAKE + 1024) and refused(v_scale=2 * FAKE - 16)


def test_a_prefix_in_many_parts_before_a_very_wide_page_table_is_refused():
    """Few query rows over a long prefix: what every sequence has of its own is counted in 32-bit tiles over the batch."""
    L = _lib.lib()

    def refused(B, pages):
        status = L.dt_prefix_attn_fwd(cache(page_size=256, kv_heads=1), 5 * FAKE, 128, 128, 0, 1 << 40, None, None, 7 * FAKE,
                                      1 << 20, 9 * FAKE, pages, pages, 10 * FAKE, None, B, 1, 1, 0.1, None, 0, None)
        assert status == 1 and (b"2^36" in L.dt_last_error()) != (b"workspace" in L.dt_last_error()), L.dt_last_error()
        return b"2^36" in L.dt_last_error()

    assert refused(64, 1 << 22) and refused(2048, 1 << 18)
    assert not refused(63, 1 << 22) and not refused(64, (1 << 22) - 1)
    assert not refused(10000, 4) and not refused(1 << 20, 4)  # no limit on the batch itself


def test_overlapping_gradients_are_refused_and_others_pass_that_check():
    """As for the outputs above: rows of logits and of their gradient, with a device or without (N * V ends it)."""
    L = _lib.lib()

    def refused(delta, N=1 << 20, V=1 << 30, ld=1 << 30, dld=1 << 30, elem=4):
        x = 1 << 56
        status = L.dt_token_log_probs_bwd(x, int(elem == 4), ld, N, V, None, 0, 5 * FAKE, 6 * FAKE, None, None, x + delta, dld, None)
        assert status == 1 and (b"overlap" in L.dt_last_error()) != (b"too large" in L.dt_last_error())
        return b"overlap" in L.dt_last_error()

    row = 4 << 30
    assert refused(4) and refused(-4) and refused(row - 4) and refused(row) and refused(-row) and refused(3 * row)
    assert refused(0, ld=(1 << 30) + 4) and refused(0, dld=1 << 40) and refused(2, elem=2)
    assert not refused(0) and not refused(row << 20) and not refused(-(row << 20))
    assert not refused(row, ld=2 << 30, dld=2 << 30) and refused(row - 4, ld=2 << 30, dld=2 << 30)
