"""CPU tests of the serving operators' refusals: the C ABI checks its arguments before it touches
a device, and the Python forms check tensors before they call it."""
import ctypes

import pytest
import torch

import dirktensor_b200 as dt
from dirktensor_b200 import _lib

FAKE = 1 << 20  # 16-byte aligned, never dereferenced: every case fails validation first


def cache(**kw):
    f = dict(k=FAKE, v=FAKE, k_scale=FAKE, v_scale=FAKE, num_pages=8, page_size=64, kv_heads=4, format=0)
    f.update(kw)
    return ctypes.byref(_lib.dt_kv_cache(*(f[n] for n, _ in _lib.dt_kv_cache._fields_)))


def append(c, k=FAKE, kb=4 * 128, kt=4 * 128, v=FAKE, f32=0, table=FAKE, stride=4, n=4, B=1, T=1):
    return _lib.lib().dt_kv_cache_append(c, k, kb, kt, v, kb, kt, f32, table, stride, n, None, None, B, T, None)


@pytest.mark.parametrize("bad, word", [
    (dict(format=2), b"format"), (dict(page_size=48), b"page_size"), (dict(page_size=8), b"page_size"),
    (dict(page_size=512), b"page_size"), (dict(num_pages=0), b"num_pages"), (dict(kv_heads=0), b"kv_heads"),
    (dict(num_pages=1 << 23, page_size=256), b"2^31"), (dict(k=None), b"null"), (dict(v_scale=None), b"null"),
    (dict(v=FAKE + 8), b"aligned"),
])
def test_cache_descriptor_is_checked(bad, word):
    L = _lib.lib()
    calls = [lambda c: append(c),
             lambda c: L.dt_kv_cache_read(c, FAKE, FAKE, 0, FAKE, 4, 4, None, None, 1, 1, None),
             lambda c: L.dt_cache_attn_fwd(c, FAKE, 512, 512, 0, FAKE, None, None, FAKE, 4, 4, FAKE, None, 1, 1, 4, 0.1, FAKE, 1 << 30, None),
             lambda c: L.dt_prefix_attn_fwd(c, FAKE, 512, 512, 0, FAKE, None, None, FAKE, 64, FAKE, 4, 4, FAKE, None, 1,
                                            1, 4, 0.1, FAKE, 1 << 30, None)]
    for call in calls:
        assert call(cache(**bad)) == 1 and word in L.dt_last_error(), L.dt_last_error()
        assert call(None) == 1


def test_append_and_read_refusals():
    L = _lib.lib()
    assert append(cache(), k=None) == 1 and b"k must be" in L.dt_last_error()
    assert append(cache(), v=FAKE + 2) == 1 and b"v must be" in L.dt_last_error()
    assert append(cache(), kt=4 * 128 + 4) == 1 and b"strides" in L.dt_last_error()      # 8 bytes off
    assert append(cache(), kt=4 * 128 + 2, f32=1) == 1 and b"strides" in L.dt_last_error()
    assert append(cache(), table=None) == 1 and b"page_table" in L.dt_last_error()
    assert append(cache(), stride=3) == 1 and b"page_table_stride" in L.dt_last_error()
    assert append(cache(), T=-1) == 1
    assert append(cache(), B=0, table=None, k=None) == 0 and append(cache(), T=0, k=None) == 0  # empty: no-op
    assert L.dt_kv_cache_read(cache(), None, FAKE, 0, FAKE, 4, 4, None, None, 1, 1, None) == 1
    assert L.dt_kv_cache_read(cache(), FAKE, FAKE + 8, 0, FAKE, 4, 4, None, None, 1, 1, None) == 1
    assert L.dt_kv_cache_read(cache(), None, None, 0, None, 4, 4, None, None, 0, 1, None) == 0


def test_attention_refusals():
    L = _lib.lib()

    def attn(c=None, q=FAKE, qb=512, o=FAKE, table=FAKE, n=4, lens=FAKE, B=1, T=1, H=4):
        return L.dt_cache_attn_fwd(c or cache(), q, qb, 512, 0, o, None, None, table, 4, n, lens, None, B, T, H, 0.1, FAKE, 1 << 30, None)

    assert attn(H=6) == 1 and b"multiple of kv_heads" in L.dt_last_error()
    assert attn(q=None) == 1 and attn(q=FAKE + 8) == 1 and attn(qb=510) == 1
    assert attn(o=None) == 1 and b"o must be" in L.dt_last_error()
    assert attn(lens=None) == 1 and b"seq_lens" in L.dt_last_error()
    assert attn(table=None) == 1 and attn(B=-1) == 1
    assert attn(B=1 << 20, T=1 << 10, H=4) == 1 and b"2^31" in L.dt_last_error()
    assert attn(B=0) == 0 and attn(T=0) == 0 and attn(H=0) == 0

    def prefix(pages=FAKE, n=100, ws=FAKE, size=1 << 30):
        return L.dt_prefix_attn_fwd(cache(), FAKE, 512, 512, 0, FAKE, None, None, pages, n, None, 0, 0, None, None, 1, 1,
                                    4, 0.1, ws, size, None)

    assert prefix(n=-1) == 1 and b"prefix_len" in L.dt_last_error()
    assert prefix(pages=None) == 1 and b"prefix_len" in L.dt_last_error()
    assert prefix(ws=None) == 1 and b"workspace" in L.dt_last_error()
    assert prefix(size=64) == 1 and b"workspace" in L.dt_last_error()
    assert prefix(ws=FAKE + 8) == 1 and b"workspace" in L.dt_last_error()
    assert L.dt_prefix_attn_workspace_bytes(0, 1, 4, 4, 0, 64, 4, 100) == 0
    assert L.dt_prefix_attn_workspace_bytes(4, 1, 4, 4, 0, 64, 4, 0) == L.dt_cache_attn_workspace_bytes(4, 1, 4, 4, 0, 64, 4)
    # one part of the prefix and no keys of their own: (m, l, ...) and 128 sums per row
    assert L.dt_prefix_attn_workspace_bytes(4, 1, 4, 4, 0, 64, 0, 100) == 16 * 16 + 16 * 512
    # few items of many keys are shared out, and need room for the parts
    assert L.dt_cache_attn_workspace_bytes(1, 1, 4, 4, 0, 64, 4096) > 0
    assert attn(n=1 << 26) == 1 and b"page_table_stride" in L.dt_last_error()
    st = L.dt_cache_attn_fwd(cache(), FAKE, 512, 512, 0, FAKE, None, None, FAKE, 1 << 26, 1 << 26, FAKE, None, 1, 1, 4, 0.1,
                             FAKE, 1 << 40, None)
    assert st == 1 and b"2^30" in L.dt_last_error()


def test_log_prob_refusals():
    L = _lib.lib()

    def fwd(x=FAKE, ld=100, N=1, V=100, t=FAKE, top=0, lp=FAKE, ids=FAKE):
        return L.dt_token_log_probs(x, 1, ld, N, V, t, 0, top, lp, None, None, ids, FAKE, None)

    assert fwd(x=None) == 1 and fwd(ld=99) == 1 and fwd(x=FAKE + 2) == 1 and fwd(V=0) == 1 and fwd(N=-1) == 1
    assert fwd(top=33) == 1 and b"top" in L.dt_last_error()
    assert fwd(V=10, top=11) == 1 and fwd(top=-1) == 1 and fwd(top=3, ids=None) == 1
    assert fwd(t=None) == 1 and b"targets" in L.dt_last_error()
    assert fwd(N=0, x=None) == 0

    def bwd(x=FAKE, dx=FAKE, ld=100, N=1, t=FAKE, lse=FAKE, ent=FAKE, g=FAKE, h=None):
        return L.dt_token_log_probs_bwd(x, 1, 100, N, 100, t, 0, lse, ent, g, h, dx, ld, None)

    assert bwd(x=None) == 1 and bwd(dx=None) == 1 and bwd(dx=FAKE + 2) == 1 and bwd(ld=99) == 1 and bwd(lse=None) == 1
    assert bwd(t=None) == 1 and b"targets" in L.dt_last_error()
    assert bwd(h=FAKE, ent=None) == 1 and b"entropy" in L.dt_last_error()
    assert bwd(N=0, x=None) == 0


def test_python_forms_refuse_host_tensors_and_wrong_types():
    codes, scales = torch.zeros((2, 1, 16, 128), dtype=torch.int8), torch.zeros((2, 1, 16))
    with pytest.raises(ValueError, match="CUDA"):
        dt.KVCache.from_tensors(codes, codes, scales, scales)
    with pytest.raises(ValueError, match="format"):
        dt.KVCache(4, format="int4")
    with pytest.raises(ValueError, match="CUDA"):
        dt.token_log_probs(torch.zeros((2, 8)), torch.zeros((2,), dtype=torch.int64))
    with pytest.raises(ValueError, match="CUDA"):
        dt.token_log_probs_backward(torch.zeros((2, 8)), None, torch.zeros(2), None, None)


def test_importing_the_package_does_not_need_the_serving_module():
    """The serving names resolve on first use; the rest of the package works without torch."""
    import subprocess
    import sys

    code = "import sys; import dirktensor_b200; assert 'dirktensor_b200.serving' not in sys.modules; " \
           "assert 'torch' not in sys.modules; dirktensor_b200.KVCache; assert 'torch' in sys.modules"
    subprocess.run([sys.executable, "-c", code], check=True)


def test_gradient_that_overlaps_its_logits_is_refused():
    L = _lib.lib()

    def refused(delta, N=4, V=100, ld=100, dld=100, f32=1):
        status = L.dt_token_log_probs_bwd(FAKE, f32, ld, N, V, None, 0, FAKE, FAKE, None, None, FAKE + delta, dld, None)
        return status == 1 and b"overlap" in L.dt_last_error()

    assert refused(4) and refused(-4) and refused(396) and refused(2, f32=0)      # part of a row
    assert refused(400) and refused(-400) and refused(1200)                       # another row's place
    assert refused(0, ld=104) and refused(0, dld=1 << 40) and refused(400, ld=1 << 40)
    assert refused(500, ld=250, N=2) and refused(-500, ld=250)   # rows at 500 and 900 bytes: in 1000..1399; at -100: in 0..399
    assert not refused(404, ld=202, dld=202, V=101)              # halves of the same rows
    assert refused(404, ld=201, dld=201, V=101) and refused(400, ld=201, dld=201, V=101)
    assert not refused(0) and not refused(1600) and not refused(-1600) and not refused(0, N=1, ld=104)
    assert not refused(400, N=1) and refused(396, N=1) and not refused(0, N=0)


def test_cache_arrays_cannot_be_replaced_under_their_addresses():
    for name in ("k", "v", "k_scale", "v_scale"):
        with pytest.raises(AttributeError):
            setattr(dt.KVCache.__new__(dt.KVCache), name, None)
