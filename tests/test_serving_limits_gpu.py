"""GPU tests of what the serving operators take and refuse at the edges of their arguments."""
import math

import pytest
import torch

from serving_ref import D
from test_serving_gpu import attention_case, ints

pytestmark = pytest.mark.gpu

SCALE = 1.0 / math.sqrt(D)
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def dt(cuda):
    import dirktensor_b200

    return dirktensor_b200


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_outputs_in_place_and_outputs_that_overlap(dt, cuda, dtype):
    B, T = 30, 5
    c, pages, table, lens, q = attention_case(dt, cuda, 61, "int8", dtype, B, T, 2, 2, 16, [20 + i for i in range(B)], 200)
    both = torch.empty((B + 1, T, 4, D), dtype=dtype, device=cuda)
    for call in (lambda x, **kw: dt.cache_attention_forward(x, c, table, lens, SCALE, **kw),
                 lambda x, **kw: dt.prefix_attention_forward(x, c, pages, 200, table, lens, SCALE, **kw),
                 lambda x, **kw: dt.prefix_attention_forward(x, c, pages, 200, None, None, SCALE, **kw)):
        want = call(q)
        x = q.clone()
        assert call(x, out=x) is x and torch.equal(x, want)
        both[:B] = q
        with pytest.raises(dt.DTError, match="overlap"):
            call(both[:B], out=both[1:])
        assert torch.equal(both[:B], q)
        x = torch.zeros((B, T, 3, 4, D), dtype=dtype, device=cuda)
        x[:, :, 1] = q
        with pytest.raises(dt.DTError, match="overlap"):
            call(x[:, :, 1], out=x.view(-1)[:q.numel()].view(q.shape))
        assert torch.equal(call(x[:, :, 1]), want)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B, T", [(1, 1), (3, 1), (1, 4)])
def test_strides_of_dimensions_of_one_do_not_matter(dt, cuda, dtype, B, T):
    """Their strides lead nowhere: every row starts on a 16-byte boundary whatever they are."""
    c, pages, table, lens, q = attention_case(dt, cuda, 62, "int8", dtype, B, T, 2, 1, 16, [20] * B, 40)
    odd = q.as_strided(q.shape, (q.stride(0) if B > 1 else 7, q.stride(1) if T > 1 else 3, D, 1))
    assert torch.equal(dt.cache_attention_forward(odd, c, table, lens, SCALE), dt.cache_attention_forward(q, c, table, lens, SCALE))
    assert torch.equal(dt.prefix_attention_forward(odd, c, pages, 40, table, lens, SCALE),
                       dt.prefix_attention_forward(q, c, pages, 40, table, lens, SCALE))
    c.append(odd, odd, table)
    k, v = c.k.clone(), c.v_scale.clone()
    c.append(q, q, table)
    assert torch.equal(c.k, k) and torch.equal(c.v_scale, v)


def test_append_past_the_last_position_takes_no_slot(dt, cuda):
    """Positions end at 2^31 - 1: tokens past it are skipped, and give way to those that are written."""
    page, last = 256, (1 << 31) // 256 - 1
    c = dt.KVCache(3, page, 1)
    table = torch.full((2, last + 3), -1, dtype=torch.int32, device=cuda)
    table[0, 0], table[1, last], table[1, last + 1] = 0, 1, 0
    k = torch.randn((2, 20, 1, D), generator=torch.Generator(device=cuda).manual_seed(1), device=cuda)
    start = ints(cuda, 0, (1 << 31) - 10)
    c.append(k, k, table, start)
    back, _ = c.read(table, start, 20, dtype=F32)
    dt.check_device_error()
    assert bool((c.k_scale[0, 0, :20] > 0).all()) and bool((c.k_scale[1, 0, 246:] > 0).all())
    assert int((c.k_scale > 0).sum()) == 30
    assert bool((back[0] != 0).any(-1).all()) and bool((back[1, :10] != 0).any(-1).all()) and bool((back[1, 10:] == 0).all())


def test_a_large_batch_behind_a_prefix(dt, cuda):
    """More than 8192 sequences: what some of them get is what they get alone, within the bounds."""
    import serving_ref as ref

    B, some = 9001, [0, 1, 127, 128, 255, 256, 4500, 8191, 8192, 8999, 9000]
    c, pages, table, lens, q = attention_case(dt, cuda, 63, "int8", BF16, B, 1, 1, 1, 16, [i % 31 for i in range(B)], 300)
    got = dt.prefix_attention_forward(q, c, pages, 300, table, lens, SCALE, return_stats=True)
    dt.check_device_error()
    want = ref.attention(q[some], c, table[some], lens[some], SCALE, prefix_pages=pages, prefix_len=300)
    ref.check_attention([x[some] for x in got], want)


def test_a_cache_that_shares_its_arrays_is_read_and_not_written(dt, cuda):
    c, _, table, lens, q = attention_case(dt, cuda, 64, "int8", BF16, 2, 1, 2, 1, 16, [20, 7])
    same = dt.KVCache.from_tensors(c.k, c.k, c.k_scale, c.k_scale)
    k, v = same.read(table, None, 20)
    assert torch.equal(k, v)
    other = dt.KVCache.from_tensors(c.k, c.k.clone(), c.k_scale, c.k_scale.clone())
    assert torch.equal(dt.cache_attention_forward(q, same, table, lens, SCALE), dt.cache_attention_forward(q, other, table, lens, SCALE))
    before = c.k.clone()
    with pytest.raises(dt.DTError, match="overlap"):
        same.append(q, q, table)
    assert torch.equal(c.k, before)
