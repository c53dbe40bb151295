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


def winners(table, start, lens, page, T):
    """Slot (page * page size + offset) and token number b * T + t of each token that stays, in 64-bit indexes."""
    B = table.shape[0]
    t = torch.arange(T, device=table.device)
    pos = start.long()[:, None] + t
    at = torch.gather(table.long(), 1, (pos // page).clamp(max=table.shape[1] - 1))
    live = (t < lens.long()[:, None]) & (pos // page < table.shape[1]) & (at >= 0)
    slot = (at * page + pos % page)[live]
    token = (torch.arange(B, device=table.device)[:, None] * T + t)[live]
    best = torch.full((int(slot.max()) + 1,), -1, dtype=torch.int64, device=table.device)
    best.scatter_reduce_(0, slot, token, "amax")
    used = best >= 0
    return torch.nonzero(used)[:, 0], best[used]


@pytest.mark.parametrize("B, T, page, pool", [(9000, 1, 16, 700), (9000, 1, 64, 20000), (300, 600, 16, 4000), (2, 150000, 16, 9000),
                                              (1, 140000, 16, 9000), (5, 70001, 64, 3000)])
def test_appends_of_many_pages_keep_the_last_token_of_a_slot(dt, cuda, B, T, page, pool):
    """More page entries than one launch looks through: pages that are named twice, near and far apart, short and long lengths."""
    g = torch.Generator(device=cuda).manual_seed(B + T)
    heads, per = 1, -(-(T + 40) // page)
    c = dt.KVCache(pool, page, heads)
    table = torch.randint(-1, pool, (B, per), generator=g, device=cuda).to(torch.int32)
    start = torch.randint(0, 40, (B,), generator=g, device=cuda).to(torch.int32)
    lens = torch.randint(0, T + 3, (B,), generator=g, device=cuda).to(torch.int32)
    lens[-1] = T
    k = torch.randn((B, T, heads, D), generator=g, device=cuda).to(BF16)
    c.append(k, k.flip(1), table, start, lens)
    dt.check_device_error()
    slot, token = winners(table, start, lens.clamp(max=T), page, T)
    for x, scales, codes in ((k, c.k_scale, c.k), (k.flip(1), c.v_scale, c.v)):
        y = x.reshape(-1, D)[token].float()
        amax = y.abs().amax(-1)
        assert torch.equal(scales.view(-1)[slot], amax / torch.full_like(amax, 127.0))
        assert torch.equal(codes.view(-1, D)[slot], (y * 127 / amax[:, None]).round().to(torch.int8))
        assert int((scales > 0).sum()) == len(slot)


def test_the_time_of_an_append_grows_with_its_tokens(dt, cuda):
    """4 million tokens on pages of their own: the search for tokens that share a slot took 163 ms, by the square of the
    tokens; in stretches it is some 3 ms."""
    T, page = 1 << 22, 16
    c = dt.KVCache(T // page, page, 1)
    table = torch.randperm(T // page, device=cuda).to(torch.int32)[None]
    k = torch.ones((1, 1, 1, D), dtype=BF16, device=cuda).expand(1, T, 1, D)
    times = []
    for _ in range(4):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        c.append(k, k, table)
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b))
    assert bool((c.k_scale > 0).all()) and min(times) < 60.0, times


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_long_append_in_every_type(dt, cuda, fmt, dtype):
    """Tokens of a sequence that a later launch writes, on pages that earlier ones name too, and past the last position."""
    from serving_ref import TOP

    g = torch.Generator(device=cuda).manual_seed(7)
    T, page, heads, pool = 100003, 16, 2, 5000
    c = dt.KVCache(pool, page, heads, fmt)
    table = torch.randint(0, pool, (1, 6300), generator=g, device=cuda).to(torch.int32)
    start, lens = ints(cuda, 9), ints(cuda, 99990)
    k, v = (torch.randn((1, T, heads, D), generator=g, device=cuda).to(dtype) for _ in range(2))
    c.append(k, v, table, start, lens)
    dt.check_device_error()
    slot, token = winners(table, start, lens, page, T)
    for x, scales, codes in ((k, c.k_scale, c.k), (v, c.v_scale, c.v)):
        y = x[0, token].float()
        amax = y.abs().amax(-1)
        assert torch.equal(scales[slot // page, :, slot % page], amax / torch.full_like(amax, TOP[fmt]))
        want = y * TOP[fmt] / amax[..., None]
        got = codes.view(torch.int8)[slot // page, :, slot % page]
        assert torch.equal(got, (want.round() if fmt == "int8" else want).to(codes.dtype).view(torch.int8))
    before = c.k.clone(), c.k_scale.clone()
    c.append(k, v, torch.zeros((1, (1 << 27) + 10), dtype=torch.int32, device=cuda), ints(cuda, (1 << 31) - 40000), ints(cuda, 39990))
    used = torch.zeros(pool, dtype=torch.bool, device=cuda)
    used[0] = True
    assert torch.equal(before[0].view(torch.int8)[~used], c.k.view(torch.int8)[~used])
    where = ((1 << 31) - 40000 + torch.arange(39990, device=cuda)) % page
    for off in range(page):
        last = int(torch.nonzero(where == off)[-1])
        amax = k[0, last].float().abs().amax(-1)
        assert torch.equal(c.k_scale[0, :, off], amax / torch.full_like(amax, TOP[fmt]))
    c.append(k, v, torch.zeros((1, (1 << 27) + 10), dtype=torch.int32, device=cuda), ints(cuda, (1 << 31) - 5), None)
    first = k[0, :5].float().abs().amax(-1)
    assert torch.equal(c.k_scale[0, :, 11:], (first / torch.full_like(first, TOP[fmt])).T)
