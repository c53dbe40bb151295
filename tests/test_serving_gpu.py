"""GPU tests of the serving operators against their plain 64-bit forms."""
import math

import pytest
import torch

import serving_ref as ref
from serving_ref import D, EPS32, HALF, TOP

pytestmark = pytest.mark.gpu

SCALE = 1.0 / math.sqrt(D)
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def dt(cuda):
    import dirktensor_b200

    return dirktensor_b200


def gen(cuda, seed):
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    return g


def ints(cuda, *v):
    return torch.tensor(v, dtype=torch.int32, device=cuda)


def new_rows(g, shape, dtype, cuda):
    return (torch.randn(shape, generator=g, device=cuda) * torch.exp(torch.randn(shape[:-1] + (1,), generator=g, device=cuda))).to(dtype)


def nearest_code_error(fmt, x, got, scale):
    """How far a stored value is from x beyond what rounding to the nearest code allows (<= 0: right)."""
    amax = x.abs().amax(-1, keepdim=True)
    y = x * TOP[fmt] / amax
    code = got / scale
    # the quotient is off by two roundings of fp32; then half a step of the code
    half = torch.full_like(y, 0.5) if fmt == "int8" else torch.maximum(y.abs() * 2.0 ** -4, torch.full_like(y, 2.0 ** -10))
    return float(((code - y).abs() - half - 2 * EPS32 * TOP[fmt] * 1.01).max())


# ---------------------------------------------------------------- the cache

@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B, T, heads, page", [(1, 1, 1, 16), (3, 1, 16, 64), (2, 37, 3, 32), (5, 129, 8, 16), (2, 700, 16, 256)])
def test_append_and_read_back(dt, cuda, fmt, dtype, B, T, heads, page):
    g = gen(cuda, B * 1000 + T)
    per_row = -(-(T + 21) // page)
    c = dt.KVCache(B * per_row + 3, page, heads, fmt)
    for t in (c.k_scale, c.v_scale):
        t.fill_(-7.0)  # what no call writes stays as it was
    table = ref.pages_of(g, c.num_pages, B, per_row, cuda)
    start = torch.arange(B, device=cuda, dtype=torch.int32) * 5
    k, v = new_rows(g, (B, T, heads, D), dtype, cuda), new_rows(g, (B, T, heads, D), dtype, cuda)
    c.append(k, v, table, start)
    k32, v32 = c.read(table, start, T, dtype=F32)
    kb, vb = c.read(table, start, T, dtype=BF16)
    dt.check_device_error()
    pos = start.long()[:, None] + torch.arange(T, device=cuda)
    at = torch.gather(table.long(), 1, pos // page)
    for x, codes, scales, back, back16 in ((k, c.k, c.k_scale, k32, kb), (v, c.v, c.v_scale, v32, vb)):
        sc = scales[at, :, pos % page].double()
        amax = x.double().abs().amax(-1)
        assert float(((sc - amax / TOP[fmt]).abs() / (amax / TOP[fmt])).max()) <= EPS32
        stored = codes.view(torch.int8)[at, :, pos % page].view(codes.dtype).float()
        assert nearest_code_error(fmt, x.double(), stored.double() * sc[..., None], sc[..., None]) <= 0
        assert torch.equal(back, stored * scales[at, :, pos % page][..., None])   # code * scale, one rounding
        assert torch.equal(back16, back.to(BF16))
        touched = torch.zeros_like(scales, dtype=torch.bool)
        touched[at, :, pos % page] = True
        assert bool((scales[~touched] == -7.0).all()) and int(codes.view(torch.int8)[~touched].abs().max()) == 0


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_codes_of_bf16_rows_are_the_plain_forms_bit_for_bit(dt, cuda, fmt):
    """x * Q is exact for bf16 x, so every tie is a tie, and goes to the even code."""
    g = gen(cuda, 5)
    x = torch.randn((1, 64, 4, D), generator=g, device=cuda).to(BF16)
    x[..., 0] = 4.0  # an amax of few bits makes ties of many values
    x[..., 1:64] = (torch.randint(-512, 512, (1, 64, 4, 63), generator=g, device=cuda).float() / 128).to(BF16)
    c = dt.KVCache(4, 16, 4, fmt)
    table = ints(cuda, 2, 0, 3, 1)[None]
    c.append(x, x, table)
    y = x.float() * TOP[fmt] / x.float().abs().amax(-1, keepdim=True)
    want = (y.round() if fmt == "int8" else y).to(c.k.dtype).view(torch.int8)
    got = c.k.view(torch.int8)[table[0].long()].permute(0, 2, 1, 3).reshape(64, 4, D)
    assert torch.equal(got, want[0])


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_of_zeros_tiny_huge_and_not_finite_values(dt, cuda, fmt, dtype):
    x = torch.zeros((1, 8, 1, D), device=cuda)
    x[0, 1] = 2.0 ** -101
    x[0, 2, 0, :] = torch.linspace(-1, 1, D, device=cuda) * 2.0 ** -99
    x[0, 3, 0, :] = torch.linspace(-1, 1, D, device=cuda) * 3e38
    x[0, 4, 0, 7] = math.inf
    x[0, 5, 0, 100] = math.nan
    x[0, 6, 0, 100] = -math.inf
    x[0, 7, 0, 3] = 1.0
    x = x.to(dtype)
    c = dt.KVCache(1, 16, 1, fmt)
    table = ints(cuda, 0)[None]
    c.append(x, x, table)
    back = c.read(table, None, 9, lens=ints(cuda, 9), dtype=F32)[0][0, :, 0]
    assert bool((back[:2] == 0).all()) and torch.equal(c.k_scale[0, 0, :2], torch.zeros(2, device=cuda))
    for r in (2, 3, 7):
        step = float(x[0, r].float().abs().max()) * (0.5 / 127 if fmt == "int8" else 2.0 ** -4)
        assert torch.isfinite(back[r]).all() and float((back[r] - x[0, r, 0].float()).abs().max()) <= step * 1.0001
    for r in (4, 5, 6):
        assert torch.isnan(back[r]).all()
    assert bool((back[8] == 0).all())


def test_append_skips_padding_and_tokens_without_a_page(dt, cuda):
    g = gen(cuda, 9)
    B, T, heads = 4, 40, 2
    c = dt.KVCache(6, 16, heads, "int8")
    c.k_scale.fill_(-7.0)
    table = ints(cuda, 0, 1, 2, -1, 6, 3, 4, 1 << 30, 5, -5, 5, 5).view(4, 3)
    table[3] = ints(cuda, 5, -5, 99)
    start, lens = ints(cuda, 0, 0, -3, 30), ints(cuda, 40, 40, 40, 5)
    k = new_rows(g, (B, T, heads, D), F32, cuda)
    c.append(k, k, table, start, lens)
    back = c.read(table, start, T, lens, dtype=F32)[0]
    dt.check_device_error()
    for b in range(B):
        for t in range(T):
            pos = int(start[b]) + t
            page = int(table[b, pos // 16]) if 0 <= pos < 48 else -1
            live = t < int(lens[b]) and 0 <= page < 6
            assert bool((back[b, t] != 0).any()) == live, (b, t)
    written = sum(1 for b in range(B) for t in range(T) if bool((back[b, t] != 0).any()))
    assert int((c.k_scale != -7.0).sum()) == heads * written
    # lengths of zero, negative and past T; a position that passes 2^31
    before = c.k.clone(), c.k_scale.clone()
    c.append(k, k, table, start, ints(cuda, 0, -1, 0, -2147483648))
    c.append(k, k, table, ints(cuda, 2147483647, 2147483600, 48, -40), ints(cuda, 1 << 30, 40, 40, 40))
    assert torch.equal(before[0], c.k) and torch.equal(before[1], c.k_scale)


@pytest.mark.parametrize("B, T", [(7, 1), (3, 50), (2, 900)])
def test_two_tokens_of_a_call_on_one_slot_keep_the_last(dt, cuda, B, T):
    """The page table names a page twice: the token of the highest (sequence, position) stays, whole."""
    g = gen(cuda, 10 * B + T)
    heads, page = 3, 16
    per_row = -(-(T + 8) // page)
    c = dt.KVCache(B * per_row, page, heads, "int8")
    table = ref.pages_of(g, c.num_pages, B, per_row, cuda)
    table[-1] = table[0]                        # the last sequence takes the first one's pages
    if per_row > 2:
        table[1, 2] = table[1, 0]               # and one sequence takes a page of its own twice
    start = torch.randint(0, 8, (B,), generator=g, device=cuda).to(torch.int32)
    if T == 1:
        table[3], start[3], start[0], start[-1] = table[0], 5, 5, 5
    k, v = new_rows(g, (B, T, heads, D), BF16, cuda), new_rows(g, (B, T, heads, D), BF16, cuda)
    slots = {}
    for b in range(B):
        for t in range(T):
            pos = int(start[b]) + t
            slots[(int(table[b, pos // page]), pos % page)] = (b, t)
    for _ in range(3):
        c.append(k, v, table, start)
    order = list(slots.items())
    who = torch.tensor([bt for _, bt in order], device=cuda)
    where = torch.tensor([s for s, _ in order], device=cuda)
    for x, codes, scales in ((k, c.k, c.k_scale), (v, c.v, c.v_scale)):
        y = x[who[:, 0], who[:, 1]].float()
        amax = y.abs().amax(-1)
        # (a tensor divided by a number is multiplied by its reciprocal, which rounds twice)
        assert torch.equal(scales[where[:, 0], :, where[:, 1]], amax / torch.full_like(amax, 127.0))
        assert torch.equal(codes[where[:, 0], :, where[:, 1]], (y * 127 / amax[..., None]).round().to(torch.int8))


def test_append_reads_strided_rows_and_slices_of_a_fused_projection(dt, cuda):
    g = gen(cuda, 3)
    B, T, heads = 2, 9, 4
    fused = torch.randn((B, T, 3, heads, D), generator=g, device=cuda).to(BF16)
    c, c2 = dt.KVCache(4, 16, heads, "e4m3"), dt.KVCache(4, 16, heads, "e4m3")
    big = ints(cuda, 3, 9, 9, 1, 8, 8).view(2, 3)
    c.append(fused[:, :, 1], fused[:, :, 2], big[:, :1])
    c2.append(fused[:, :, 1].contiguous(), fused[:, :, 2].contiguous(), big[:, :1].contiguous())
    assert torch.equal(c.k.view(torch.int8), c2.k.view(torch.int8)) and torch.equal(c.v_scale, c2.v_scale)
    with pytest.raises(ValueError, match="16-byte"):
        c.append(fused.view(B, T, -1)[..., 4:4 + heads * D].view(B, T, heads, D), fused[:, :, 2], big[:, :1])
    with pytest.raises(ValueError, match="heads"):
        c.append(fused[:, :, 1, :2], fused[:, :, 2, :2], big)


# ------------------------------------------------------- attention over it

CASES = [
    # B, T, heads, group, page, longest, ragged lengths of a batch
    (1, 1, 1, 1, 16, [1]),
    (1, 1, 16, 1, 64, [513]),
    (9, 1, 2, 1, 16, [0, 1, 15, 16, 17, 63, 64, 65, 130]),
    (4, 1, 4, 4, 32, [31, 32, 33, 257]),
    (3, 3, 2, 8, 64, [3, 66, 200]),
    (2, 9, 3, 1, 128, [9, 150]),
    (3, 20, 1, 3, 16, [5, 20, 77]),
    (2, 1, 1, 20, 64, [300, 1025]),
    (1, 1, 2, 1, 256, [5000]),
]


def attention_case(dt, cuda, seed, fmt, dtype, B, T, heads, group, page, lens, prefix=0):
    g = gen(cuda, seed)
    per_row = max(1, -(-max(lens) // page))
    shared = -(-prefix // page)
    c = dt.KVCache.from_tensors(*ref.make_cache(g, fmt, B * per_row + shared + 2, heads, page, cuda))
    order = torch.randperm(c.num_pages, generator=g, device=cuda).to(torch.int32)
    table = order[shared:shared + B * per_row].view(B, per_row).contiguous()
    q = (torch.randn((B, T, heads * group, D), generator=g, device=cuda) * 2).to(dtype)
    return c, order[:shared].contiguous(), table, ints(cuda, *lens), q


def poison(c, table, seq_lens, prefix_pages=None, prefix_len=0):
    """NaN scales and codes wherever no key of any sequence lies: what is masked must not reach an output."""
    seen = torch.zeros(c.k_scale.shape, dtype=torch.bool, device=c.device)
    spans = [(table[b], min(int(seq_lens[b]), table.shape[1] * c.page_size)) for b in range(len(seq_lens))] if table is not None else []
    if prefix_len:
        spans.append((prefix_pages, prefix_len))
    for pages, n in spans:
        for j in range(n):
            p = int(pages[j // c.page_size])
            if 0 <= p < c.num_pages:
                seen[p, :, j % c.page_size] = True
    for t in (c.k_scale, c.v_scale):
        t[~seen] = math.nan
    for t in (c.k, c.v):
        t.view(torch.int8)[~seen] = 0x7f  # e4m3's NaN


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "b%d_t%d_h%d_g%d_p%d" % c[:5])
def test_cache_attention(dt, cuda, fmt, dtype, case):
    B, T, heads, group, page, lens = case
    c, _, table, seq_lens, q = attention_case(dt, cuda, 1, fmt, dtype, B, T, heads, group, page, lens)
    poison(c, table, seq_lens)
    got = dt.cache_attention_forward(q, c, table, seq_lens, SCALE, return_stats=True)
    dt.check_device_error()
    ref.check_attention(got, ref.attention(q, c, table, seq_lens, SCALE))
    assert torch.equal(dt.cache_attention_forward(q, c, table, seq_lens, SCALE), got.output)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_cache_attention_ragged_queries_and_bad_pages(dt, cuda, fmt, dtype):
    """q_lens of zero, all and more; lengths negative and past the table; pages outside the pool are not seen."""
    B, T = 6, 5
    c, _, table, _, q = attention_case(dt, cuda, 2, fmt, dtype, B, T, 2, 2, 16, [80] * B)
    seq_lens, q_lens = ints(cuda, 3, 60, -4, 200, 80, 33), ints(cuda, 3, 0, 5, 9, -1, 2)
    table[1, 1], table[3, 2], table[5, 0], table[5, 1] = -1, c.num_pages, 1 << 30, -(1 << 31)
    poison(c, table, seq_lens)
    got = dt.cache_attention_forward(q, c, table, seq_lens, SCALE, q_lens=q_lens, return_stats=True)
    dt.check_device_error()
    want = ref.attention(q, c, table, seq_lens.clamp_min(0), SCALE, q_lens=q_lens.clamp_min(0))
    ref.check_attention(got, want)
    assert bool((got.output[1] == 0).all()) and bool((got.softmax_l[4] == 0).all())


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_cache_attention_scales_far_apart_and_zero(dt, cuda, fmt):
    """Scales over many orders of magnitude, rows of zeros, and a sharply peaked softmax."""
    for dtype in (BF16, F32):
        c, _, table, lens, q = attention_case(dt, cuda, 3, fmt, dtype, 3, 1, 2, 1, 32, [200, 64, 7])
        g = gen(cuda, 33)
        c.v_scale.mul_(torch.exp2(torch.randint(-30, 30, c.v_scale.shape, generator=g, device=cuda).float()))
        c.k_scale.mul_(torch.exp2(torch.randint(-6, 3, c.k_scale.shape, generator=g, device=cuda).float()))
        c.k_scale[:, :, 3] = 0.0
        c.v_scale[:, :, 5] = 0.0
        got = dt.cache_attention_forward(q, c, table, lens, SCALE, return_stats=True)
        ref.check_attention(got, ref.attention(q, c, table, lens, SCALE))
        # queries far from 1, small and large
        for f in (2.0 ** -40, 2.0 ** 12):
            y = (q.float() * f).to(dtype)
            got = dt.cache_attention_forward(y, c, table, lens, SCALE / f, return_stats=True)
            ref.check_attention(got, ref.attention(y, c, table, lens, SCALE / f))
        # a query of zeros: an even average
        z = torch.zeros_like(q)
        got = dt.cache_attention_forward(z, c, table, lens, SCALE, return_stats=True)
        ref.check_attention(got, ref.attention(z, c, table, lens, SCALE))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_key_that_is_not_finite_reaches_only_the_queries_that_see_it(dt, cuda, dtype):
    c, _, table, lens, q = attention_case(dt, cuda, 4, "int8", dtype, 2, 3, 2, 1, 16, [40, 40])
    want = dt.cache_attention_forward(q, c, table, lens, SCALE)
    c.k_scale[int(table[0, 2]), 0, 39 - 32] = math.nan  # the last key of sequence 0, head 0
    got = dt.cache_attention_forward(q, c, table, lens, SCALE)
    assert torch.isnan(got[0, 2, 0]).all()
    hit = torch.zeros(q.shape[:3], dtype=torch.bool, device=cuda)
    hit[0, 2, 0] = True
    assert torch.equal(got[~hit], want[~hit])
    c.k_scale[int(table[0, 2]), 0, 39 - 32] = 1.0
    c.v_scale[int(table[0, 2]), 0, 39 - 32] = math.nan
    assert torch.isnan(dt.cache_attention_forward(q, c, table, lens, SCALE)[0, 2, 0]).all()
    q = q.clone()
    q[1, 1, 1, 9] = math.nan
    got = dt.cache_attention_forward(q, c, table, lens, SCALE)
    assert torch.isnan(got[1, 1, 1]).all() and torch.equal(got[1, [0, 2]], want[1, [0, 2]])


def test_cache_attention_long_sequence_is_split_and_joined(dt, cuda):
    for fmt, dtype in (("int8", BF16), ("e4m3", F32)):
        c, _, table, lens, q = attention_case(dt, cuda, 6, fmt, dtype, 1, 1, 1, 2, 64, [40001])
        got = dt.cache_attention_forward(q, c, table, lens, SCALE, return_stats=True)
        ref.check_attention(got, ref.attention(q, c, table, lens, SCALE))


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("group, T", [(1, 1), (8, 1), (4, 5)])
def test_few_long_sequences_are_shared_out_over_the_gpu(dt, cuda, fmt, dtype, group, T):
    """Even shares of all tiles, whatever the lengths: none, one key, one tile, many, and padding queries."""
    for lens, q_lens in (([9001], None), ([0], None), ([T], None), ([0, 8200, 33, 1000], [T, T, 0, T])):
        B = len(lens)
        c, _, _, seq_lens, q = attention_case(dt, cuda, 41, fmt, dtype, B, T, 1, group, 64, lens)
        table = torch.full((B, 160), -1, dtype=torch.int32, device=cuda)
        table[:, :-(-max(lens) // 64)] = torch.arange(B * -(-max(lens) // 64), device=cuda, dtype=torch.int32).view(B, -1)
        ql = None if q_lens is None else ints(cuda, *q_lens)
        poison(c, table, seq_lens)
        got = dt.cache_attention_forward(q, c, table, seq_lens, SCALE, q_lens=ql, return_stats=True)
        dt.check_device_error()
        ref.check_attention(got, ref.attention(q, c, table, seq_lens, SCALE, q_lens=ql))


def test_more_items_than_fit_take_the_longest_sequences_first(dt, cuda):
    """40 x 16 items, a wide page table, equal and zero lengths among the sequences."""
    B = 40
    lens = [0, 1, 70, 70, 70, 33, 0, 140] * 5
    c, _, _, seq_lens, q = attention_case(dt, cuda, 42, "int8", BF16, B, 1, 16, 1, 64, lens)
    table = torch.full((B, 40), 1 << 30, dtype=torch.int32, device=cuda)
    table[:, :3] = torch.randperm(c.num_pages, device=cuda)[: 3 * B].view(B, 3).to(torch.int32)
    poison(c, table, seq_lens)
    got = dt.cache_attention_forward(q, c, table, seq_lens, SCALE, return_stats=True)
    ref.check_attention(got, ref.attention(q, c, table, seq_lens, SCALE))


def test_an_empty_page_table_and_outputs_in_the_queries_own_memory(dt, cuda):
    c, _, table, lens, q = attention_case(dt, cuda, 43, "int8", BF16, 2, 3, 2, 2, 16, [20, 33])
    got = dt.cache_attention_forward(q, c, table[:, :0], lens, SCALE, return_stats=True)
    assert all(bool((x == 0).all()) for x in got)
    want = dt.cache_attention_forward(q, c, table, lens, SCALE)
    q2 = q.clone()
    assert torch.equal(dt.cache_attention_forward(q2, c, table, lens, SCALE, out=q2), want)
    before = c.k.clone()
    kv = torch.ones((2, 1, 2, D), dtype=BF16, device=cuda)
    c.append(kv, kv, table[:, :0])
    assert torch.equal(c.k, before)
    assert bool((c.read(table[:, :0], None, 5)[0] == 0).all())
    assert dt.cache_attention_forward(q[:0], c, table[:0], lens[:0], SCALE).shape == (0, 3, 4, D)
    assert dt.cache_attention_forward(q[:, :0], c, table, lens, SCALE).shape == (2, 0, 4, D)


def test_strided_queries_given_outputs_and_refusals(dt, cuda):
    c, _, table, lens, q = attention_case(dt, cuda, 7, "int8", BF16, 2, 2, 4, 1, 16, [20, 33])
    fused = torch.zeros((2, 2, 3, 4, D), dtype=BF16, device=cuda)
    fused[:, :, 0] = q
    out = torch.empty_like(q)
    assert dt.cache_attention_forward(fused[:, :, 0], c, table, lens, SCALE, out=out) is out
    assert torch.equal(out, dt.cache_attention_forward(q, c, table, lens, SCALE))
    wide = torch.full((2, 7), -1, dtype=torch.int32, device=cuda)
    wide[:, :table.shape[1]] = table
    assert torch.equal(dt.cache_attention_forward(q, c, wide[:, :table.shape[1]], lens, SCALE), out)
    for bad in (dict(q=q.half()), dict(q=q[:, :, :3]), dict(table=table.long()), dict(lens=lens[:1]), dict(lens=lens.cpu()),
                dict(table=table[:1])):
        a = dict(q=q, table=table, lens=lens)
        a.update(bad)
        with pytest.raises((ValueError, RuntimeError)):
            dt.cache_attention_forward(a["q"], c, a["table"], a["lens"], SCALE)
    with pytest.raises(ValueError, match="out must"):
        dt.cache_attention_forward(q, c, table, lens, SCALE, out=out.float())


# ------------------------------------------------------- a shared prefix

PREFIX_CASES = [
    # B, T, heads, group, page, prefix, lengths behind it
    (1, 1, 1, 1, 16, 1, [0]),
    (3, 1, 2, 1, 16, 100, [0, 1, 40]),
    (5, 2, 2, 2, 32, 129, [2, 3, 31, 64, 90]),
    (40, 1, 1, 4, 64, 500, [i for i in range(40)]),
    (130, 1, 2, 1, 64, 300, [1 + i % 70 for i in range(130)]),
    (70, 3, 1, 2, 128, 1000, [3 + i for i in range(70)]),
    (4, 1, 3, 1, 64, 0, [5, 0, 64, 65]),
    (17, 1, 1, 20, 16, 640, [7] * 17),
]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("case", PREFIX_CASES, ids=lambda c: "b%d_t%d_h%d_g%d_p%d_n%d" % c[:6])
def test_prefix_attention(dt, cuda, fmt, dtype, case):
    B, T, heads, group, page, prefix, lens = case
    c, pages, table, seq_lens, q = attention_case(dt, cuda, 11, fmt, dtype, B, T, heads, group, page, lens, prefix)
    poison(c, table, seq_lens, pages, prefix)
    got = dt.prefix_attention_forward(q, c, pages, prefix, table, seq_lens, SCALE, return_stats=True)
    dt.check_device_error()
    # bf16 queries: the weights of the prefix's keys are rounded to bf16 for the second product
    want = ref.attention(q, c, table, seq_lens, SCALE, prefix_pages=pages, prefix_len=prefix, p_half=2.0 ** -8 if dtype == BF16 else 0.0)
    ref.check_attention(got, want)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_prefix_attention_without_own_keys_with_padding_and_bad_pages(dt, cuda, dtype):
    B, T = 36, 2
    c, pages, table, _, q = attention_case(dt, cuda, 12, "int8", dtype, B, T, 2, 2, 16, [20] * B, 333)
    p_half = 2.0 ** -8 if dtype == BF16 else 0.0
    got = dt.prefix_attention_forward(q, c, pages, 333, None, None, SCALE, return_stats=True)
    ref.check_attention(got, ref.attention(q, c, None, None, SCALE, prefix_pages=pages, prefix_len=333, p_half=p_half))
    pages[3], pages[20], table[2, 0] = -1, c.num_pages + 5, 1 << 30
    seq_lens = torch.arange(B, device=cuda, dtype=torch.int32) - 2
    q_lens = ints(cuda, *[i % 4 - 1 for i in range(B)])
    poison(c, table, seq_lens, pages, 333)
    got = dt.prefix_attention_forward(q, c, pages, 333, table, seq_lens, SCALE, q_lens=q_lens, return_stats=True)
    dt.check_device_error()
    want = ref.attention(q, c, table, seq_lens.clamp_min(0), SCALE, q_lens=q_lens.clamp_min(0), prefix_pages=pages,
                         prefix_len=333, p_half=p_half)
    ref.check_attention(got, want)
    assert bool((got.output[0] == 0).all()) and bool((got.softmax_l[0] == 0).all())  # q_lens -1
    # a prefix whose every page is missing leaves the sequence's own keys
    got = dt.prefix_attention_forward(q, c, torch.full_like(pages, -1), 333, table, seq_lens, SCALE, return_stats=True)
    ref.check_attention(got, ref.attention(q, c, table, seq_lens.clamp_min(0), SCALE))


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads, group", [(1, 3), (2, 20)])
def test_a_long_prefix_in_many_parts(dt, cuda, fmt, dtype, heads, group):
    """More parts than the sequences' own kernel joins, with and without keys of their own."""
    B, prefix = 3, 5003
    c, pages, table, lens, q = attention_case(dt, cuda, 44, fmt, dtype, B, 1, heads, group, 32, [0, 40, 700], prefix)
    poison(c, table, lens, pages, prefix)
    p_half = 2.0 ** -8 if dtype == BF16 else 0.0
    got = dt.prefix_attention_forward(q, c, pages, prefix, table, lens, SCALE, return_stats=True)
    dt.check_device_error()
    ref.check_attention(got, ref.attention(q, c, table, lens, SCALE, prefix_pages=pages, prefix_len=prefix, p_half=p_half))
    got = dt.prefix_attention_forward(q, c, pages, prefix, None, None, -SCALE, return_stats=True)
    ref.check_attention(got, ref.attention(q, c, None, None, -SCALE, prefix_pages=pages, prefix_len=prefix, p_half=p_half))


def test_prefix_scales_that_grow_along_it_and_queries_far_from_one(dt, cuda):
    """The running factor of the weights has to follow v_scale, upwards and with zeros before."""
    for dtype in (BF16, F32):
        c, pages, table, lens, q = attention_case(dt, cuda, 45, "int8", dtype, 4, 1, 1, 1, 64, [3, 9, 0, 64], 1500)
        order = pages.long()
        grow = torch.exp2(torch.linspace(-40, 12, len(order), device=cuda))
        c.v_scale[order] *= grow[:, None, None]
        c.v_scale[order[:4]] = 0.0
        q = (q.float() * torch.tensor([1.0, 2.0 ** -30, 0.0, 2.0 ** 6], device=cuda)[:, None, None, None]).to(dtype)
        p_half = 2.0 ** -8 if dtype == BF16 else 0.0
        got = dt.prefix_attention_forward(q, c, pages, 1500, table, lens, SCALE, return_stats=True)
        o, m, l, o_tol, m_tol, l_tol = ref.attention(q, c, table, lens, SCALE, prefix_pages=pages, prefix_len=1500, p_half=p_half)
        # the prefix's weights are scaled by the largest v_scale, at most 2^6 above which lies 2^15: each is off by at most
        # half of fp16's smallest step, 2^-25, so by 2^-31 of that scale, for codes of at most 127 over weights of at least 1
        o_tol = o_tol + 2.0 ** -31 * float(c.v_scale[torch.isfinite(c.v_scale)].max()) * 127 * 1500
        ref.check_attention(got, (o, m, l, o_tol, m_tol, l_tol))


def test_prefix_attention_equals_the_cache_attention_of_the_whole(dt, cuda):
    """The same keys through one table per sequence: the two paths agree within their bounds."""
    c, pages, table, lens, q = attention_case(dt, cuda, 13, "e4m3", BF16, 48, 1, 2, 1, 32, [33] * 48, 160)
    whole = torch.cat((pages[None].expand(48, -1), table), dim=1).contiguous()
    a = dt.prefix_attention_forward(q, c, pages, 160, table, lens, SCALE, return_stats=True)
    b = dt.cache_attention_forward(q, c, whole, lens + 160, SCALE, return_stats=True)
    want = ref.attention(q, c, whole, lens + 160, SCALE, p_half=2.0 ** -8)
    ref.check_attention(a, want)
    ref.check_attention(b, want)
    with pytest.raises(ValueError, match="prefix_len"):
        dt.prefix_attention_forward(q, c, pages, 161, table, lens, SCALE)
    with pytest.raises(ValueError, match="together"):
        dt.prefix_attention_forward(q, c, pages, 160, table, None, SCALE)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_prefix_key_that_is_not_finite_reaches_its_head_only(dt, cuda, dtype):
    c, pages, table, lens, q = attention_case(dt, cuda, 14, "int8", dtype, 40, 1, 2, 1, 16, [9] * 40, 200)
    want = dt.prefix_attention_forward(q, c, pages, 200, table, lens, SCALE)
    c.v_scale[int(pages[5]), 1, 4] = math.nan
    got = dt.prefix_attention_forward(q, c, pages, 200, table, lens, SCALE)
    assert torch.equal(got[:, :, 0], want[:, :, 0]) and torch.isnan(got[:, :, 1]).all()


# ------------------------------------------------------- log probabilities

def log_prob_ref(x, targets):
    x = x.double()
    lse = torch.logsumexp(x, -1)
    lp = x - lse[..., None]
    p = torch.exp(lp)
    ent = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(-1)
    V = x.shape[-1]
    has = (targets >= 0) & (targets < V)
    got = torch.gather(lp, -1, torch.where(has, targets, torch.zeros_like(targets)).long()[..., None])[..., 0]
    return torch.where(has, got, torch.zeros_like(got)), ent, lse, lp, p


def sum_bound(x):
    """Relative error of sum e^(x - m) in fp32: each term by |x - m| + 8 half steps (argument, base change,
    exponential), the sums by V / 512 + 32 (a thread's share, then a tree), doubled."""
    x = x.double()
    away = (x.amax(-1, keepdim=True) - x).clamp(max=100.0)
    p = torch.softmax(x, -1)
    return 2 * EPS32 * ((p * torch.where(p > 0, away, torch.zeros_like(away))).sum(-1) * 3 + 8 + x.shape[-1] / 512 + 32)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N, V, top", [(1, 1, 1), (3, 2, 2), (2, 31, 31), (5, 257, 20), (4, 1000, 0), (7, 1003, 5), (2, 4096, 32),
                                       (33, 8191, 8), (3, 50257, 20), (4, 100352, 20), (300, 5000, 3)])
def test_token_log_probs(dt, cuda, dtype, N, V, top):
    g = gen(cuda, N * 7 + V)
    x = (torch.randn((N, V), generator=g, device=cuda) * 3).to(dtype)
    x[0, V // 2] += 9
    t = torch.randint(0, V, (N,), generator=g, device=cuda)
    t[N // 2] = V // 2
    r = dt.token_log_probs(x, t, top=top)
    lp, ent, lse, all_lp, _ = log_prob_ref(x, t)
    tol = sum_bound(x) + 4 * EPS32 * (lse.abs() + x.double().abs().amax(-1))
    assert bool(((r.lse.double() - lse).abs() <= tol).all())
    assert bool(((r.log_prob.double() - lp).abs() <= tol + 4 * EPS32 * lp.abs()).all())
    spread = (x.double().amax(-1, keepdim=True) - x.double()).amax(-1).clamp(max=100.0)
    assert bool(((r.entropy.double() - ent).abs() <= sum_bound(x) * (1 + 2 * torch.minimum(spread, ent + 20))).all())
    if top:
        v, i = torch.sort(x.float(), dim=1, descending=True, stable=True)
        assert torch.equal(r.top_ids.long(), i[:, :top])
        want = torch.gather(all_lp, 1, i[:, :top])
        assert bool(((r.top_log_probs.double() - want).abs() <= tol[:, None] + 4 * EPS32 * want.abs()).all())
    else:
        assert r.top_ids is None


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_log_probs_ties_masks_and_values_that_are_not_finite(dt, cuda, dtype):
    V, top = 5003, 12
    x = torch.randn((10, V), generator=gen(cuda, 1), device=cuda)
    low = torch.finfo(dtype).min
    x[0] = 0.25                                  # all alike: the lowest ids
    x[1] = torch.tensor([1.0, 2.0, 2.0, 1.0], device=cuda).repeat(V // 4 + 1)[:V]
    x[2, 5:] = -math.inf                         # a mask that leaves five
    x[3] = -math.inf                             # one that leaves nothing
    x[4, :-3] = low                              # the type's lowest value as a mask
    x[5] = low
    x[6, 77] = math.nan
    x[7, 4000] = math.inf
    x[8] = 0.0
    x[8, ::2] = -0.0                             # zeros of either sign are equal
    x[9] = -math.inf
    x[9, 4321] = -3.0                            # one token left
    x = x.to(dtype)
    t = torch.tensor([3, 0, 2, 9, V - 1, 8, 1, 4000, -100, 4321], device=cuda)
    r = dt.token_log_probs(x, t.to(torch.int32), top=top)
    dt.check_device_error()
    assert r.top_ids[0].tolist() == list(range(top)) and r.top_ids[8].tolist() == list(range(top))
    assert r.top_ids[1].tolist() == torch.sort(x[1].float(), descending=True, stable=True)[1][:top].tolist()
    assert sorted(r.top_ids[2, :5].tolist()) == [0, 1, 2, 3, 4] and r.top_ids[2, 5:].tolist() == list(range(5, top))
    assert bool((r.top_log_probs[2, 5:] == -math.inf).all())
    assert float(r.lse[3]) == -math.inf and float(r.log_prob[3]) == -math.inf and float(r.entropy[3]) == 0.0
    assert r.top_ids[3].tolist() == list(range(top)) and bool((r.top_log_probs[3] == -math.inf).all())
    assert sorted(r.top_ids[4, :3].tolist()) == [V - 3, V - 2, V - 1] and r.top_ids[4, 3:].tolist() == list(range(top - 3))
    for row in (0, 2, 4, 5, 8):
        keep = x[row].double()
        lse = torch.logsumexp(keep, 0)
        p = torch.softmax(keep, 0)
        ent = -(p[p > 0] * torch.log(p[p > 0])).sum()
        assert abs(float(r.entropy[row]) - float(ent)) <= 1e-5 * (1 + float(ent))  # 100 half steps of a sum of 5003
        assert abs(float(r.lse[row]) - float(lse)) <= 1e-5 + abs(float(lse)) * 2 ** -22
    assert float(r.entropy[9]) == 0.0 and float(r.log_prob[9]) == 0.0 and float(r.lse[9]) == -3.0
    assert abs(float(r.log_prob[5]) + math.log(V)) < 1e-4
    for row in (6, 7):
        assert math.isnan(float(r.entropy[row])) and math.isnan(float(r.log_prob[row]))
    assert int(r.top_ids[7, 0]) == 4000 and 77 not in r.top_ids[6].tolist()
    assert float(r.log_prob[8]) == 0.0
    x[6] = math.nan
    assert dt.token_log_probs(x, t, top=3).top_ids[6].tolist() == [0, 1, 2]


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_log_probs_of_few_long_rows_with_ties_and_values_that_are_not_finite(dt, cuda, dtype):
    """Rows over clusters: what one CTA of them sees has to reach the row's result."""
    V, top = 100352, 32
    x = (torch.randn((5, V), generator=gen(cuda, 6), device=cuda) * 2).to(dtype)
    x[0] = 1.5
    x[1, V - 1] = math.nan
    x[2] = -math.inf
    x[2, 70000] = 4.0
    x[3, 1000::7] = 50.0                       # more ties than are collected
    x[4, :99000] = torch.finfo(dtype).min
    t = torch.tensor([5, 0, 70000, 1000, 100000], device=cuda)
    r = dt.token_log_probs(x, t, top=top)
    assert r.top_ids[0].tolist() == list(range(top)) and abs(float(r.log_prob[0]) + math.log(V)) < 1e-4
    assert math.isnan(float(r.lse[1])) and V - 1 not in r.top_ids[1].tolist()
    for row in (1, 3, 4):
        y = x[row].float().nan_to_num(nan=-math.inf)
        assert r.top_ids[row].tolist() == torch.sort(y, descending=True, stable=True)[1][:top].tolist()
    assert float(r.log_prob[2]) == 0.0 and r.top_ids[2].tolist() == [70000] + list(range(top - 1))
    n = len(range(1000, V, 7))
    assert abs(float(r.log_prob[3]) + math.log(n)) < 1e-4 and abs(float(r.entropy[3]) - math.log(n)) < 1e-4


def test_log_probs_shapes_strides_and_refusals(dt, cuda):
    g = gen(cuda, 2)
    wide = torch.randn((4, 6, 1010), generator=g, device=cuda)
    t = torch.randint(0, 1003, (4, 6), generator=g, device=cuda)
    a = dt.token_log_probs(wide[..., 3:1006], t, top=4)               # rows spaced apart, not 16-byte aligned
    b = dt.token_log_probs(wide[..., 3:1006].contiguous(), t, top=4)
    assert a.log_prob.shape == (4, 6) and a.top_ids.shape == (4, 6, 4)
    assert torch.equal(a.top_ids, b.top_ids)
    tol = sum_bound(wide[..., 3:1006]) * 2 + 16 * EPS32 * b.lse.abs().double()
    assert bool(((a.lse.double() - b.lse.double()).abs() <= tol).all())
    none = dt.token_log_probs(wide[0, 0])
    assert none.log_prob is None and none.lse.shape == ()
    empty = dt.token_log_probs(wide[:0], t[:0], top=2)
    assert empty.top_ids.shape == (0, 6, 2)
    for bad in (lambda: dt.token_log_probs(wide[:, :3], t[:, :3]), lambda: dt.token_log_probs(wide, t, top=33),
                lambda: dt.token_log_probs(wide, t.float()), lambda: dt.token_log_probs(wide, t[:3]),
                lambda: dt.token_log_probs(wide.half(), t), lambda: dt.token_log_probs(wide.transpose(1, 2), t),
                lambda: dt.token_log_probs(wide[:, :1].expand(4, 6, 1010), t),
                lambda: dt.token_log_probs(wide[0, 0].expand(4, 6, 1010), t)):
        with pytest.raises(ValueError):
            bad()


def grad_ref(x, t, g, h):
    x = x.double().requires_grad_(True)
    lp = torch.log_softmax(x, -1)
    has = (t >= 0) & (t < x.shape[-1])
    total = 0.0
    if g is not None:
        total = (torch.gather(lp, -1, torch.where(has, t, torch.zeros_like(t)).long()[..., None])[..., 0] * g.double() * has).sum()
    if h is not None:
        total = total - ((torch.exp(lp) * lp).sum(-1) * h.double()).sum()
    return torch.autograd.grad(total, x)[0]


def grad_bound(x, g, h, dtype):
    """Half a step of the type, plus the fp32 error of each term: p is off by |x| + |lse| + |x - lse| + 8 half
    steps, and what it multiplies by as many."""
    x = x.double()
    lse = torch.logsumexp(x, -1, keepdim=True)
    lp = x - lse
    p = torch.exp(lp)
    ent = -(p * lp).sum(-1, keepdim=True)
    g = torch.zeros_like(ent) if g is None else g.double()[..., None].abs()
    h = torch.zeros_like(ent) if h is None else h.double()[..., None].abs()
    steps = 4 * (x.abs() + lse.abs() + lp.abs()) + 64 + sum_bound(x)[..., None] / EPS32
    return EPS32 * steps * p * (g + h * (lp.abs() + ent + 1)) + 4 * EPS32 * g * (p + 1e-30)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N, V", [(1, 1), (2, 7), (3, 256), (5, 1003), (9, 4096), (2, 100352), (200, 777)])
@pytest.mark.parametrize("which", ["both", "log_prob", "entropy"])
def test_token_log_probs_backward(dt, cuda, dtype, N, V, which):
    gn = gen(cuda, N + V)
    x = (torch.randn((N, V), generator=gn, device=cuda) * 3).to(dtype)
    t = torch.randint(0, V, (N,), generator=gn, device=cuda)
    if N > 1:
        t[1] = -100
    g = torch.randn((N,), generator=gn, device=cuda) if which != "entropy" else None
    h = torch.randn((N,), generator=gn, device=cuda) if which != "log_prob" else None
    r = dt.token_log_probs(x, t)
    got = dt.token_log_probs_backward(x, t if g is not None else None, r.lse, r.entropy if h is not None else None, g, h)
    dt.check_device_error()
    want = grad_ref(x, t, g, h)
    tol = HALF[dtype] * want.abs() * 1.01 + grad_bound(x, g, h, dtype)
    if g is not None:
        tol += 4 * EPS32 * torch.zeros_like(want).scatter_(1, t.clamp(0)[:, None], g.double().abs()[:, None])
    # a product below the type's smallest normal value may come back as zero
    assert bool(((got.double() - want).abs() <= tol + 2.0 ** -126).all()), float(((got.double() - want).abs() - tol).max())
    y = x.clone()
    assert dt.token_log_probs_backward(y, t if g is not None else None, r.lse, r.entropy if h is not None else None, g, h, out=y) is y
    assert torch.equal(y, got)  # in place


def test_log_probs_gradient_against_differences(dt, cuda):
    """Central differences of the forward pass in 64 bits, and the forward kernel's own outputs moved along a direction."""
    gn = gen(cuda, 77)
    x = torch.randn((4, 50), generator=gn, device=cuda) * 2
    t = torch.randint(0, 50, (4,), generator=gn, device=cuda)
    g, h = torch.randn((4,), generator=gn, device=cuda), torch.randn((4,), generator=gn, device=cuda)
    r = dt.token_log_probs(x, t)
    dx = dt.token_log_probs_backward(x, t, r.lse, r.entropy, g, h).double()
    d = torch.randn((4, 50), generator=gn, device=cuda)

    def f(y):
        lp, ent, _, _, _ = log_prob_ref(y, t)
        return lp * g.double() + ent * h.double()

    e = 2.0 ** -14
    slope = (f(x.double() + e * d.double()) - f(x.double() - e * d.double())) / (2 * e)
    # cut-off error e^2 / 6 * third derivative (bounded by 50 |d|^3 here), rounding 2^-52 / e
    tol = 1e-5 * (1 + d.double().abs().amax(-1) ** 3) * (1 + g.double().abs() + h.double().abs()) * 4
    assert bool((((dx * d.double()).sum(-1) - slope).abs() <= tol).all())


def test_log_probs_backward_masked_rows_and_logits(dt, cuda):
    x = torch.randn((3, 600), generator=gen(cuda, 4), device=cuda)
    x[0] = -math.inf
    x[1, 100:] = -math.inf
    x[2, 5:] = torch.finfo(F32).min
    t = torch.tensor([4, 3, 1], device=cuda)
    one = torch.ones(3, device=cuda)
    r = dt.token_log_probs(x, t)
    d = dt.token_log_probs_backward(x, t, r.lse, r.entropy, one, one)
    assert bool((d[0] == 0).all()) and bool((d[1, 100:] == 0).all()) and bool((d[2, 5:] == 0).all())
    want = grad_ref(x[1:2, :100], t[1:2], one[1:2], one[1:2])
    tol = EPS32 * want.abs() + grad_bound(x[1:2, :100], one[1:2], one[1:2], F32) + 8 * EPS32
    assert bool(((d[1:2, :100].double() - want).abs() <= tol).all())


def test_model_log_probs_score_a_prompt(dt, cuda):
    import common

    embed, layers, norm, head = common.model_weights(3, 1, 1024)
    model = dt.OlmoModel.from_weights(embed, layers, norm, head)
    ids = torch.randint(0, 1024, (2, 33), generator=gen(cuda, 8), device=cuda)
    r = model.log_probs(ids, top=3)
    logits = model.forward(ids)
    nxt = torch.cat((ids[:, 1:], torch.full((2, 1), -100, device=cuda)), dim=1)
    lp, ent, _, _, _ = log_prob_ref(logits, nxt)
    tol = sum_bound(logits) + 8 * EPS32 * (lp.abs() + logits.double().abs().amax(-1))
    assert r.log_prob.shape == (2, 33) and bool((r.log_prob[:, -1] == 0).all())
    assert bool(((r.log_prob.double() - lp).abs() <= tol).all())
    assert torch.equal(r.top_ids.long(), torch.sort(logits, dim=-1, descending=True, stable=True)[1][..., :3])
    model.close()


# ------------------------------------------------------- together, as they are used

@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_prefill_then_decode_through_the_cache(dt, cuda, fmt):
    """A prefilled batch goes into the cache, tokens follow one by one, each attends to what is there;
    the same numbers come from attention over what the cache reads back."""
    g = gen(cuda, 21)
    B, heads, page, prompt, steps = 3, 4, 16, 45, 6
    lens = ints(cuda, 45, 17, 30)
    per_row = -(-(prompt + steps) // page)
    c = dt.KVCache(B * per_row, page, heads, fmt)
    table = ref.pages_of(g, c.num_pages, B, per_row, cuda)
    k, v = (new_rows(g, (B, prompt, heads, D), BF16, cuda) for _ in range(2))
    c.append(k, v, table, None, lens)
    for i in range(steps):
        kn, vn, q = (torch.randn((B, 1, heads, D), generator=g, device=cuda).to(BF16) for _ in range(3))
        c.append(kn, vn, table, lens)
        lens = lens + 1
        got = dt.cache_attention_forward(q, c, table, lens, SCALE, return_stats=True)
        ref.check_attention(got, ref.attention(q, c, table, lens, SCALE))
    kr, vr = c.read(table, None, prompt + steps, lens, dtype=F32)
    w = torch.einsum("bhd,bkhd->bhk", q[:, 0].double(), kr.double()) * SCALE
    w = w.masked_fill(torch.arange(prompt + steps, device=cuda)[None, None] >= lens[:, None, None], -math.inf)
    o = torch.einsum("bhk,bkhd->bhd", torch.softmax(w, -1), vr.double())
    assert float((got.output[:, 0].double() - o).abs().max()) <= 2.0 ** -8 * float(o.abs().max()) * 1.05
    logits = torch.randn((B, 1000), generator=g, device=cuda)
    r = dt.token_log_probs(logits, logits.argmax(-1), top=1)
    assert torch.equal(r.top_ids[:, 0].long(), logits.argmax(-1)) and torch.equal(r.top_log_probs[:, 0], r.log_prob)


def step_of(dt, cuda, fmt):
    """One decoding step's calls on fixed buffers, and the buffers to change between steps."""
    c, pages, table, lens, q = attention_case(dt, cuda, 31, fmt, BF16, 40, 1, 2, 2, 16, [50] * 40, 200)
    k = torch.randn((40, 1, 2, D), device=cuda).to(BF16)
    logits = torch.randn((6, 3001), device=cuda)
    t = torch.zeros(6, dtype=torch.int64, device=cuda)
    at = torch.full((40,), 49, dtype=torch.int32, device=cuda)

    def step():
        c.append(k, k, table, at)
        a = dt.cache_attention_forward(q, c, table, lens, SCALE)
        p = dt.prefix_attention_forward(q, c, pages, 200, table, lens, SCALE)
        r = dt.token_log_probs(logits, t, top=4)
        dx = dt.token_log_probs_backward(logits, t, r.lse, r.entropy, r.log_prob, r.entropy)
        kr, _ = c.read(table, None, 50)
        return [a, p, r.log_prob, r.entropy, r.lse, r.top_ids, r.top_log_probs, dx, kr]

    return step, (k, q, logits)


def test_captured_steps_replay_on_new_inputs_and_two_graphs_do_not_mix(dt, cuda):
    ones, twos = step_of(dt, cuda, "int8"), step_of(dt, cuda, "e4m3")
    graphs = []
    for step, _ in (ones, twos):
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for i in range(3):
        for _, bufs in (ones, twos):
            for b in bufs:
                b.copy_(torch.randn(b.shape, device=cuda).to(b.dtype))
        torch.cuda.synchronize()
        side = [torch.cuda.Stream(), torch.cuda.Stream()]
        for s, (graph, _) in zip(side, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        replayed = [[x.clone() for x in out] for _, out in graphs]
        for (step, _), got in zip((ones, twos), replayed):
            for a, b in zip(step(), got):
                assert torch.equal(a, b)


def test_calls_on_two_streams_at_once_keep_their_results(dt, cuda):
    step, _ = step_of(dt, cuda, "int8")
    want = step()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(step())
    torch.cuda.synchronize()
    for out in got:
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_counts_past_32_bits_are_refused(dt, cuda):
    cache = dt.KVCache(1, 16, 1, device=cuda)
    one = torch.ones((1, 1, 1, 128), dtype=torch.bfloat16, device=cuda)
    table = torch.zeros((1, 1), dtype=torch.int32, device=cuda)
    many = one.expand(1, 2**32 + 1, 1, 128)  # (no memory of its own)
    for bad in (lambda: cache.append(many, many, table), lambda: cache.read(table, None, -1),
                lambda: cache.read(table, None, 2**32 + 1),
                lambda: dt.cache_attention_forward(many, cache, table, table[0], 1.0),
                lambda: dt.prefix_attention_forward(one, cache, table[0], 2**32 + 1, None, None, 1.0)):
        with pytest.raises(ValueError):
            bad()
    assert float(cache.k_scale.abs().sum()) == 0.0
    long = torch.empty(2**32 + 5, dtype=torch.bfloat16, device=cuda)  # 8.6 GB
    for bad in (long, long[:, None]):
        with pytest.raises(ValueError):
            dt.token_log_probs(bad)


def test_gradient_into_the_other_half_of_the_logits_rows(dt, cuda):
    g = gen(cuda, 5)
    both = torch.randn((9, 2, 333), generator=g, device=cuda)
    x, out, t = both[:, 0], both[:, 1], torch.randint(0, 333, (9,), generator=g, device=cuda)
    r = dt.token_log_probs(x, t)
    up = torch.randn((9,), generator=g, device=cuda)
    plain = dt.token_log_probs_backward(x.contiguous(), t, r.lse, r.entropy, up)
    kept = x.clone()
    dt.token_log_probs_backward(x, t, r.lse, r.entropy, up, out=out)
    # the same formula in the same order whatever the alignment
    assert torch.equal(x, kept) and torch.equal(out, plain)
    with pytest.raises(dt.DTError, match="overlap"):
        dt.token_log_probs_backward(both.view(18, 333)[:-1], None, r.lse.new_zeros(17), None, None,
                                    out=both.view(18, 333)[1:])
