"""GPU tests of the cache attention and the prefix attention where rows of V differ much in size.

Every value has its bound from serving_ref.attention: the second product takes the weights p * v_scale as fp16
numbers (fp32 queries: as two), scaled so that the largest of those summed so far is well inside fp16's range whatever
came before it."""
import math

import pytest
import torch

import serving_ref as ref
from serving_ref import D

pytestmark = pytest.mark.gpu

SCALE = 1.0 / math.sqrt(D)
BF16, F32 = torch.bfloat16, torch.float32
LOG2 = math.log(2.0)


@pytest.fixture(scope="module")
def dt(cuda):
    import dirktensor_b200

    return dirktensor_b200


def given(dt, cuda, fmt, dtype, B, T, heads, group, scores, sizes, page=64, spare=0):
    """A cache whose key j of every sequence and head has about the score scores[j] (in log2 units) for every query, and a V
    row of about the size sizes[j] (0: a row of zeros).  Queries are 16 in dim 0, so K's code and scale there give the score;
    the rest of K is noise below it.  Returns cache, page table [B, pages], lengths, queries."""
    g = torch.Generator(device=cuda)
    g.manual_seed(len(scores))
    n = len(scores)
    per = -(-n // page)
    c = dt.KVCache.from_tensors(*ref.make_cache(g, fmt, B * per + spare, heads, page, cuda))
    table = torch.randperm(c.num_pages, generator=g, device=cuda)[: B * per].view(B, per).to(torch.int32)
    want = torch.tensor(scores, device=cuda, dtype=torch.float64) * LOG2  # in nats
    rows = torch.arange(n, device=cuda)
    at, off = table.long()[:, rows // page], rows % page                 # [B, n], [n]
    code = torch.zeros((n, D), device=cuda)
    code[:, 0] = torch.where(want < 0, -64.0, 64.0)
    ks = (want.abs() / (SCALE * 16 * 64)).float()
    vs = torch.tensor(sizes, device=cuda, dtype=torch.float64) / ref.TOP[fmt]
    for b in range(B):
        c.k[at[b], :, off] = code.to(c.k.dtype)[:, None].expand(n, heads, D)
        c.k_scale[at[b], :, off] = ks[:, None].expand(n, heads)
        c.v_scale[at[b], :, off] = vs.float()[:, None].expand(n, heads)
    q = torch.zeros((B, T, heads * group, D), device=cuda)
    q[..., 0] = 16.0
    return c, table, torch.full((B,), n, dtype=torch.int32, device=cuda), q.to(dtype)


# Which keys come first (in every warp's first tile of 32, and the tiles after it), and which after them.
def tiny_rows(first, rest, size):
    """Rows of V of 2^size, then ordinary ones."""
    return [0.0] * (first + rest), [2.0 ** size] * first + [1.0] * rest


def zero_row_at_the_peak(first, rest, below):
    """In each tile of 32 a key with a V row of zeros leads the others by `below` log2 units; an ordinary key at
    the peak follows in each of the tiles after them."""
    scores = [0.0 if j % 32 == 5 else -float(below) for j in range(first)]
    sizes = [0.0 if j % 32 == 5 else 1.0 for j in range(first)]
    return scores + [0.0 if j % 32 == 9 else -30.0 for j in range(rest)], sizes + [1.0] * rest


EARLY = [pytest.param(tiny_rows, (size,), id="tiny%d" % size) for size in (-100, -90, -80)] + [
    pytest.param(zero_row_at_the_peak, (below,), id="zero_peak_%d" % below) for below in (78, 80, 84, 88, 96)]


# A warp's second tile comes 4 * split tiles after its first.  One item of up to 128 tiles is a cluster of 8: 1024 keys on.
# Eight items over a wide page table are shared out: 592 CTAs, 74 an item, 9472 keys on (fewer where fewer CTAs fit).
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("group", [1, 8, 20])
@pytest.mark.parametrize("early, args", EARLY)
def test_sums_of_the_first_factor_are_kept_in_later_units(dt, cuda, fmt, dtype, group, early, args):
    c, table, lens, q = given(dt, cuda, fmt, dtype, 1, 1, 1, group, *early(1024, 1999, *args))
    got = dt.cache_attention_forward(q, c, table, lens, SCALE, return_stats=True)
    ref.check_attention(got, ref.attention(q, c, table, lens, SCALE))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("early, args", EARLY)
def test_sums_of_the_first_factor_are_kept_where_keys_are_shared_out(dt, cuda, dtype, early, args):
    c, table, lens, q = given(dt, cuda, "int8", dtype, 1, 1, 8, 1, *early(9472, 14000, *args))
    got = dt.cache_attention_forward(q, c, table, lens, SCALE, return_stats=True)
    ref.check_attention(got, ref.attention(q, c, table, lens, SCALE))


def large_rows_that_vanish(first, rest, ratio, below):
    """Rows of V that are 2^ratio times as large as those that come later, whose scores are `below` log2 units higher."""
    return [-float(below)] * first + [0.0] * rest, [2.0 ** ratio] * first + [1.0] * rest


def large_rows_that_vanish_by_steps(first, rest, ratio, below):
    """The same, with the scores going up through all keys after the first ones."""
    scores, sizes = large_rows_that_vanish(first, rest, ratio, below)
    return scores[:first] + [-below * (1 - j / (rest - 1)) for j in range(rest)], sizes


VANISH = [pytest.param(f, (ratio, below), id="%s_%d_%d" % (name, ratio, below))
          for name, f in (("at_once", large_rows_that_vanish), ("by_steps", large_rows_that_vanish_by_steps))
          for ratio, below in ((24, 60), (34, 90), (34, 50), (60, 120))]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("group", [1, 8, 20])
@pytest.mark.parametrize("early, args", VANISH)
def test_large_rows_that_vanish_leave_the_later_weights_their_digits(dt, cuda, fmt, dtype, group, early, args):
    c, table, lens, q = given(dt, cuda, fmt, dtype, 1, 1, 1, group, *early(1024, 2999, *args))
    got = dt.cache_attention_forward(q, c, table, lens, SCALE, return_stats=True)
    ref.check_attention(got, ref.attention(q, c, table, lens, SCALE))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("early, args", VANISH)
def test_large_rows_that_vanish_where_keys_are_shared_out(dt, cuda, dtype, early, args):
    c, table, lens, q = given(dt, cuda, "int8", dtype, 1, 1, 8, 1, *early(9472, 30000, *args))
    got = dt.cache_attention_forward(q, c, table, lens, SCALE, return_stats=True)
    ref.check_attention(got, ref.attention(q, c, table, lens, SCALE))


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n, heads", [(70, 2), (500, 1), (20000, 8)])
def test_the_smallest_rows_that_are_kept_and_the_largest(dt, cuda, fmt, dtype, n, heads):
    """All rows of V of 2^-100 (what is smaller is stored as zeros), of 2^100, or of both in turn."""
    for sizes in ([2.0 ** -100] * n, [2.0 ** 100] * n, [2.0 ** (100 if j % 3 else -100) for j in range(n)]):
        c, table, lens, q = given(dt, cuda, fmt, dtype, 1, 1, heads, 1, [0.25 * (j % 5) for j in range(n)], sizes)
        got = dt.cache_attention_forward(q, c, table, lens, SCALE, return_stats=True)
        ref.check_attention(got, ref.attention(q, c, table, lens, SCALE))


# ------------------------------------------------------- a shared prefix

HEADS, SEEN = 75, [0, 41, 74]  # so many K/V heads that each CTA takes a whole prefix; the ones that are looked at


def prefix_ref(dt, c, pages, n, q, group):
    """softmax(scale q k^T) v over a prefix for the K/V heads in SEEN, with serving_ref.attention's bounds: (o, m, l and
    the bound of each).  Here the weights p * v_scale are scaled so that a row's largest is at least 1: each is off by at
    most 2^-25 of that, half of fp16's smallest step."""
    o, m, l, o_tol, m_tol, l_tol = ([] for _ in range(6))
    p_half = 2.0 ** -11 if q.dtype == BF16 else 0.0
    for h in SEEN:
        k, v, vs, codes, _ = ref.keys_of(c, pages, h, n)
        x = q[:, :, h * group:(h + 1) * group].double()
        s = torch.matmul(x, k.T) * SCALE
        d = (132 * 2 * ref.EPS32 * torch.matmul(x.abs(), k.abs().T) * SCALE).amax(-1)
        top = s.amax(-1)
        w = torch.exp(s - top[..., None])
        p = w / w.sum(-1, keepdim=True)
        rel = 2 * d + 8 * ref.EPS32 * (1 + (p * (top[..., None] - s)).sum(-1)) + 2 * n * ref.EPS32
        o.append(torch.matmul(p, v))
        o_tol.append(ref.HALF[q.dtype] * o[-1].abs() + 2 * (rel + p_half)[..., None] * torch.matmul(p, v.abs()) +
                     2.0 ** -25 * (p * vs.abs()).amax(-1, keepdim=True) * codes.sum(0))
        m.append(top), m_tol.append(d + ref.EPS32 * top.abs())
        l.append(w.sum(-1)), l_tol.append(rel * w.sum(-1))
    return [torch.cat(x, dim=2) for x in (o, m, l, o_tol, m_tol, l_tol)]


def check_prefix(dt, cuda, fmt, dtype, B, T, scores, sizes):
    c, table, _, q = given(dt, cuda, fmt, dtype, 1, 1, HEADS, 1, scores, sizes)
    q = q.expand(B, T, HEADS, D)
    got = dt.prefix_attention_forward(q, c, table[0], len(scores), None, None, SCALE, return_stats=True)
    dt.check_device_error()
    ref.check_attention([x[:, :, SEEN] for x in got], prefix_ref(dt, c, table[0], len(scores), q, 1))


# 128 rows at most: two warpgroups take tiles of 128 keys in turn; more: each takes 128 rows and all tiles.
PREFIX_ROWS = [pytest.param(BF16, 3, 1, id="bf16_3"), pytest.param(BF16, 41, 4, id="bf16_164"), pytest.param(F32, 2, 1, id="fp32_2"),
               pytest.param(F32, 45, 3, id="fp32_135")]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype, B, T", PREFIX_ROWS)
@pytest.mark.parametrize("size", [41, 60, 100, 112])
def test_prefix_rows_of_zeros_before_very_large_ones(dt, cuda, fmt, dtype, B, T, size):
    check_prefix(dt, cuda, fmt, dtype, B, T, [0.0] * 900, [0.0] * 300 + [2.0 ** size] * 600)


@pytest.mark.parametrize("dtype, B, T", PREFIX_ROWS)
@pytest.mark.parametrize("step", [0, 1, 2, 3])
def test_prefix_rows_that_grow_slowly(dt, cuda, dtype, B, T, step):
    """Rows of V that double `step` times every two tiles: each change of the factor, the smallest too, reaches what is summed."""
    check_prefix(dt, cuda, "int8", dtype, B, T, [0.5 * (j % 3) for j in range(1000)], [2.0 ** (step * (j // 256)) for j in range(1000)])


def large_rows_beside(first, rest, ratio, below):
    """Every other key has a row of V that is 2^ratio times as large, and a score `below` log2 units lower."""
    n = first + rest
    return [-float(below * (j % 2)) for j in range(n)], [2.0 ** (ratio * (j % 2)) for j in range(n)]


def a_row_of_zeros_leads(first, rest, ratio, below):
    """The key at the peak of every tile of 128 has a row of zeros, the others' rows are 2^ratio and far below it."""
    n = first + rest
    return [0.0 if j % 128 == 70 else -float(below) for j in range(n)], [0.0 if j % 128 == 70 else 2.0 ** ratio for j in range(n)]


PREFIX_EARLY = EARLY + VANISH + [pytest.param(f, args, id="%s_%d_%d" % ((name,) + args)) for name, f, args in (
    ("beside", large_rows_beside, (24, 70)), ("beside", large_rows_beside, (34, 90)), ("beside", large_rows_beside, (4, 30)),
    ("beside", large_rows_beside, (60, 70)), ("zeros_lead", a_row_of_zeros_leads, (0, 40)), ("zeros_lead", a_row_of_zeros_leads, (50, 70)),
    ("zeros_lead", a_row_of_zeros_leads, (-60, 30)))]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype, B, T", PREFIX_ROWS)
@pytest.mark.parametrize("early, args", PREFIX_EARLY)
def test_prefix_rows_far_apart_in_size(dt, cuda, fmt, dtype, B, T, early, args):
    check_prefix(dt, cuda, fmt, dtype, B, T, *early(256, 1300, *args))


@pytest.mark.parametrize("dtype, B, T", PREFIX_ROWS)
@pytest.mark.parametrize("size, scale", [(0.0, 1e-5), (0.0, -1e-5), (2.0 ** -100, 1e-5), (2.0 ** -60, 1e-30), (0.0, 1e-44), (1.0, 0.0),
                                         (1.0, 1e-38), (2.0 ** -100, 1.0)])
def test_prefix_of_small_queries_and_scales_with_hidden_keys(dt, cuda, dtype, B, T, size, scale):
    """A query of zeros, or a scale so small that every score is next to none: an even average, and no NaN from keys past
    the end or on a page that does not exist."""
    n, heads = 400, 2
    c, table, _, q = given(dt, cuda, "int8", dtype, 1, 1, heads, 1, [0.0] * n, [1.0] * n)
    q = (torch.randn((B, T, heads, D), device=cuda, generator=torch.Generator(device=cuda).manual_seed(3)) * size).to(dtype)
    c.k_scale.fill_(1.0)
    pages = table[0].clone()
    pages[3] = -1
    for prefix, given_pages in ((100, table[0]), (n, pages), (n - 1, table[0])):
        got = dt.prefix_attention_forward(q, c, given_pages, prefix, None, None, scale, return_stats=True)
        want = list(ref.attention(q[:2], c, None, None, scale, prefix_pages=given_pages, prefix_len=prefix))
        # The scale's product with a power of two is off by half of fp32's smallest step, 2^-150, where it is subnormal (by 2^-149
        # where it would be zero); what it multiplies, a query of at most 2^14 times one code of 64, is at most 2^20.
        want[4] = want[4] + 2.0 ** -129
        ref.check_attention([x[:2] for x in got], want)
        assert all(bool(torch.isfinite(x).all()) for x in got)
        own = dt.cache_attention_forward(q, c, given_pages[None].expand(B, -1).contiguous(),
                                         torch.full((B,), prefix + T - 1, dtype=torch.int32, device=cuda), scale)
        assert bool(torch.isfinite(own).all())


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype, B, T", PREFIX_ROWS)
@pytest.mark.parametrize("sizes", [(1.0, 1.0), (2.0 ** 40, 1.0), (2.0 ** -40, 2.0 ** 20)])
def test_scales_of_either_sign(dt, cuda, fmt, dtype, B, T, sizes):
    """A caller's own codes may have scales below zero (append writes none): their size is what the weights' factor goes by."""
    n = 1300
    c, table, lens, q = given(dt, cuda, fmt, dtype, 1, 1, HEADS, 1, [0.2 * (j % 7) for j in range(n)],
                              [sizes[j % 2] for j in range(n)])
    c.v_scale[:, :, ::2] *= -1
    c.k_scale[:, :, 1::3] *= -1
    q = q.expand(B, T, HEADS, D)
    got = dt.prefix_attention_forward(q, c, table[0], n, None, None, SCALE, return_stats=True)
    ref.check_attention([x[:, :, SEEN] for x in got], prefix_ref(dt, c, table[0], n, q, 1))
    got = dt.cache_attention_forward(q[:1, :1], c, table, lens, SCALE, return_stats=True)
    ref.check_attention([x[:, :, SEEN] for x in got], prefix_ref(dt, c, table[0], n, q[:1, :1], 1))
