"""GPU tests of the prefix attention within the bounds of what it rounds: weights to fp16 (2^-11), not to bf16 (2^-8), so
that a key that is lost or counted twice shows."""
import math

import pytest
import torch

import serving_ref as ref
from serving_ref import D, EPS32, HALF
from test_serving_gpu import PREFIX_CASES, attention_case, poison

pytestmark = pytest.mark.gpu

SCALE = 1.0 / math.sqrt(D)
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def dt(cuda):
    import dirktensor_b200

    return dirktensor_b200


def attention(q, c, table, seq_lens, scale, prefix_pages=None, prefix_len=0):
    """serving_ref.attention's values and bounds for full queries, a K/V head's rows at a time.  The step of the weights
    is the prefix form's: scaled so that a row's largest p * v_scale is at least 1, each is off by at most 2^-25 of that."""
    B, T, H, _ = q.shape
    group = H // c.kv_heads
    out = [torch.zeros(q.shape[:n], dtype=torch.float64, device=q.device) for n in (4, 3, 3, 4, 3, 3)]
    p_half = 2.0 ** -11 if q.dtype == BF16 else 0.0
    for b in range(B):
        own = 0 if table is None else max(0, min(int(seq_lens[b]), table.shape[1] * c.page_size))
        for h in range(c.kv_heads):
            spans = [(prefix_pages, prefix_len)] * (prefix_len > 0) + ([(table[b], own)] if own else [])
            if not spans:
                continue
            k, v, vs, codes, ok = (torch.cat(x) for x in zip(*(ref.keys_of(c, pages, h, n) for pages, n in spans)))
            t = torch.arange(T, device=q.device)[:, None]
            j = torch.arange(len(k), device=q.device)[None] - prefix_len
            see = (ok[None] & ((j < 0) | (j < own - T + t + 1)))[:, None]                 # [T, 1, keys]
            k, v, vs, codes = (torch.where(ok if x.dim() == 1 else ok[:, None], x, torch.zeros_like(x)) for x in (k, v, vs, codes))
            x = q[b, :, h * group:(h + 1) * group].double()
            s = (torch.matmul(x, k.T) * scale).masked_fill(~see, -math.inf)
            d = (132 * 2 * EPS32 * torch.matmul(x.abs(), k.abs().T) * abs(scale)).masked_fill(~see, 0.0).amax(-1)
            top = s.amax(-1)
            some = torch.isfinite(top)
            top = torch.where(some, top, torch.zeros_like(top))
            w = torch.exp(s - top[..., None])
            l = w.sum(-1)
            p = w / torch.where(some, l, torch.ones_like(l))[..., None]
            away = (p * torch.where(see, top[..., None] - s, torch.zeros_like(s))).sum(-1)
            rel = 2 * d + 8 * EPS32 * (1 + away) + 2 * see.sum(-1) * EPS32
            o = torch.matmul(p, v)
            o_tol = (HALF[q.dtype] * o.abs() + 2 * (rel + p_half)[..., None] * torch.matmul(p, v.abs()) +
                     2.0 ** -25 * (p * vs).amax(-1, keepdim=True) * torch.matmul(see.double(), codes))
            for at, y in zip(out, (o, top, l, o_tol, d + EPS32 * top.abs(), rel * l)):
                at[b, :, h * group:(h + 1) * group] = y
    return out


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("case", PREFIX_CASES, ids=lambda c: "b%d_t%d_h%d_g%d_p%d_n%d" % c[:6])
def test_prefix_attention_within_the_bounds_of_fp16_weights(dt, cuda, fmt, dtype, case):
    B, T, heads, group, page, prefix, lens = case
    c, pages, table, seq_lens, q = attention_case(dt, cuda, 51, fmt, dtype, B, T, heads, group, page, lens, prefix)
    poison(c, table, seq_lens, pages, prefix)
    got = dt.prefix_attention_forward(q, c, pages, prefix, table, seq_lens, SCALE, return_stats=True)
    dt.check_device_error()
    ref.check_attention(got, attention(q, c, table, seq_lens, SCALE, pages, prefix))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads, group", [(1, 3), (2, 20)])
def test_a_long_prefix_in_many_parts_within_the_bounds(dt, cuda, dtype, heads, group):
    c, pages, table, lens, q = attention_case(dt, cuda, 52, "int8", dtype, 3, 1, heads, group, 32, [0, 40, 700], 5003)
    pages[7], table[2, 3] = -1, c.num_pages
    poison(c, table, lens, pages, 5003)
    got = dt.prefix_attention_forward(q, c, pages, 5003, table, lens, SCALE, return_stats=True)
    ref.check_attention(got, attention(q, c, table, lens, SCALE, pages, 5003))
    got = dt.prefix_attention_forward(q, c, pages, 5003, None, None, -SCALE, return_stats=True)
    ref.check_attention(got, attention(q, c, None, None, -SCALE, pages, 5003))


def test_both_forms_of_the_same_keys_within_the_bounds(dt, cuda):
    c, pages, table, lens, q = attention_case(dt, cuda, 53, "e4m3", BF16, 48, 1, 2, 1, 32, [33] * 48, 160)
    whole = torch.cat((pages[None].expand(48, -1), table), dim=1).contiguous()
    a = dt.prefix_attention_forward(q, c, pages, 160, table, lens, SCALE, return_stats=True)
    b = dt.cache_attention_forward(q, c, whole, lens + 160, SCALE, return_stats=True)
    want = attention(q, c, whole, lens + 160, SCALE)
    ref.check_attention(a, want)
    ref.check_attention(b, ref.attention(q, c, whole, lens + 160, SCALE))
