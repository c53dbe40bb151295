"""Plain 64-bit forms of the serving operators, and the error bounds that the tests hold them to."""
from __future__ import annotations

import torch

D = 128
TOP = {"int8": 127.0, "e4m3": 448.0}
CODE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
EPS32 = 2.0 ** -24                                        # half a step of fp32
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: EPS32}  # half a step, relative to the value


def values(codes, scales):
    """code * scale in 64 bits."""
    return codes.float().double() * scales.double()[..., None]


def make_cache(gen, fmt, pages, heads, page, device):
    """Random codes and scales as a KVCache's four arrays."""
    out = []
    for _ in range(2):
        x = (torch.randn((pages, heads, page, D), generator=gen, device=device) * TOP[fmt] / 3).clamp(-TOP[fmt], TOP[fmt])
        out.append((x.round() if fmt == "int8" else x).to(CODE[fmt]))
        out.append(torch.exp(torch.randn((pages, heads, page), generator=gen, device=device) * 0.5) * 3 / TOP[fmt])
    return out[0], out[2], out[1], out[3]  # k, v, k_scale, v_scale


def pages_of(gen, pages, B, per_row, device):
    """A page table [B, per_row] of distinct pages in random order."""
    return torch.randperm(pages, generator=gen, device=device)[: B * per_row].view(B, per_row).to(torch.int32)


def keys_of(cache, pages, head, n):
    """K and V rows 0 .. n - 1 of one head along a list of pages, V's scales and |codes|, and which rows exist."""
    ok = (pages >= 0) & (pages < cache.num_pages)
    at = torch.where(ok, pages, torch.zeros_like(pages)).long()
    k = values(cache.k.view(torch.int8)[at, head].view(cache.k.dtype), cache.k_scale[at, head]).reshape(-1, D)[:n]
    v = values(cache.v.view(torch.int8)[at, head].view(cache.v.dtype), cache.v_scale[at, head]).reshape(-1, D)[:n]
    codes = cache.v.view(torch.int8)[at, head].view(cache.v.dtype).float().double().reshape(-1, D)[:n].abs()
    return k, v, cache.v_scale[at, head].double().reshape(-1)[:n], codes, ok.repeat_interleave(cache.page_size)[:n]


def attention(q, cache, table, seq_lens, scale, q_lens=None, prefix_pages=None, prefix_len=0, p_half=0.0):
    """Output, m, l and how far each may be off: (o, m, l, o_tol, m_tol, l_tol), all fp64.

    A score is a sum of 128 products in fp32 and two roundings of its scales: off by at most
    d = (128 + 4) * 2 * EPS32 * sum |q k| (twice, since the tensor cores may cut instead of round).
    A weight is then off by a factor of about 1 +- (2 d + 8 EPS32 (1 + |s - m|)), the sums of n
    weights by n * 2 * EPS32 more; p_half is half a step of the type that the weights are rounded to
    for the second product (for bf16 queries at least fp16's, 2^-11).
    """
    B, T, H, _ = q.shape
    group = H // cache.kv_heads
    if q.dtype == torch.bfloat16:
        p_half = max(p_half, 2.0 ** -11)
    qd = q.double()
    o = torch.zeros((B, T, H, D), dtype=torch.float64, device=q.device)
    m, l = torch.zeros((B, T, H), dtype=torch.float64, device=q.device), torch.zeros((B, T, H), dtype=torch.float64, device=q.device)
    o_tol, m_tol, l_tol = torch.zeros_like(o), torch.zeros_like(m), torch.zeros_like(l)
    cap = 0 if table is None else table.shape[1] * cache.page_size
    for b in range(B):
        n_q = T if q_lens is None else min(int(q_lens[b]), T)
        for h in range(H):
            parts = []
            if prefix_len:
                parts.append(keys_of(cache, prefix_pages, h // group, prefix_len))
            own = 0 if table is None else min(int(seq_lens[b]), cap)
            if own > 0:
                parts.append(keys_of(cache, table[b], h // group, own))
            for t in range(n_q):
                last = 0 if table is None else max(0, min(int(seq_lens[b]) - n_q + t + 1, cap))
                seen = []
                for i, part in enumerate(parts):
                    n = prefix_len if prefix_len and i == 0 else last
                    seen.append([x[:n][part[-1][:n]] for x in part[:-1]])
                if sum(len(x[0]) for x in seen) == 0:
                    continue
                k, v, vs, codes = (torch.cat(x) for x in zip(*seen))
                s = k @ qd[b, t, h] * scale
                d = float((132 * 2 * EPS32 * (k.abs() @ qd[b, t, h].abs()) * abs(scale)).max())
                m[b, t, h] = s.max()
                w = torch.exp(s - s.max())
                l[b, t, h] = w.sum()
                p = w / w.sum()
                o[b, t, h] = p @ v
                rel = 2 * d + 8 * EPS32 * (1 + float((p * (s.max() - s)).sum())) + 2 * len(k) * EPS32 + p_half
                o_tol[b, t, h] = HALF[q.dtype] * o[b, t, h].abs() + 2 * rel * (p @ v.abs())
                # The second product takes p * v_scale as fp16 numbers (fp32 queries: as two), scaled so that a row's largest
                # is at least 2^8: each is off by at most half of fp16's smallest step, 2^-25, so by 2^-33 of the largest.
                o_tol[b, t, h] += 2.0 ** -33 * float((p * vs).max()) * codes.sum(0)
                m_tol[b, t, h] = d + EPS32 * abs(float(s.max()))
                l_tol[b, t, h] = (2 * d + 8 * EPS32 * (1 + float((p * (s.max() - s)).sum())) + 2 * len(k) * EPS32) * w.sum()
    return o, m, l, o_tol, m_tol, l_tol


def check_attention(got, ref):
    """Every value within its own bound; exact zeros (padding, rows without keys) stay zeros."""
    for name, g, r, tol in zip(("output", "softmax_m", "softmax_l"), got, ref[:3], ref[3:]):
        far = (g.double() - r).abs() - tol
        assert torch.isfinite(g.float()).all(), f"{name}: not finite"
        assert float(far.max()) <= 0, f"{name}: off by {float((g.double() - r).abs().max()):.3g}, {float(far.max()):.3g} over its bound"
