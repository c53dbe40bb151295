"""What serving and scoring with the framework cost: the quantised K/V cache, the attention that reads
it, attention over a shared prefix, and the log probabilities of given tokens with their gradient.

``listed()`` and ``draw()`` give cases, ``prepare()`` a case's inputs on the GPU, ``run()`` one pass:
the operators' plain forms in elementary torch operations where ``own`` is false, the framework's own
entry points where it is true.  ``work()`` counts what a pass cannot do without, and ``exact()`` gives
its outputs in 64 bits.

The cache keeps one 8-bit code per value and one fp32 scale per row of 128 values (one token, one
head), in pages of ``page`` tokens: codes [pages, heads, page, 128], scales [pages, heads, page].
"""
import math

import torch

own = False

D = 128             # head size
VOCAB = 100352      # the model's vocabulary
CODES = {"int8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
TINY = 2.0 ** -100  # rows whose largest value is below this are stored as zeros


def listed():
    return [
        # one new token for each of a few sequences: what every decoding step writes
        dict(name="append_step", op="update", fmt="int8", dtype="bf16", out="bf16", B=8, T=1, heads=16, page=64, pos=1000),
        # a prefilled batch goes into the cache from fp32 K and V: the largest write
        dict(name="append_prefill", op="update", fmt="e4m3", dtype="fp32", out="bf16", B=4, T=4096, heads=16, page=64, pos=0),
        # a chunk behind a ragged history, few K/V heads, small pages
        dict(name="append_chunk", op="update", fmt="int8", dtype="bf16", out="fp32", B=5, T=331, heads=8, page=16, pos=77),
        # one sequence, one token: latency
        dict(name="attend_one", op="attend", fmt="int8", dtype="bf16", B=1, T=1, heads=16, group=1, page=64, length=513, ragged=False),
        # a serving batch of the model's own heads at ragged lengths: bandwidth
        dict(name="attend_batch", op="attend", fmt="int8", dtype="bf16", B=64, T=1, heads=16, group=1, page=64, length=4096, ragged=True),
        # one very long sequence: the key axis has to be split
        dict(name="attend_long", op="attend", fmt="e4m3", dtype="fp32", B=1, T=1, heads=8, group=1, page=128, length=131071, ragged=False),
        # a few drafted tokens checked at once, grouped heads
        dict(name="attend_draft", op="attend", fmt="e4m3", dtype="bf16", B=16, T=4, heads=8, group=4, page=32, length=2047, ragged=True),
        # a batch of answers to one long document
        dict(name="prefix_batch", op="prefix", fmt="int8", dtype="bf16", B=64, T=1, heads=16, group=1, page=64, prefix=8192, length=300, ragged=True),
        # many samples of one prompt, grouped heads
        dict(name="prefix_samples", op="prefix", fmt="e4m3", dtype="bf16", B=200, T=1, heads=8, group=4, page=64, prefix=6143, length=128, ragged=True),
        # scores of the next token of a small batch, with alternatives
        dict(name="logprobs_step", op="logprobs", dtype="fp32", N=4, V=VOCAB, top=20),
        # scores of a whole prompt: the largest read
        dict(name="logprobs_prompt", op="logprobs", dtype="fp32", N=2048, V=VOCAB, top=5),
        # gradient of log probabilities and entropies for training on them
        dict(name="logprobs_grad", op="logprobs_grad", dtype="bf16", N=1023, V=VOCAB),
    ]


def _between(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["update", "attend", "attend", "prefix", "logprobs", "logprobs_grad"])
    c = dict(op=op)
    if op in ("logprobs", "logprobs_grad"):
        V = rng.choice([VOCAB, VOCAB, _between(rng, 1000, VOCAB)])
        c.update(dtype=rng.choice(["fp32", "bf16"]), N=_between(rng, 1, 600), V=V)
        if op == "logprobs":
            c["top"] = rng.choice([0, 1, 5, 20])
        return c
    c.update(fmt=rng.choice(["int8", "e4m3"]), dtype=rng.choice(["bf16", "bf16", "fp32"]), page=rng.choice([16, 32, 64, 128]))
    if op == "update":
        B = _between(rng, 1, 64)
        c.update(out=rng.choice(["bf16", "fp32"]), B=B, T=_between(rng, 1, max(1, 12000 // B)), heads=rng.choice([1, 2, 8, 16]),
                 pos=rng.randrange(0, 3000))
        return c
    B = _between(rng, 1, 128)
    heads = rng.choice([1, 4, 8, 16])
    if op == "prefix":
        c.update(dtype="bf16", B=B, T=rng.choice([1, 1, 1, 2]), heads=heads, group=rng.choice([1, 1, 2, 4]),
                 prefix=_between(rng, 100, 8000), length=_between(rng, 2, 300), ragged=True)
        return c
    c.update(B=B, T=rng.choice([1, 1, 2, 5]), heads=heads, group=rng.choice([1, 1, 2, 8]),
             length=_between(rng, 5, max(6, 120000 // B)), ragged=rng.random() < 0.7)
    return c


def _lengths(c):
    """The batch's cache lengths: even, or spread from a quarter of the longest up to it."""
    B, L, least = c["B"], c["length"], c["T"]
    if not c["ragged"] or B == 1:
        return [max(L, least)] * B
    return [max(least, int(round(L * (0.25 + 0.75 * i / (B - 1))))) for i in range(B)]


def _cache(g, fmt, pages, heads, page):
    """Codes and scales of a pool of pages, as rows of roughly normal values leave them."""
    code_type, top = CODES[fmt]
    kv = []
    for _ in range(2):
        x = torch.randn((pages, heads, page, D), generator=g, device="cuda", dtype=torch.float16) * (top / 3)
        x = x.clamp_(-top, top)
        kv.append((x.round_() if fmt == "int8" else x).to(code_type))
        kv.append(torch.exp(torch.randn((pages, heads, page), generator=g, device="cuda") * 0.2) * (3.0 / top))
    return dict(k=kv[0], k_scale=kv[1], v=kv[2], v_scale=kv[3])


def _tables(g, B, per_row, first=0, pages=None):
    """A page table [B, per_row] of a pool's pages in random order, from page `first` on."""
    order = torch.randperm((pages or first + B * per_row) - first, generator=g, device="cuda")[: B * per_row] + first
    return order.to(torch.int32).view(B, per_row)


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + 17)
    s = dict(case=c)
    if c["op"] in ("logprobs", "logprobs_grad"):
        N, V = c["N"], c["V"]
        # a peaked distribution over a noisy tail, as a language model's logits are
        x = torch.randn((N, V), generator=g, device="cuda") * 2.0
        hot = torch.randint(0, V, (N, 16), generator=g, device="cuda")
        x.scatter_add_(1, hot, torch.rand((N, 16), generator=g, device="cuda") * 12.0)
        s["logits"] = x.to(TYPES[c["dtype"]])
        s["targets"] = torch.where(torch.rand((N,), generator=g, device="cuda") < 0.7, hot[:, 0],
                                   torch.randint(0, V, (N,), generator=g, device="cuda")).to(torch.int32)
        if c["op"] == "logprobs_grad":
            # the statistics that the forward pass left, and the gradients that came back
            xf = s["logits"].float()
            s["lse"] = torch.logsumexp(xf, dim=1)
            p = torch.exp(xf - s["lse"][:, None])
            s["entropy"] = s["lse"] - (p * xf).sum(dim=1)
            s["d_log_prob"] = torch.randn((N,), generator=g, device="cuda")
            s["d_entropy"] = torch.randn((N,), generator=g, device="cuda") * 0.01
        return s
    B, T, heads, page = c["B"], c["T"], c["heads"], c["page"]
    if c["op"] == "update":
        last = c["pos"] + T + B  # each sequence starts one token behind the one before it
        per_row = -(-last // page)
        s.update(_cache(g, c["fmt"], B * per_row, heads, page))
        s["table"] = _tables(g, B, per_row)
        s["start"] = (torch.arange(B, device="cuda") + c["pos"]).to(torch.int32)
        for n in ("new_k", "new_v"):
            s[n] = (torch.randn((B, T, heads, D), generator=g, device="cuda") *
                    torch.exp(torch.randn((B, T, heads, 1), generator=g, device="cuda"))).to(TYPES[c["dtype"]])
        return s
    per_row = -(-max(_lengths(c)) // page)
    shared = -(-c["prefix"] // page) if c["op"] == "prefix" else 0
    pages = shared + B * per_row
    s.update(_cache(g, c["fmt"], pages, heads, page))
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    s["table"] = order[shared:].view(B, per_row).contiguous()
    if shared:
        s["prefix_pages"] = order[:shared].contiguous()
    lens = torch.tensor(_lengths(c), dtype=torch.int32, device="cuda")
    s["lens"] = lens[torch.randperm(B, generator=g, device="cuda")].contiguous()
    s["q"] = (torch.randn((B, T, heads * c["group"], D), generator=g, device="cuda") * 2.0).to(TYPES[c["dtype"]])
    return s


SCALE = 1.0 / math.sqrt(D)


def _own(s):
    import dirktensor_b200 as dt

    c = s["case"]
    op = c["op"]
    if op == "logprobs":
        r = dt.token_log_probs(s["logits"], s["targets"], top=c["top"])
        out = dict(log_prob=r.log_prob, entropy=r.entropy, lse=r.lse)
        return dict(out, top_ids=r.top_ids, top_log_probs=r.top_log_probs) if c["top"] else out
    if op == "logprobs_grad":
        return dt.token_log_probs_backward(s["logits"], s["targets"], s["lse"], s["entropy"], s["d_log_prob"], s["d_entropy"])
    cache = s.get("cache")
    if cache is None:  # a program keeps its cache object
        cache = s["cache"] = dt.KVCache.from_tensors(s["k"], s["v"], s["k_scale"], s["v_scale"])
    if op == "update":
        cache.append(s["new_k"], s["new_v"], s["table"], s["start"])
        return cache.read(s["table"], s["start"], c["T"], dtype=TYPES[c["out"]])
    if op == "attend":
        return dt.cache_attention_forward(s["q"], cache, s["table"], s["lens"], SCALE)
    return dt.prefix_attention_forward(s["q"], cache, s["prefix_pages"], c["prefix"], s["table"], s["lens"], SCALE)


def _quantised(x, fmt):
    code_type, top = CODES[fmt]
    amax = x.abs().amax(dim=-1, keepdim=True)
    some = amax >= TINY
    # the product is exact for bf16 values, and so a value half-way between two codes stays there
    y = torch.where(some, x * top / amax, torch.zeros_like(x))
    return (torch.round(y) if fmt == "int8" else y).to(code_type), torch.where(some, amax / top, torch.zeros_like(amax))[..., 0]


def _where(s, T):
    """Page and offset of the T tokens of each sequence from its start on."""
    page = s["case"]["page"]
    pos = s["start"].long()[:, None] + torch.arange(T, device="cuda")
    return torch.gather(s["table"].long(), 1, pos // page), pos % page


def _gathered(codes, scales, table):
    """The values of a page table's pages, [rows, heads, tokens, D] in 32 bits."""
    x = codes.view(torch.int8)[table.long()].view(codes.dtype).float() * scales[table.long()][..., None]
    rows, n, heads, page, _ = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(rows, heads, n * page, D)


def _visible(lens, T, L):
    """[B, T, L]: the keys that each query sees."""
    last = lens.long()[:, None] - T + 1 + torch.arange(T, device="cuda")
    return torch.arange(L, device="cuda")[None, None, :] < last[:, :, None]


def run(state):
    if own:
        return _own(state)
    s, c = state, state["case"]
    op = c["op"]
    if op in ("logprobs", "logprobs_grad"):
        x = s["logits"].float()
        t = s["targets"].long()[:, None]
        if op == "logprobs":
            m = x.amax(dim=1, keepdim=True)
            e = torch.exp(x - m)
            z = e.sum(dim=1, keepdim=True)
            lse = torch.log(z)
            out = dict(log_prob=(torch.gather(x, 1, t) - m - lse)[:, 0],
                       entropy=(lse - ((x - m) * e).sum(dim=1, keepdim=True) / z)[:, 0], lse=(m + lse)[:, 0])
            if c["top"]:
                v, i = torch.sort(x, dim=1, descending=True, stable=True)
                out["top_ids"] = i[:, : c["top"]].to(torch.int32)
                out["top_log_probs"] = v[:, : c["top"]] - m - lse
            return out
        lp = x - s["lse"][:, None]
        p = torch.exp(lp)
        g = -p * (s["d_log_prob"][:, None] + s["d_entropy"][:, None] * (lp + s["entropy"][:, None]))
        g = g.scatter_add(1, t, s["d_log_prob"][:, None])
        return g.to(x.dtype if c["dtype"] == "fp32" else TYPES[c["dtype"]])
    if op == "update":
        at, off = _where(s, c["T"])
        out = []
        for new, codes, scales in ((s["new_k"], s["k"], s["k_scale"]), (s["new_v"], s["v"], s["v_scale"])):
            q, sc = _quantised(new.float(), c["fmt"])
            codes.view(torch.int8)[at, :, off] = q.view(torch.int8)
            scales[at, :, off] = sc
            x = codes.view(torch.int8)[at, :, off].view(codes.dtype).float() * scales[at, :, off][..., None]
            out.append(x.to(TYPES[c["out"]]))
        return tuple(out)
    B, T, heads, group = c["B"], c["T"], c["heads"], c["group"]
    # queries of one K/V head side by side: [B, heads, T * group, D]
    q = s["q"].float().view(B, T, heads, group, D).permute(0, 2, 1, 3, 4).reshape(B, heads, T * group, D)
    k, v = _gathered(s["k"], s["k_scale"], s["table"]), _gathered(s["v"], s["v_scale"], s["table"])
    w = torch.matmul(q, k.transpose(2, 3)) * SCALE
    seen = _visible(s["lens"], T, k.shape[2]).repeat_interleave(group, dim=1)[:, None]
    w = w.masked_fill(~seen, float("-inf"))
    if op == "prefix":
        pages = s["prefix_pages"][None]
        pk, pv = (_gathered(s[n], s[n + "_scale"], pages)[0, :, : c["prefix"]] for n in ("k", "v"))
        rows = q.permute(1, 0, 2, 3).reshape(heads, B * T * group, D)
        pw = (torch.matmul(rows, pk.transpose(1, 2)) * SCALE).view(heads, B, T * group, -1).permute(1, 0, 2, 3)
        m = torch.maximum(w.amax(dim=-1, keepdim=True), pw.amax(dim=-1, keepdim=True))
        p, pp = torch.exp(w - m), torch.exp(pw - m)
        o = torch.matmul(p, v)
        o += torch.matmul(pp.permute(1, 0, 2, 3).reshape(heads, B * T * group, -1), pv).view(heads, B, T * group, D).permute(1, 0, 2, 3)
        o /= p.sum(dim=-1, keepdim=True) + pp.sum(dim=-1, keepdim=True)
    else:
        p = torch.exp(w - w.amax(dim=-1, keepdim=True))
        o = torch.matmul(p, v) / p.sum(dim=-1, keepdim=True)
    return o.view(B, heads, T, group, D).permute(0, 2, 1, 3, 4).reshape(B, T, heads * group, D).to(TYPES[c["dtype"]])


def work(case):
    c = case
    size = {"bf16": 2, "fp32": 4}
    if c["op"] in ("logprobs", "logprobs_grad"):
        n = c["N"] * c["V"]
        passes = 1 if c["op"] == "logprobs" else 2
        return {"bytes": n * size[c["dtype"]] * passes + c["N"] * 20, "flops": 5 * n}
    row = D + 4  # codes and scale of one token and head
    if c["op"] == "update":
        n = 2 * c["B"] * c["T"] * c["heads"]
        return {"bytes": n * (D * size[c["dtype"]] + 2 * row + D * size[c["out"]]), "flops": 4 * n * D}
    keys, queries = sum(_lengths(c)), c["T"] * c["heads"] * c["group"]
    extra = c.get("prefix", 0)
    return {"bytes": 2 * (keys + extra) * c["heads"] * row + 2 * c["B"] * queries * D * size[c["dtype"]],
            "flops": 4 * D * queries * (keys + c["B"] * extra)}


def _pool_rows(codes, scales, pages, head, upto):
    """The first `upto` rows of one head along a list of pages, in 64 bits."""
    x = codes.view(torch.int8)[pages, head].view(codes.dtype).double() * scales[pages, head].double()[..., None]
    return x.reshape(-1, D)[:upto]


def exact(case, seed):
    c = case
    s = prepare(case, seed)
    if c["op"] in ("logprobs", "logprobs_grad"):
        got = dict(log_prob=[], entropy=[], lse=[], top_log_probs=[])
        grads = []
        for at in range(0, c["N"], 64):
            x = s["logits"][at:at + 64].double()
            lp = torch.log_softmax(x, dim=1)
            t = s["targets"][at:at + 64].long()
            rows = torch.arange(len(t), device="cuda")
            if c["op"] == "logprobs":
                got["log_prob"].append(lp[rows, t])
                got["entropy"].append(-(torch.exp(lp) * lp).sum(1))
                got["lse"].append(torch.logsumexp(x, dim=1))
                got["top_log_probs"].append(torch.topk(lp, max(1, c["top"]), dim=1).values)
            else:  # by automatic differentiation of the definition
                x.requires_grad_(True)
                with torch.enable_grad():
                    lp = torch.log_softmax(x, dim=1)
                    h = -(torch.exp(lp) * lp).sum(1)
                    total = (lp[rows, t] * s["d_log_prob"][at:at + 64].double()).sum() + (h * s["d_entropy"][at:at + 64].double()).sum()
                    grads.append(torch.autograd.grad(total, x)[0].float())
        if c["op"] == "logprobs_grad":
            return torch.cat(grads)
        out = {n: torch.cat(v) for n, v in got.items()}
        if not c["top"]:
            del out["top_log_probs"]
        else:
            out["top_ids"] = None
        return out
    if c["op"] == "update":
        out = []
        for x in (s["new_k"], s["new_v"]):
            x = x.double()
            most, top = x.abs().amax(dim=-1, keepdim=True), CODES[c["fmt"]][1]
            y = x * top / most
            if c["fmt"] == "int8":
                y = torch.round(y)
            else:  # three bits behind the leading one, down to 2^-9
                e = torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -40))).clamp_min(-6.0)
                y = torch.round(y * torch.exp2(3 - e)) * torch.exp2(e - 3)
            out.append((y * most / top).to(torch.float32 if y.numel() > 2 ** 26 else torch.float64))
        return tuple(out)
    B, T, heads, group = c["B"], c["T"], c["heads"], c["group"]
    q = s["q"].double()
    out = torch.zeros((B, T, heads * group, D), dtype=torch.float64, device="cuda")
    lens = s["lens"].tolist()
    for h in range(heads):
        mine = slice(h * group, (h + 1) * group)
        if c["op"] == "prefix":
            shared = [_pool_rows(s[n], s[n + "_scale"], s["prefix_pages"].long(), h, c["prefix"]) for n in ("k", "v")]
        for b in range(B):
            k, v = (_pool_rows(s[n], s[n + "_scale"], s["table"][b].long(), h, lens[b]) for n in ("k", "v"))
            hidden = 0
            if c["op"] == "prefix":
                k, v, hidden = torch.cat((shared[0], k)), torch.cat((shared[1], v)), c["prefix"]
            for t in range(T):
                n = hidden + lens[b] - T + t + 1
                w = torch.softmax(q[b, t, mine] @ k[:n].T * SCALE, dim=-1)
                out[b, t, mine] = w @ v[:n]
    return out
