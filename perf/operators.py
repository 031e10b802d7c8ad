"""The operators of one serving step over a paged 16-bit KV cache, measured on real step shapes.

plan (page allocation, block tables, slot maps) -> qk (q/k norms, rotary positions, cache write)
-> attention (new tokens of every request over its pages) -> verify (drafted tokens against the
target's probabilities).  Head layouts and vocabularies are those of the Qwen2.5-0.5B,
Llama-3.2-1B, Llama-3-8B and OLMoE configurations.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
# q heads, kv heads, head_dim
HEADS = {"qwen2.5-0.5b": (14, 2, 64), "llama3.2-1b": (32, 8, 64), "llama3-8b": (32, 8, 128), "olmoe": (16, 16, 128)}
VOCABS = (50304, 128256, 151936)


# ---------------------------------------------------------------- cases

def _attention(name=None, model="llama3-8b", dtype="bf16", page=64, requests=1, ctx=(0, 0), new=(1, 1), chunk_every=1,
               window=0, softcap=0.0, alibi=False, lengths=1):
    c = {"op": "attention", "model": model, "dtype": dtype, "page": page, "requests": requests, "ctx_lo": ctx[0],
         "ctx_hi": ctx[1], "new_lo": new[0], "new_hi": new[1], "chunk_every": chunk_every, "window": window,
         "softcap": softcap, "alibi": alibi, "lengths": lengths}
    return dict(c, name=name) if name else c


def _qk(name=None, model="llama3-8b", dtype="bf16", page=64, tokens=1, norm="head", interleaved=False, rotary=1.0,
        far=4096):
    c = {"op": "qk", "model": model, "dtype": dtype, "page": page, "tokens": tokens, "norm": norm,
         "interleaved": interleaved, "rotary": rotary, "far": far}
    return dict(c, name=name) if name else c


def _plan(name=None, requests=16, page=64, ctx=(0, 4096), new=(1, 1), chunk_every=1, lengths=1):
    c = {"op": "plan", "requests": requests, "page": page, "ctx_lo": ctx[0], "ctx_hi": ctx[1], "new_lo": new[0],
         "new_hi": new[1], "chunk_every": chunk_every, "lengths": lengths}
    return dict(c, name=name) if name else c


def _verify(name=None, requests=4, drafts=(1, 4), vocab=128256, one_hot=False, lengths=1):
    c = {"op": "verify", "requests": requests, "new_lo": drafts[0] + 1, "new_hi": drafts[1] + 1, "vocab": vocab,
         "one_hot": one_hot, "lengths": lengths}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one chat sequence, one token a step: latency
        _attention("attention, one sequence", requests=1, ctx=(575, 575), lengths=1),
        # a full decode batch of long documents: the cache's bandwidth
        _attention("attention, long decode", requests=16, ctx=(24000, 32767), lengths=2),
        # four drafted tokens and the last accepted one, odd group of seven heads
        _attention("attention, drafts", model="qwen2.5-0.5b", dtype="fp16", page=16, requests=48, ctx=(200, 4000),
                   new=(5, 5), lengths=3),
        # the second half of a long prompt
        _attention("attention, prompt chunk", requests=1, ctx=(4096, 4096), new=(4096, 4096), lengths=4),
        # chunks of prompts among decoding requests, capped scores and a sliding window
        _attention("attention, mixed window", model="llama3.2-1b", dtype="bf16", page=32, requests=16, ctx=(100, 5000),
                   new=(100, 700), chunk_every=4, window=1024, softcap=50.0, lengths=5),
        # one decode batch, norm over the whole row
        _qk("qk, decode batch", model="olmoe", tokens=16, norm="row"),
        # an odd prompt chunk, half of each head rotated in interleaved pairs, far positions
        _qk("qk, ragged chunk", model="qwen2.5-0.5b", dtype="fp16", page=16, tokens=777, interleaved=True, rotary=0.5,
            far=131072),
        # a long chunk
        _qk("qk, long chunk", tokens=16384, far=32768),
        # a decode step of a small server
        _plan("plan, decode", requests=16, ctx=(0, 4096)),
        # a step of a big one: prompts arriving among decoding requests
        _plan("plan, arrivals", requests=1024, page=16, ctx=(0, 16384), new=(16, 1024), chunk_every=8, lengths=2),
        # prompt-lookup drafts of a few sequences
        _verify("verify, lookup", requests=4, drafts=(0, 4), vocab=50304, one_hot=True),
        # a batch with a draft model
        _verify("verify, batch", requests=64, drafts=(1, 5), vocab=151936, lengths=2),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(max(lo, 1)), math.log(max(hi, 1) + 0.49)))))))


def draw(rng):
    op = rng.choice(["attention"] * 5 + ["qk"] * 2 + ["plan"] + ["verify"] * 2)
    lengths = rng.randrange(1 << 20)
    if op == "qk":
        return _qk(None, rng.choice(list(HEADS)), rng.choice(list(DTYPES)), rng.choice([16, 32, 64, 128]),
                   _spread(rng, 1, 16000), rng.choice(["head", "row", "none"]), rng.random() < 0.4,
                   rng.choice([1.0, 1.0, 0.5]), _spread(rng, 64, 1 << 20))
    if op == "plan":
        return _plan(None, _spread(rng, 1, 1000), rng.choice([16, 32, 64, 128]), (0, _spread(rng, 16, 16000)),
                     (1, _spread(rng, 1, 1000)), rng.choice([1, 2, 8]), lengths)
    if op == "verify":
        lo = rng.randrange(0, 3)
        return _verify(None, _spread(rng, 1, 60), (lo, lo + rng.randrange(0, 4)), rng.choice(VOCABS + (32003,)),
                       rng.random() < 0.4, lengths)
    most = listed()[3]
    most_bytes, most_flops = work(listed()[1])["bytes"], work(most)["flops"]
    while True:
        kind = rng.choice(["decode", "drafts", "chunk", "mixed"])
        model, dtype, page = rng.choice(list(HEADS)), rng.choice(list(DTYPES)), rng.choice([16, 32, 64, 128])
        window = rng.choice([0, 0, 0, _spread(rng, 64, 4096)])
        softcap = rng.choice([0.0, 0.0, 30.0])
        alibi = rng.random() < 0.2
        if kind in ("decode", "drafts"):
            n = 1 if kind == "decode" else rng.randrange(2, 9)
            hi = _spread(rng, 16, 32000)
            c = _attention(None, model, dtype, page, _spread(rng, 1, 64), (rng.randrange(0, hi), hi), (n, n), 1, window,
                           softcap, alibi, lengths)
        elif kind == "chunk":
            lo = _spread(rng, 16, 4000)
            c = _attention(None, model, dtype, page, _spread(rng, 1, 8), (0, _spread(rng, 16, 8000)),
                           (lo, _spread(rng, lo, 4000)), 1, window, softcap, alibi, lengths)
        else:
            c = _attention(None, model, dtype, page, rng.randrange(4, 40), (0, _spread(rng, 100, 8000)),
                           (16, _spread(rng, 64, 1000)), rng.randrange(2, 8), window, softcap, alibi, lengths)
        w = work(c)
        hq, hk, d = HEADS[model]
        ctx, new = _lengths(c)
        far = max(a + b for a, b in zip(ctx, new))
        padded = len(ctx) * 4 * max(hq * max(new) * far, 2 * hk * far * d)
        if w["bytes"] <= most_bytes and w["flops"] <= most_flops and padded <= 4.5e9:
            return c


def _lengths(case):
    """Context and new tokens of every request: the new ones of each chunk_every-th from the range, 1 for the others."""
    rng = random.Random(case["lengths"])
    n = case["requests"]
    ctx = [_spread(rng, case["ctx_lo"], case["ctx_hi"]) if case["ctx_hi"] else 0 for _ in range(n)] if "ctx_hi" in case else [0] * n
    new = [_spread(rng, case["new_lo"], case["new_hi"]) if i % case.get("chunk_every", 1) == 0 else 1 for i in range(n)]
    return ctx, new


def _pages(tokens, page):
    return -(-tokens // page)


def _visible(ctx, new, window):
    """How many keys the new tokens of one request see, over all of them."""
    w = window or ctx + new
    full = max(0, min(new, w - ctx))  # tokens that see everything before them
    return full * ctx + full * (full + 1) // 2 + (new - full) * w


def _kept(ctx, new, window):
    """Keys of one request that any of its new tokens sees."""
    return ctx + new - (max(0, ctx + 1 - window) if window else 0)


def work(case):
    op = case["op"]
    if op == "attention":
        hq, hk, d = HEADS[case["model"]]
        pairs = list(zip(*_lengths(case)))
        keys = sum(_kept(c, n, case["window"]) for c, n in pairs)
        seen = sum(_visible(c, n, case["window"]) for c, n in pairs)
        t = sum(n for _, n in pairs)
        return {"bytes": 4 * keys * hk * d + 4 * t * hq * d + 4 * t * hq, "flops": 4 * d * hq * seen}
    if op == "qk":
        hq, hk, d = HEADS[case["model"]]
        return {"bytes": 4 * case["tokens"] * (hq + 2 * hk) * d + 8 * case["tokens"],
                "flops": 10 * case["tokens"] * (hq + hk) * d}
    ctx, new = _lengths(case)
    if op == "plan":
        taken = sum(_pages(c + n, case["page"]) - _pages(c, case["page"]) for c, n in zip(ctx, new))
        return {"bytes": 12 * len(ctx) + 8 * taken + 16 * len(ctx) + 8 * sum(new), "flops": 10 * sum(new)}
    rows = len(ctx) if case["one_hot"] else 2 * len(ctx)
    return {"bytes": 4 * rows * case["vocab"] + 16 * sum(new), "flops": 2 * rows * case["vocab"]}


# ---------------------------------------------------------------- inputs

def _ints(values, device="cuda"):
    return torch.tensor(values, dtype=torch.int32, device=device)


def _tables(ctx, new, page, g, extra=8):
    """Block tables over scattered pages (unused entries -1) and the number of pages."""
    need = [_pages(c + n, page) for c, n in zip(ctx, new)]
    total = sum(need) + extra
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    width = max(max(need), 1)
    at = torch.arange(width, device="cuda")[None, :]
    many = torch.tensor(need, device="cuda")[:, None]
    first = torch.cumsum(many, 0) - many
    return torch.where(at < many, order[(first + at).clamp(max=total - 1)], -1).to(torch.int32).contiguous(), total


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape, dtype=torch.float32: torch.randn(shape, generator=g, device="cuda", dtype=dtype)  # noqa: E731
    op = case["op"]
    s = {"case": case, "op": op}
    if op in ("attention", "qk"):
        hq, hk, d = HEADS[case["model"]]
        dtype, page = DTYPES[case["dtype"]], case["page"]
    if op == "attention":
        ctx, new = _lengths(case)
        table, total = _tables(ctx, new, page, g)
        t = sum(new)
        s["q"] = (normal(t, hq, d) * 1.5).to(dtype)
        s["k_cache"] = normal(total, hk, page, d, dtype=dtype)
        s["v_cache"] = normal(total, hk, page, d, dtype=dtype)
        # keys of a trained model have a few channels much larger than the rest
        s["k_cache"][..., :: d // 4] *= 3
        s["table"] = table
        s["cu_new"] = _ints([sum(new[:i]) for i in range(len(new) + 1)])
        s["seq_len"] = _ints([c + n for c, n in zip(ctx, new)])
        s["max_new"] = max(new)
        s["max_len"] = max(c + n for c, n in zip(ctx, new))
        s["slopes"] = torch.tensor([2.0 ** (-8.0 * (i + 1) / hq) for i in range(hq)], device="cuda") if case["alibi"] else None
        if own:
            from vvli_b200.paged import PagedAttention

            s["attention"] = PagedAttention(hq, hk, d, page, dtype=dtype, softcap=case["softcap"], window=case["window"],
                                            alibi=s["slopes"])
    elif op == "qk":
        t = case["tokens"]
        qkv = normal(t, (hq + 2 * hk) * d)
        qkv[:, :: d // 4] *= 4
        qkv = qkv.to(dtype)  # the rows of a fused projection
        s["q"] = qkv[:, : hq * d].view(t, hq, d)
        s["k"] = qkv[:, hq * d : (hq + hk) * d].view(t, hk, d)
        s["v"] = qkv[:, (hq + hk) * d :].view(t, hk, d)
        total = _pages(t, page) + 4
        s["k_cache"] = normal(total, hk, page, d, dtype=dtype)
        s["v_cache"] = normal(total, hk, page, d, dtype=dtype)
        s["slots"] = torch.randperm(total * page, generator=g, device="cuda")[:t].to(torch.int32)
        s["positions"] = torch.randint(0, case["far"], (t,), generator=g, device="cuda").to(torch.int32)
        half = int(d * case["rotary"]) // 2
        s["inv_freq"] = 500000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
        spans = (hq * d, hk * d) if case["norm"] == "row" else (d, d)
        s["weights"] = [None if case["norm"] == "none" else (1 + 0.2 * normal(n)).to(dtype) for n in spans]
    elif op == "plan":
        ctx, new = _lengths(case)
        owned = [_pages(c, case["page"]) for c in ctx]
        need = sum(_pages(c + n, case["page"]) - o for c, n, o in zip(ctx, new, owned))
        total = sum(owned) + need + need // 4 + 4
        order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
        width = max(_pages(c + n, case["page"]) for c, n in zip(ctx, new)) + 2
        at = torch.arange(width, device="cuda")[None, :]
        many = torch.tensor(owned, device="cuda")[:, None]
        first = torch.cumsum(many, 0) - many
        s["table"] = torch.where(at < many, order[(first + at).clamp(max=total - 1)], -1).to(torch.int32).contiguous()
        s["free_pages"] = order[sum(owned) :].contiguous()
        s["free_count"] = _ints([total - sum(owned)])
        s["context"], s["new"], s["owned"] = _ints(ctx), _ints(new), _ints(owned)
        s["tokens"] = sum(new)
    else:
        _, new = _lengths(case)
        t, v = sum(new), case["vocab"]
        logits = normal(t, v) * 3
        s["target"] = torch.softmax(logits, -1)
        s["draft"] = None if case["one_hot"] else torch.softmax(logits + normal(t, v), -1)
        drawn = torch.multinomial(s["target"] if s["draft"] is None else s["draft"], 1, generator=g)[:, 0]
        # row r holds the token it was fed; the draft made after row r is fed to row r + 1
        s["tokens"] = torch.roll(drawn, 1).to(torch.int32)
        s["cu_rows"] = _ints([sum(new[:i]) for i in range(len(new) + 1)])
        s["u_accept"] = torch.rand(t, generator=g, device="cuda")
        s["u_sample"] = torch.rand(len(new), generator=g, device="cuda")
    return s


# ---------------------------------------------------------------- one pass

def run(s):
    op, case = s["op"], s["case"]
    if own:
        if op == "attention":
            return s["attention"](s["q"], s["k_cache"], s["v_cache"], s["table"], s["cu_new"], s["seq_len"], s["max_new"],
                                  lse=True)
        if op == "qk":
            from vvli_b200.paged import qk_norm_rope_write

            q = qk_norm_rope_write(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], s["positions"],
                                   s["inv_freq"], s["weights"][0], s["weights"][1], norm=case["norm"],
                                   interleaved=case["interleaved"])
            return q, s["k_cache"], s["v_cache"]
        if op == "plan":
            from vvli_b200.paged import plan_step

            p = plan_step(s["context"], s["new"], s["owned"], s["table"], s["free_pages"], s["free_count"], case["page"],
                          s["tokens"])
            return p.cu_new, p.seq_len, p.positions, p.slots, p.owned, p.free_count, p.status, s["table"]
        from vvli_b200.speculative import verify_drafts

        return verify_drafts(s["target"], s["draft"], s["tokens"], s["cu_rows"], s["u_accept"], s["u_sample"])
    return {"attention": _plain_attention, "qk": _plain_qk, "plan": _plain_plan, "verify": _plain_verify}[op](s)


def _rows(cu, total):
    """Request and place in it of every row."""
    row = torch.arange(total, device=cu.device)
    b = torch.searchsorted(cu[1:].long().contiguous(), row, right=True)
    return b, row - cu.long()[b]


def _plain_attention(s):
    case = s["case"]
    q, table = s["q"], s["table"]
    hq, hk, d = HEADS[case["model"]]
    page, n, length = case["page"], s["max_new"], s["max_len"]
    t, requests = q.shape[0], table.shape[0]
    b, i = _rows(s["cu_new"], t)
    padded = torch.zeros(requests, n, hq, d, device=q.device)
    padded[b, i] = q.float()
    padded = padded.view(requests, n, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(requests, hk, hq // hk * n, d)
    used = table[:, : _pages(length, page)].long().clamp(min=0)
    k = s["k_cache"][used].permute(0, 2, 1, 3, 4).reshape(requests, hk, -1, d).float()
    scores = torch.matmul(padded, k.transpose(-1, -2)).view(requests, hk, hq // hk, n, -1).mul_(1 / math.sqrt(d))
    del k
    if case["softcap"]:
        scores = torch.tanh(scores / case["softcap"]) * case["softcap"]
    new = (s["cu_new"][1:] - s["cu_new"][:-1]).long()
    at = (s["seq_len"].long() - new)[:, None] + torch.arange(n, device=q.device)  # position of every row
    key = torch.arange(scores.shape[-1], device=q.device)
    far = key[None, None, :] - at[:, :, None]
    if s["slopes"] is not None:
        scores = scores + s["slopes"].view(1, hk, hq // hk, 1, 1) * far[:, None, None].float()
    hidden = far > 0
    if case["window"]:
        hidden = hidden | (far <= -case["window"])
    scores.masked_fill_(hidden[:, None, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    scores.sub_(top).exp_()
    total = scores.sum(-1, keepdim=True)
    v = s["v_cache"][used].permute(0, 2, 1, 3, 4).reshape(requests, hk, -1, d).float()
    out = torch.matmul(scores.view(requests, hk, hq // hk * n, -1), v).view(requests, hk, hq // hk, n, d) / total
    lse = top + total.log()
    out = out.permute(0, 3, 1, 2, 4).reshape(requests, n, hq, d)[b, i]
    lse = lse.permute(0, 3, 1, 2, 4).reshape(requests, n, hq)[b, i]
    return out.to(q.dtype), lse


def _plain_qk(s):
    case = s["case"]
    angle = s["positions"].double()[:, None] * s["inv_freq"]
    cos, sin = angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]
    half = s["inv_freq"].numel()

    def turned(x, weight):
        t, h, d = x.shape
        y = x.float()
        if case["norm"] == "head":
            y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * weight.float()
        elif case["norm"] == "row":
            y = y.reshape(t, -1)
            y = (y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * weight.float()).view(t, h, d)
        r = y[..., : 2 * half]
        if case["interleaved"]:
            a, b = r[..., 0::2], r[..., 1::2]
            r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = r[..., :half], r[..., half:]
            r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([r, y[..., 2 * half :]], -1).to(x.dtype)

    q, k = turned(s["q"], s["weights"][0]), turned(s["k"], s["weights"][1])
    slot = s["slots"].long()
    place, off = slot // case["page"], slot % case["page"]
    s["k_cache"][place, :, off] = k
    s["v_cache"][place, :, off] = s["v"]
    return q, s["k_cache"], s["v_cache"]


def _plain_plan(s):
    page, table = s["case"]["page"], s["table"]
    context, new, owned = s["context"].long(), s["new"].long(), s["owned"].long()
    free = s["free_count"].long()
    zero = torch.zeros(1, dtype=torch.long, device=table.device)
    cu = torch.cat([zero, torch.cumsum(new, 0)])
    need = ((context + new + page - 1) // page - owned).clamp(min=0)
    upto = torch.cumsum(need, 0)
    fits = (need == 0) | (upto <= free)
    need = torch.where(fits, need, 0)
    at = torch.arange(table.shape[1], device=table.device)[None, :]
    nth = at - owned[:, None]
    take = (nth >= 0) & (nth < need[:, None])
    source = free - 1 - ((upto - need)[:, None] + nth)
    table.copy_(torch.where(take, s["free_pages"][source.clamp(0, s["free_pages"].numel() - 1)], table))
    b, i = _rows(cu, s["tokens"])
    position = context[b] + i
    slots = table[b, position // page].long() * page + position % page
    slots = torch.where(fits[b], slots, -1)
    small = lambda x: x.to(torch.int32)  # noqa: E731
    return (small(cu), small(torch.where(fits, context + new, 0)), small(position), small(slots), small(owned + need),
            small(free - need.sum()), small(~fits), table)


def _plain_verify(s):
    target, draft, cu = s["target"], s["draft"], s["cu_rows"].long()
    t, v = target.shape
    b, i = _rows(cu, t)
    last = cu[1:] - 1
    row = torch.arange(t, device=target.device)
    fed = torch.roll(s["tokens"].long(), -1)  # the draft that row r has to judge
    p = target.gather(1, fed[:, None])[:, 0].double()
    q = torch.ones_like(p) if draft is None else draft.gather(1, fed[:, None])[:, 0].double()
    taken = (s["u_accept"].double() * q < p) & (row != last[b])
    # rows before the first one that is not taken
    stop = torch.where(taken, t, i)
    accepted = torch.full((cu.numel() - 1,), t, dtype=torch.long, device=target.device).scatter_reduce(0, b, stop, "amin")
    at = cu[:-1] + accepted
    weight = target[at].double()
    drafted = at != last
    if draft is None:
        weight.scatter_(1, fed[at][:, None], torch.where(drafted, 0.0, weight.gather(1, fed[at][:, None])[:, 0])[:, None])
    else:
        weight = torch.where(drafted[:, None], (weight - draft[at].double()).clamp(min=0), weight)
    total = torch.cumsum(weight, -1)
    above = total > s["u_sample"].double()[:, None] * total[:, -1:]
    token = above.to(torch.int8).argmax(-1)
    out = torch.where(i < accepted[b], fed, -1)
    out[at] = token
    return accepted.to(torch.int32), out.to(torch.int32)


# ---------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        hq, hk, d = HEADS[case["model"]]
        cu, ends, page = s["cu_new"].tolist(), s["seq_len"].tolist(), case["page"]
        out = torch.zeros(cu[-1], hq, d, dtype=torch.float64, device="cuda")
        lse = torch.zeros(cu[-1], hq, dtype=torch.float64, device="cuda")
        for b, end in enumerate(ends):
            lo, hi = cu[b], cu[b + 1]
            pages = s["table"][b, : _pages(end, page)].long()
            pos = torch.arange(end - (hi - lo), end, device="cuda")[:, None]
            key = torch.arange(end, device="cuda")[None, :]
            seen = key <= pos
            if case["window"]:
                seen &= key > pos - case["window"]
            for h in range(hk):
                k = s["k_cache"][pages, h].reshape(-1, d)[:end].double()
                v = s["v_cache"][pages, h].reshape(-1, d)[:end].double()
                for j in range(h * (hq // hk), (h + 1) * (hq // hk)):
                    x = s["q"][lo:hi, j].double() @ k.T / math.sqrt(d)
                    if case["softcap"]:
                        x = case["softcap"] * torch.tanh(x / case["softcap"])
                    if case["alibi"]:
                        x = x + s["slopes"][j].double() * (key - pos)
                    x = x.masked_fill(~seen, float("-inf"))
                    lse[lo:hi, j] = torch.logsumexp(x, -1)
                    out[lo:hi, j] = torch.exp(x - lse[lo:hi, j, None]) @ v
        return out, lse
    if case["op"] == "qk":
        freq, pos, slots = s["inv_freq"], s["positions"].double(), s["slots"].long()
        results = []
        for x, w in ((s["q"], s["weights"][0]), (s["k"], s["weights"][1])):
            y = x.double().clone()
            dims = (1, 2) if case["norm"] == "row" else (2,)
            if case["norm"] != "none":
                y = y / torch.sqrt(torch.mean(y * y, dim=dims, keepdim=True) + 1e-6)
                y = y * (w.double().view(1, *x.shape[1:]) if case["norm"] == "row" else w.double())
            for f in range(freq.numel()):
                a, b = (2 * f, 2 * f + 1) if case["interleaved"] else (f, f + freq.numel())
                turn = torch.polar(torch.ones_like(pos), pos * freq[f])[:, None] * torch.complex(y[..., a], y[..., b])
                y[..., a], y[..., b] = turn.real, turn.imag
            results.append(y)
        caches = []
        for cache, rows in ((s["k_cache"], results[1]), (s["v_cache"], s["v"].double())):
            c = cache.double().transpose(1, 2).reshape(-1, cache.shape[1], cache.shape[3])
            c[slots] = rows
            caches.append(c.view(cache.shape[0], cache.shape[2], cache.shape[1], cache.shape[3]).transpose(1, 2))
        return results[0], caches[0], caches[1]
    return None
