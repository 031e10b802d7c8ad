"""The paged operators together: speculative decoding steps of a one-layer model, with page plans, rejected
drafts and requests that come and go, against the dense computation in 64 bits.  Needs a B200."""

import math

import pytest

import paged_ref as ref

pytestmark = pytest.mark.gpu

HQ, HK, D, H, V, PAGE = 8, 2, 64, 128, 97, 16


class Model:
    """Embedding, one attention layer with q / k norms and rotation, and an LM head, in bf16 weights."""

    def __init__(self, torch):
        g = torch.Generator().manual_seed(7)
        rnd = lambda *s: (torch.randn(*s, generator=g) / math.sqrt(s[-1])).to(torch.bfloat16)  # noqa: E731
        self.embed = torch.randn(V, H, generator=g).to(torch.bfloat16)
        self.wqkv, self.wo, self.head = rnd((HQ + 2 * HK) * D, H), rnd(H, HQ * D), rnd(V, H) * 3
        self.qn, self.kn = ((1 + 0.2 * torch.randn(D, generator=g)).to(torch.bfloat16) for _ in range(2))
        self.freq = 10000.0 ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))

    def dense(self, torch, tokens):
        """Attention rows and probabilities of every position of one token list, in 64 bits."""
        x = self.embed[tokens].double()
        qkv = x @ self.wqkv.double().T
        n, pos = len(tokens), torch.arange(len(tokens))
        q, k, v = (qkv[:, a * D:b * D].view(n, b - a, D) for a, b in ((0, HQ), (HQ, HQ + HK), (HQ + HK, HQ + 2 * HK)))
        q = ref.qk_rows(q, self.qn, "head", 1e-6, pos, self.freq, False)
        k = ref.qk_rows(k, self.kn, "head", 1e-6, pos, self.freq, False)
        k, v = (y.repeat_interleave(HQ // HK, 1) for y in (k, v))
        s = torch.einsum("qhd,khd->hqk", q, k) / math.sqrt(D)
        s = s.masked_fill(pos[None, None, :] > pos[None, :, None], -math.inf)
        a = torch.einsum("hqk,khd->qhd", torch.softmax(s, -1), v)
        return a, torch.softmax((x + a.reshape(n, -1) @ self.wo.double().T) @ self.head.double().T, -1)


def test_speculative_steps():
    import torch
    from vvli_b200.paged import PagedAttention, plan_step, qk_norm_rope_write
    from vvli_b200.speculative import verify_drafts
    m = Model(torch)
    dev = {n: getattr(m, n).cuda() for n in ("embed", "wqkv", "wo", "head", "qn", "kn", "freq")}
    g = torch.Generator().manual_seed(11)
    B, pages, width, rows = 6, 40, 12, 256  # rows: the prompts (217 tokens) and 4 drafts each
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    caches = [torch.full((pages, HK, PAGE, D), math.nan, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    free = ints(torch.randperm(pages, generator=g).tolist())
    count, owned, table = ints([pages]), ints([0] * B), ints([[-1] * width] * B)
    attention = PagedAttention(HQ, HK, D, PAGE)
    history = [torch.randint(0, V, (n,), generator=g).tolist() for n in (1, 30, 64, 17, 5, 100)]  # prompts
    cached = [0] * B
    accepted_ever = rejected_ever = 0
    for step in range(7):
        if step == 4:  # request 2 ends: its pages go back on the stack, and another takes its place
            n, c = int(owned[2]), int(count)
            free[c:c + n] = table[2, :n]
            count += n
            owned[2], cached[2], history[2] = 0, 0, torch.randint(0, V, (40,), generator=g).tolist()
        # every request feeds what is not cached yet (a prompt, or the token drawn last) and up to 4 drafts
        fed = [h[c:] for h, c in zip(history, cached)]
        drafts = [torch.randint(0, V, (int(torch.randint(0, 5, (1,), generator=g)),), generator=g).tolist() for _ in fed]
        exact = [m.dense(torch, h + d) for h, d in zip(history, drafts)]
        for b, d in enumerate(drafts):  # some drafts that the target likes
            if d and step % 2:
                d[0] = int(exact[b][1][len(history[b]) - 1].argmax())
        exact = [m.dense(torch, h + d) for h, d in zip(history, drafts)]
        new = [len(f) + len(d) for f, d in zip(fed, drafts)]
        tokens = sum((f + d for f, d in zip(fed, drafts)), [])
        T = len(tokens)
        plan = plan_step(ints(cached), ints(new), owned, table, free, count, PAGE, rows, inplace=True)
        assert plan.status.tolist() == [0] * B and int(plan.cu_new[-1]) == T
        x = torch.zeros(rows, H, dtype=torch.bfloat16, device="cuda")
        x[:T] = dev["embed"][torch.tensor(tokens, device="cuda")]
        qkv = x @ dev["wqkv"].T
        q, k, v = (qkv[:, a * D:b * D].view(rows, b - a, D) for a, b in ((0, HQ), (HQ, HQ + HK), (HQ + HK, HQ + 2 * HK)))
        q = qk_norm_rope_write(q, k, v, *caches, plan.slots, plan.positions, dev["freq"], dev["qn"], dev["kn"])
        out = attention(q, *caches, table, plan.cu_new, plan.seq_len, max(new))[:T]
        probs = torch.softmax((x[:T].float() + out.reshape(T, -1).float() @ dev["wo"].float().T) @ dev["head"].float().T, -1)
        # q, k, v are rounded to bf16 twice (projection, norm), the probabilities and the output once: each
        # half a step (2^-8) of its value, which the softmax of scores of about 1 passes on about once
        want = torch.cat([a[-n:] for (a, _), n in zip(exact, new)])
        assert float((out.cpu().double() - want).norm() / want.norm()) < 6 * 2.0**-8
        # verification of the drafts: row r of request b is judged from the last fed token on
        starts = plan.cu_new.tolist()
        judged = [r for b in range(B) for r in range(starts[b] + len(fed[b]) - 1, starts[b + 1])]
        cu = [0]
        for d in drafts:
            cu.append(cu[-1] + len(d) + 1)
        target = probs[torch.tensor(judged, device="cuda")].contiguous()
        want_p = torch.cat([p[-(len(d) + 1):] for (_, p), d in zip(exact, drafts)])
        assert float((target.cpu().double() - want_p).abs().max()) < 0.05
        toks = ints([tokens[r] for r in judged])
        ua, us = torch.rand(len(judged), generator=g), torch.rand(B, generator=g)
        acc, emitted = verify_drafts(target, None, toks, ints(cu), ua.cuda(), us.cuda())
        want_acc, want_out = ref.verify(target.cpu(), None, toks.cpu(), cu, ua, us)
        assert acc.tolist() == want_acc and emitted.tolist() == want_out
        for b in range(B):
            n = want_acc[b]
            cached[b] = len(history[b]) + n  # rejected drafts' slots and pages are simply used again
            history[b] = history[b] + want_out[cu[b]:cu[b] + n + 1]
            accepted_ever += n
            rejected_ever += len(drafts[b]) - n
    assert accepted_ever > 3 and rejected_ever > 3 and attention.status() == 0


def test_rows_to_judge_of_a_mixed_step():
    # A decode token with drafts, a prompt's end with and without drafts, the middle of a prompt, a request that feeds
    # nothing, and one that gets no pages: only rows from the last known token on are judged, of those that want a token.
    import torch
    from vvli_b200.paged import PagedAttention, plan_step, qk_norm_rope_write
    from vvli_b200.speculative import verify_drafts
    m = Model(torch)
    dev = {n: getattr(m, n).cuda() for n in ("embed", "wqkv", "wo", "head", "qn", "kn", "freq")}
    g = torch.Generator().manual_seed(21)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    history = [torch.randint(0, V, (n,), generator=g).tolist() for n in (20, 33, 50, 40, 5, 90)]
    known, drafts = [1, 33, 30, 25, 0, 90], [3, 0, 2, 0, 0, 1]  # fed tokens before the drafts, and drafts
    want_token = [True, True, True, False, False, True]       # request 3 has more of its prompt to come
    B, rows, pages, width = len(history), 256, 13, 8          # the first five take 2 + 3 + 4 + 3 + 1 pages: none is left
    cached = [len(h) - k for h, k in zip(history, known)]
    fed = [h[len(h) - k:] + torch.randint(0, V, (n,), generator=g).tolist() for h, k, n in zip(history, known, drafts)]
    table = torch.full((B, width), -1, dtype=torch.int32)
    owned, order = [-(-c // PAGE) for c in cached], torch.randperm(pages, generator=g).to(torch.int32)
    for b in range(B):
        table[b, :owned[b]] = order[sum(owned[:b]):sum(owned[:b + 1])]
    free = order[sum(owned):].cuda()
    caches = [torch.zeros(pages, HK, PAGE, D, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    for b in range(B):  # what is cached already
        if cached[b]:
            x = m.embed[torch.tensor(history[b][:cached[b]])].cuda()
            k, v = ((x @ dev["wqkv"][a * D:(a + HK) * D].T).view(-1, HK, D) for a in (HQ, HQ + HK))
            at = torch.arange(cached[b])
            slots = (table[b][at // PAGE] * PAGE + at % PAGE).int().cuda()
            q = torch.zeros(cached[b], HQ, D, dtype=torch.bfloat16, device="cuda")
            qk_norm_rope_write(q, k, v, *caches, slots, at.int().cuda(), dev["freq"], dev["qn"], dev["kn"])
    table = table.cuda()
    new = [len(f) for f in fed]
    step = plan_step(ints(cached), ints(new), ints(owned), table, free, ints([free.numel()]), PAGE, rows)
    assert step.status.tolist() == [0, 0, 0, 0, 0, 1]
    fed_tokens = torch.zeros(rows, dtype=torch.int32, device="cuda")
    fed_tokens[:sum(new)] = ints(sum(fed, []))
    x = dev["embed"][fed_tokens.long()]
    qkv = x @ dev["wqkv"].T
    q, k, v = (qkv[:, a * D:b * D].view(rows, b - a, D) for a, b in ((0, HQ), (HQ, HQ + HK), (HQ + HK, HQ + 2 * HK)))
    q = qk_norm_rope_write(q, k, v, *caches, step.slots, step.positions, dev["freq"], dev["qn"], dev["kn"])
    out = PagedAttention(HQ, HK, D, PAGE)(q, *caches, table, step.cu_new, step.seq_len, max(new))
    requests, most = B, sum(n + 1 for n in drafts)
    wanted = ints([n + 1 if w else 0 for n, w in zip(drafts, want_token)])
    wanted = torch.where(step.status == 0, wanted, 0)
    cu_rows = torch.nn.functional.pad(wanted.cumsum(0), (1, 0)).int()
    i = torch.arange(most, device=wanted.device)
    b = torch.searchsorted(cu_rows[1:], i, right=True).clamp(max=requests - 1)
    judged = (step.cu_new[b + 1] - cu_rows[b + 1] + i).clamp(0, rows - 1)
    ends = [sum(new[:b + 1]) for b in range(B)]
    want_rows = sum((list(range(ends[b] - drafts[b] - 1, ends[b])) for b in (0, 1, 2)), [])
    assert cu_rows.tolist() == [0, 4, 5, 8, 8, 8, 8] and judged[:8].tolist() == want_rows
    target = torch.softmax((x[judged].float() + out[judged].reshape(most, -1).float() @ dev["wo"].float().T)
                           @ dev["head"].float().T, -1)
    exact = [m.dense(torch, h[:c] + f)[1][-(n + 1):] for h, c, f, n in zip(history, cached, fed, drafts)]
    assert float((target[:8].cpu().double() - torch.cat(exact[:3])).abs().max()) < 0.05  # as above
    ua, us = torch.rand(most, generator=g) * 0.1, torch.rand(B, generator=g)
    accepted, tokens = verify_drafts(target, None, fed_tokens[judged], cu_rows, ua.cuda(), us.cuda())
    want = ref.verify(target.cpu(), None, fed_tokens[judged].cpu(), cu_rows.tolist(), ua, us)
    assert accepted.tolist() == want[0] and accepted.tolist()[3:] == [0, 0, 0] and tokens[:8].tolist() == want[1][:8]
    assert all(tokens[a + n].item() >= 0 for a, n in zip((0, 4, 5), want[0]))  # a token for each that wants one


# A fresh process: which kernels have run before is the point.
CAPTURE = """
import torch
from vvli_b200.paged import PagedAttention, qk_norm_rope_write
from vvli_b200.speculative import verify_drafts
ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
g = torch.Generator(device="cuda").manual_seed(1)

def call(dtype, d, n, softcap, norm, odd):
    att = PagedAttention(4, 2, d, 16, dtype=dtype, softcap=softcap)
    q, k, v = rnd(n, 4, d).to(dtype), rnd(n, 2, d).to(dtype), rnd(n, 2, d).to(dtype)
    caches = [torch.zeros(20, 2, 16, d, dtype=dtype, device="cuda") for _ in range(2)]
    at = torch.arange(n, device="cuda", dtype=torch.int32)
    freq = 0.5 ** torch.arange(8, dtype=torch.float64, device="cuda")
    table, cu, seq = ints([list(range(20))]), ints([0, n]), ints([n])
    target = torch.softmax(rnd(3, 1000 + odd), -1)
    tokens, cu3, ua, us = ints([1, 2, 3]), ints([0, 3]), torch.full((3,), 0.01, device="cuda"), torch.full((1,), 0.5, device="cuda")
    def step():
        x = qk_norm_rope_write(q, k, v, *caches, at, at, freq, norm=norm, interleaved=bool(odd))
        return x, att(x, *caches, table, cu, seq, n), *verify_drafts(target, None, tokens, cu3, ua, us)
    return step

call(torch.bfloat16, 64, 1, 0.0, "none", 0)()
torch.cuda.synchronize()
for dtype, d, n, softcap, norm, odd in ((torch.bfloat16, 64, 200, 0.0, "head", 0), (torch.float16, 128, 300, 30.0, "row", 1),
                                        (torch.float16, 64, 5, 0.0, "head", 1)):
    step = call(dtype, d, n, softcap, norm, odd)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    torch.cuda.synchronize()
    got = [x.clone() for x in got]
    for a, b in zip(got, step()):
        assert torch.equal(a, b)
    assert float(got[1].float().abs().max()) > 0.1
print("captured")
"""


def test_captures_of_variants_that_have_not_run():
    # one call of each operator, then captures with other types, sizes, features and alignments
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    p = subprocess.run([sys.executable, "-c", CAPTURE], cwd=root, capture_output=True, text=True, timeout=300)
    assert p.returncode == 0 and p.stdout.endswith("captured\n"), p.stderr[-2000:]


def test_a_step_without_requests():
    import torch
    from vvli_b200.paged import PagedAttention, plan_step, qk_norm_rope_write
    from vvli_b200.speculative import verify_drafts
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    none, table = ints([]), ints([]).view(0, 4)
    caches = [torch.zeros(3, HK, PAGE, D, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    attention = PagedAttention(HQ, HK, D, PAGE)
    for rows in (0, 5):
        for count, left in ((2, 2), (9, 3), (-1, 0)):
            for inplace in (False, True):
                free_count = ints([count])
                step = plan_step(none, none, none, table, ints([2, 0, 1]), free_count, PAGE, rows, inplace=inplace)
                assert [x.tolist() for x in step] == [[0], [], [0] * rows, [-1] * rows, [], [left], []]
                assert free_count.tolist() == [left if inplace else count]
        q, k = (torch.ones(rows, h, D, dtype=torch.bfloat16, device="cuda") for h in (HQ, HK))
        q = qk_norm_rope_write(q, k, k, *caches, step.slots, step.positions)
        assert not any(bool(c.any()) for c in caches)
        out = torch.full((rows, HQ, D), 7.0, dtype=torch.bfloat16, device="cuda")
        assert attention(q, *caches, table, step.cu_new, step.seq_len, 0, out=out) is out and bool((out == 7).all())
        assert attention(q, *caches, table, step.cu_new, step.seq_len, 0, lse=True)[1].shape == (rows, HQ)
        accepted, tokens = verify_drafts(torch.ones(rows, 9, device="cuda"), None, step.positions, step.cu_new,
                                         torch.ones(rows, device="cuda"), torch.ones(0, device="cuda"))
        assert accepted.numel() == 0 and tokens.shape == (rows,)
