"""The paged serving step's plan and q / k operators against plain implementations in 64 bits.  Needs a B200."""

import random

import pytest

import paged_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    assert torch.cuda.is_available()
    return torch


def ints(torch, v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------- plan

def make_plan(seed, B, page, ctx, new, spare, width_slack=1, over=0):
    """Lengths, tables and a free stack; `over` requests own a page more than they use, as after a rollback."""
    r = random.Random(seed)
    context = [r.randint(0, ctx) for _ in range(B)]
    news = [r.randint(0, new) for _ in range(B)]
    owned = [-(-c // page) + (1 if i < over else 0) for i, c in enumerate(context)]
    need = sum(max(0, -(-(c + n) // page) - o) for c, n, o in zip(context, news, owned))
    pages = sum(owned) + need + max(spare, 0)
    ids = list(range(pages))
    r.shuffle(ids)
    width = max(max(o, -(-(c + n) // page)) for c, n, o in zip(context, news, owned)) + width_slack
    table, at = [], 0
    for o in owned:
        table.append(ids[at:at + o] + [-7] * (width - o))
        at += o
    free = ids[at:] + [-9] * 3
    return context, news, owned, table, free, max(0, need + spare), page, pages


def check_plan(torch, case, max_tokens, inplace=False):
    from vvli_b200.paged import plan_step
    context, new, owned, table, free, count, page, pages = case
    tab = ints(torch, table)
    own, cnt = ints(torch, owned), ints(torch, [count])
    p = plan_step(ints(torch, context), ints(torch, new), own, tab, ints(torch, free), cnt, page, max_tokens,
                  inplace=inplace)
    want = ref.plan(context, new, owned, table, free, count, page, max_tokens)
    for name, w in zip(p._fields, want):
        assert getattr(p, name).tolist() == w, name
    assert tab.tolist() == table
    if inplace:
        assert own.tolist() == want[4] and cnt.tolist() == want[5]
    return want


@pytest.mark.parametrize("B,page,ctx,new", [(1, 64, 0, 1), (1, 16, 1000, 300), (16, 64, 4096, 1), (33, 128, 500, 70),
                                            (1024, 16, 300, 6), (1500, 32, 60, 9), (8192, 16, 40, 3)])
@pytest.mark.parametrize("inplace", [False, True])
def test_plan(torch, B, page, ctx, new, inplace):
    case = make_plan(B + page, B, page, ctx, new, spare=5, over=B // 3)
    check_plan(torch, case, sum(case[1]) + 7, inplace)  # rows behind the last request: slot -1


@pytest.mark.parametrize("spare", [-1, -9, -100000])
def test_plan_pages_run_out(torch, spare):
    case = make_plan(5, 200, 16, 100, 40, spare=spare)
    want = check_plan(torch, case, sum(case[1]))
    assert 1 in want[6] and (spare < -1000) == (want[5] == [0] and all(a == b for a, b in zip(want[4], case[2])))


def test_plan_refused_requests(torch):
    # a table row that is too short, rows past max_tokens, negative lengths, bad pages in the table
    case = list(make_plan(8, 40, 16, 200, 50, spare=30, width_slack=0))
    case[0][3] = 16 * len(case[3][0]) + 1
    case[1][4], case[0][5], case[2][6] = -3, -1, -5
    case[3][7][0], case[3][8][0], case[3][9][0] = -1, 2**31 - 1, 2**27 - 1
    want = check_plan(torch, tuple(case), sum(max(0, n) for n in case[1]) - 60)
    assert {0, 2, 3} <= set(want[6])
    check_plan(torch, make_plan(9, 3, 64, 10, 10, spare=0), 0)  # no rows wanted


def test_plan_spare_free_count(torch):
    case = list(make_plan(10, 6, 16, 50, 50, spare=3))
    case[5] = 10**6  # more than the stack holds: cut
    check_plan(torch, tuple(case), 400)
    case = list(make_plan(10, 6, 16, 50, 50, spare=3))
    case[5] = -2
    check_plan(torch, tuple(case), 400)


# ---------------------------------------------------------------- q / k norm, rotation, cache write

def make_qk(torch, seed, T, hq, hk, d, page, dtype, norm, pairs, far=4096, fused=True, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    qkv = (rnd(T, (hq + 2 * hk) * d + (8 if fused else 0)) * scale).to(dtype)
    w = (hq + 2 * hk) * d
    parts = [qkv[:, :hq * d].view(T, hq, d), qkv[:, hq * d:(hq + hk) * d].view(T, hk, d),
             qkv[:, (hq + hk) * d:w].view(T, hk, d)]
    pages = -(-T // page) + 2
    caches = [rnd(pages, hk, page, d).to(dtype) for _ in range(2)]
    slots = torch.randperm(pages * page, generator=g)[:T].to(torch.int32)
    slots[::5] = -1
    if T > 6:
        slots[6] = pages * page  # outside
    positions = torch.randint(0, far, (T,), generator=g).to(torch.int32)
    freq = 10000.0 ** (-torch.arange(pairs, dtype=torch.float64) / max(pairs, 1)) if pairs else None
    weights = [None if norm == "none" else (1 + 0.3 * rnd((h * d) if norm == "row" else d)).to(dtype) for h in (hq, hk)]
    return parts, caches, slots, positions, freq, weights


def check_qk(torch, inp, norm, interleaved, eps=1e-6, inplace=False, far=4096):
    from vvli_b200.paged import qk_norm_rope_write
    (q, k, v), caches, slots, positions, freq, weights = inp
    T, hq, d = q.shape
    dtype, page = q.dtype, caches[0].shape[2]
    base = q._base if q._base is not None else q
    dev = base.cuda()  # one fused tensor on the device, viewed as on the host
    on = lambda x: dev.as_strided(x.shape, x.stride(), x.storage_offset())  # noqa: E731
    gc = [c.cuda() for c in caches]
    gq = on(q)
    out = qk_norm_rope_write(gq, on(k), on(v), gc[0], gc[1], slots.cuda(), positions.cuda(),
                             None if freq is None else freq.cuda(), *[None if w is None else w.cuda() for w in weights],
                             norm=norm, eps=eps, interleaved=interleaved, out=gq if inplace else None)
    torch.cuda.synchronize()
    want_q = ref.qk_rows(q, weights[0], norm, eps, positions, freq, interleaved)
    want_k = ref.qk_rows(k, weights[1], norm, eps, positions, freq, interleaved)
    half, tiny = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2

    def close(got, want):
        # Rounding to the type (half a step, or half the smallest subnormal), and
        # fp32 before it: the mean square (a sum over d or a whole row, in
        # partial sums of at most 2^6 terms each: 2^6 * 2^-24, halved by the
        # root), three products, the sine, cosine and the turn, each within
        # 2^-22 of the pair's length; the pair is at most the head's largest
        # value times sqrt(2): together below 2^-17 of it.
        bound = half * want.abs() * (1 + 2**-8) + tiny + 2.0**-17 * want.abs().amax(-1, keepdim=True)
        assert bool(((got.double() - want).abs() <= bound).all())

    close(out.cpu(), want_q)
    flat = [c.transpose(1, 2).reshape(-1, c.shape[1], d) for c in caches]  # [pages * page][hk][d]
    for got, before, rows in zip(gc, flat, (want_k, v.double())):
        got = got.cpu().transpose(1, 2).reshape(-1, before.shape[1], d)
        written = torch.zeros(before.shape[0], dtype=torch.bool)
        for t in range(T):
            s = int(slots[t])
            if 0 <= s < before.shape[0]:
                written[s] = True
                if rows is want_k:
                    close(got[s], rows[t])
                else:
                    assert torch.equal(got[s], v[t])
        assert torch.equal(got[~written], before[~written])


@pytest.mark.parametrize("norm", ["none", "head", "row"])
@pytest.mark.parametrize("hq,hk,d,pairs,page,interleaved", [
    (32, 8, 128, 64, 64, False), (14, 2, 64, 32, 16, True), (16, 16, 128, 64, 128, False), (3, 1, 16, 8, 32, False),
    (5, 5, 48, 16, 16, True), (2, 1, 256, 128, 32, False), (7, 1, 96, 16, 64, False), (4, 2, 80, 0, 16, False)])
def test_qk(torch, norm, hq, hk, d, pairs, page, interleaved):
    for T, dtype in ((1, torch.bfloat16), (13, torch.float16), (70, torch.bfloat16)):
        inp = make_qk(torch, T + d, T, hq, hk, d, page, dtype, norm, pairs)
        check_qk(torch, inp, norm, interleaved)


def test_qk_in_place_far_positions_and_large_values(torch):
    inp = make_qk(torch, 1, 37, 8, 4, 128, 64, torch.bfloat16, "head", 64, far=1 << 30)
    check_qk(torch, inp, "head", False, inplace=True)
    inp = make_qk(torch, 2, 9, 8, 4, 64, 16, torch.bfloat16, "row", 32, far=1 << 20, scale=1e15)
    check_qk(torch, inp, "row", True, inplace=True)
    inp = make_qk(torch, 3, 9, 8, 4, 64, 16, torch.float16, "head", 32, scale=1e-4)
    check_qk(torch, inp, "head", False, eps=0.0)


def test_qk_missing_weights_and_no_tokens(torch):
    inp = list(make_qk(torch, 4, 11, 4, 2, 64, 32, torch.float16, "head", 16))
    inp[5] = [None, None]
    check_qk(torch, tuple(inp), "head", False)
    from vvli_b200.paged import qk_norm_rope_write
    e = torch.empty(0, 4, 64, dtype=torch.bfloat16, device="cuda")
    c = torch.zeros(2, 4, 16, 64, dtype=torch.bfloat16, device="cuda")
    assert qk_norm_rope_write(e, e, e, c, c, ints(torch, []), norm="none").shape == (0, 4, 64)


def test_qk_pages_apart_and_past_32_bits(torch):
    # caches as halves of one [pages][2][hk][page][d] tensor, and slots whose element offset passes 2^32
    from vvli_b200.paged import qk_norm_rope_write
    hk, page, d = 8, 128, 128
    pages = (1 << 32) // (2 * hk * page * d) + 40
    both = torch.zeros(pages, 2, hk, page, d, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(3)
    q = torch.randn(5, hk, d, generator=g, device="cuda").to(torch.bfloat16)
    slots = ints(torch, [pages * page - 1, 0, (pages - 3) * page + 5, 2 * page, (pages - 20) * page])
    qk_norm_rope_write(q, q, -q, both[:, 0], both[:, 1], slots, norm="none")
    for t, s in enumerate(slots.tolist()):
        assert torch.equal(both[s // page, 0, :, s % page], q[t]) and torch.equal(both[s // page, 1, :, s % page], -q[t])
    assert int((both != 0).any(-1).sum()) == 2 * 5 * hk


def test_errors_on_the_gpu_path(torch):
    from vvli_b200.errors import VvliError
    from vvli_b200.paged import plan_step, qk_norm_rope_write
    q = torch.zeros(4, 4, 64, dtype=torch.bfloat16, device="cuda")
    c = torch.zeros(2, 4, 16, 64, dtype=torch.bfloat16, device="cuda")
    s = ints(torch, [0, 1, 2, 3])
    f = torch.ones(12, dtype=torch.float64, device="cuda")
    with pytest.raises(VvliError) as e:
        qk_norm_rope_write(q, q, q, c, c, s, s, f, norm="none")  # 12 pairs
    assert e.value.name == "InvalidArgument"
    for bad in (lambda: qk_norm_rope_write(q.float(), q, q, c, c, s), lambda: qk_norm_rope_write(q, q[:3], q, c, c, s),
                lambda: qk_norm_rope_write(q, q, q, c.half(), c, s), lambda: qk_norm_rope_write(q, q, q, c, c, s[:3]),
                lambda: qk_norm_rope_write(q, q, q, c, c, s, inv_freq=f),
                lambda: qk_norm_rope_write(q, q, q, c, c, s, q_weight=q),
                lambda: qk_norm_rope_write(q.transpose(0, 1), q, q, c, c, s),
                lambda: qk_norm_rope_write(q, q, q, c[:, :, :, ::2], c, s),
                lambda: plan_step(s, s, s.long(), s.view(4, 1), s, s[:1], 16, 4),
                lambda: plan_step(s, s, s, s, s, s[:1], 16, 4), lambda: plan_step(s, s[::2], s, s.view(4, 1), s, s, 16, 4)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(VvliError):
        plan_step(s, s, s, s.view(4, 1), s, s[:1], 24, 4)


def test_plan_and_write_captured_on_another_stream(torch):
    # A step captured once and replayed after its lengths changed, on a stream that is not the current one.
    from vvli_b200.paged import plan_step, qk_norm_rope_write
    context, new, owned, table, free, count, page, pages = make_plan(21, 12, 16, 60, 9, spare=60)
    rows = 12 * 9
    dev = dict(context=ints(torch, context), new=ints(torch, new), owned=ints(torch, owned), table=ints(torch, table),
               free=ints(torch, free), count=ints(torch, [count]))
    g = torch.Generator(device="cuda").manual_seed(5)
    k = torch.randn(rows, 2, 64, generator=g, device="cuda").half()
    caches = [torch.zeros(pages, 2, page, 64, dtype=torch.float16, device="cuda") for _ in range(2)]

    def step(stream=None):
        p = plan_step(dev["context"], dev["new"], dev["owned"], dev["table"], dev["free"], dev["count"], page, rows,
                      stream=stream)
        qk_norm_rope_write(k, k, k, *caches, p.slots, p.positions, norm="none", stream=stream)
        return p

    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    step(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p = step()
    new2 = [random.Random(3).randint(0, 9) for _ in new]
    dev["new"].copy_(ints(torch, new2))
    dev["table"].copy_(ints(torch, table))
    for c in caches:
        c.zero_()
    graph.replay()
    torch.cuda.synchronize()
    want = ref.plan(context, new2, owned, table, free, count, page, rows)
    for name, w in zip(p._fields, want):
        assert getattr(p, name).tolist() == w, name
    for t, s in enumerate(want[3]):
        if s >= 0:
            assert torch.equal(caches[0][s // page, :, s % page], k[t])
    assert int((caches[1] != 0).any(-1).sum()) == 2 * sum(s >= 0 for s in want[3])


def test_qk_row_norm_in_place_over_many_heads(torch):
    # more heads than one pass of a CTA takes: every head is read for the row's norm before any is overwritten
    inp = make_qk(torch, 11, 21, 96, 24, 128, 32, torch.bfloat16, "row", 64)
    for _ in range(3):
        check_qk(torch, inp, "row", False, inplace=True)


@pytest.mark.parametrize("norm", ["none", "head", "row"])
@pytest.mark.parametrize("T", [257, 1023, 1025, 2051])
def test_qk_many_tokens(torch, norm, T):
    # CTAs of one, two and eight tokens, the last of them with fewer
    for hq, hk, d, pairs, interleaved in ((6, 2, 64, 32, True), (3, 3, 128, 32, False)):
        inp = make_qk(torch, T, T, hq, hk, d, 16, torch.float16 if interleaved else torch.bfloat16, norm, pairs)
        check_qk(torch, inp, norm, interleaved, inplace=T == 1025)


def test_qk_row_norm_of_many_tokens_in_place_over_many_heads(torch):
    inp = make_qk(torch, 12, 1037, 20, 10, 128, 32, torch.bfloat16, "row", 64)
    check_qk(torch, inp, "row", False, inplace=True)
