"""vvli_cuda_paged_attention against a plain implementation in 64 bits.  Needs a B200."""

import math
import random

import pytest

import paged_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    assert torch.cuda.is_available()
    return torch


def make(torch, seed, lens, hq, hk, d, page, dtype, poison=True, spread=1.5, bad_pages=(), extra_rows=0, width_slack=2):
    """lens: (seq_len, new tokens) of each request. Cells of the cache past a request's end hold NaN and infinities."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-max(0, e) // page) for e, _ in lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g).tolist()
    width = max(need + [1]) + width_slack
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [-1] * (width - n))
        at += n
    k, v = (torch.randn(pages, hk, page, d, generator=g).to(dtype) for _ in range(2))
    if poison:
        for c, fill in ((k, math.nan), (v, math.inf)):
            spare = torch.ones(pages, page, dtype=torch.bool)
            for b, (e, _) in enumerate(lens):
                for j in range(need[b]):
                    spare[table[b][j], :min(page, e - j * page)] = False
            c.transpose(1, 2)[spare] = fill
    for b, j, value in bad_pages:
        table[b][j] = value
    T = sum(n for _, n in lens)
    q = (torch.randn(T + extra_rows, hq, d, generator=g) * spread).to(dtype)
    cu = [sum(n for _, n in lens[:i]) for i in range(len(lens) + 1)]
    return q, k, v, table, cu, [e for e, _ in lens]


def check(torch, inp, page, max_new=None, window=0, softcap=0.0, alibi=None, scale=None, att=None):
    from vvli_b200.paged import PagedAttention
    q, k, v, table, cu, seq = inp
    T, hq, d = q.shape
    hk, dtype = k.shape[1], q.dtype
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    if att is None:
        att = PagedAttention(hq, hk, d, page, dtype=dtype, scale=scale, softcap=softcap, window=window,
                             alibi=None if alibi is None else alibi.cuda())
    out = torch.full((T, hq, d), 7.0, dtype=dtype, device="cuda")
    lse = torch.full((T, hq), 7.0, device="cuda")
    longest = max(b - a for a, b in zip(cu, cu[1:]))
    att(q.cuda(), k.cuda(), v.cuda(), ints(table), ints(cu), ints(seq), longest if max_new is None else max_new, out=out,
        lse=lse)
    torch.cuda.synchronize()
    assert att.status() == 0
    want, wlse = ref.attention(q, k, v, table, cu, seq, d**-0.5 if scale is None else scale, window, softcap, alibi)
    rows = ~torch.isnan(wlse).any(-1)
    out, lse = out.cpu(), lse.cpu()
    assert bool((out[~rows] == 7).all()) and bool((lse[~rows] == 7).all())  # rows of no request
    got, want, lse, wlse = out[rows].double(), want[rows], lse[rows].double(), wlse[rows]
    empty = torch.isinf(wlse)
    assert torch.equal(empty, lse == -math.inf) and bool((got[empty] == 0).all())
    # Scores: 16-bit products are exact in fp32, sums of up to 128 of them stay within
    # 2^-21 of the sum of their magnitudes (at most 2^9 in these tests): a score is off
    # by less than 2^-12, with the exponential a probability and the sum of them by 2^-11.
    # Probabilities and output are rounded to the type: half a step each, of a weighted
    # mean of values (at most the largest |v|).
    half = torch.finfo(dtype).eps / 2
    big = torch.nan_to_num(v.double(), 0.0, 0.0, 0.0).abs().max()
    tol = half * want.abs() + (half + 2.0**-10) * big
    bad = (got - want).abs() > tol
    assert not bool(bad.any()), (int(bad.sum()), float(((got - want).abs() / tol).max()))
    # and on the whole: the errors of many keys average out (root mean square of a rounding: 1/sqrt(3) of half a step)
    if got.numel() > 5000:
        assert float((got - want).norm() / want.norm()) < 2 * half
    fine = ~empty
    assert bool(((lse - wlse)[fine].abs() <= 2.0**-10).all())
    return out


HEADS = [(14, 2, 64), (32, 8, 128), (4, 4, 128), (8, 1, 64), (3, 1, 128), (40, 2, 64)]


@pytest.mark.parametrize("hq,hk,d", HEADS)
@pytest.mark.parametrize("page,dtype", [(16, "bfloat16"), (32, "float16"), (64, "bfloat16"), (128, "float16")])
def test_decode(torch, hq, hk, d, page, dtype):
    lens = [(1, 1), (16, 1), (17, 1), (63, 1), (64, 1), (65, 1), (129, 1), (500, 1), (0, 0), (1000, 1), (2, 1)]
    check(torch, make(torch, d + page, lens, hq, hk, d, page, getattr(torch, dtype)), page)


@pytest.mark.parametrize("hq,hk,d", HEADS)
@pytest.mark.parametrize("n", [2, 5, 9, 33])
def test_drafts(torch, hq, hk, d, n):
    lens = [(n, n), (n + 1, n), (64 + n // 2, n), (130, n), (700, n), (65, 1), (300, max(1, n - 1))]
    check(torch, make(torch, n + hq, lens, hq, hk, d, 16 if n % 2 else 64, torch.bfloat16), 16 if n % 2 else 64)


@pytest.mark.parametrize("hq,hk,d,page,dtype", [(14, 2, 64, 16, "float16"), (32, 8, 128, 64, "bfloat16"),
                                                (4, 4, 128, 128, "bfloat16"), (6, 1, 64, 32, "bfloat16")])
def test_chunks(torch, hq, hk, d, page, dtype):
    lens = [(300, 300), (257, 100), (1, 1), (128, 128), (129, 129), (600, 129), (511, 1), (90, 64), (1000, 65)]
    check(torch, make(torch, d, lens, hq, hk, d, page, getattr(torch, dtype)), page)


@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 200, 5000])
@pytest.mark.parametrize("long", [False, True])
def test_window(torch, window, long):
    lens = [(300, 130), (200, 70), (129, 129)] if long else [(300, 3), (1, 1), (129, 4), (900, 2)]
    check(torch, make(torch, window, lens, 8, 2, 64, 32, torch.bfloat16), 32, window=window)


@pytest.mark.parametrize("softcap,with_alibi,window", [(30.0, False, 0), (0.0, True, 0), (5.0, True, 100), (50.0, False, 64)])
@pytest.mark.parametrize("long", [False, True])
def test_softcap_and_alibi(torch, softcap, with_alibi, window, long):
    alibi = torch.tensor([2.0**-i for i in range(1, 9)]) if with_alibi else None
    lens = [(300, 150), (140, 140), (80, 1)] if long else [(300, 3), (1, 1), (129, 4), (900, 2)]
    for d, dtype in ((64, torch.float16), (128, torch.bfloat16)):
        check(torch, make(torch, 5, lens, 8, 2, d, 64, dtype, spread=4.0), 64, softcap=softcap, alibi=alibi, window=window)


@pytest.mark.parametrize("softcap,spread,scale", [(50.0, 0.5, 0.125), (3.0, 1.0, 0.125), (20.0, 4.0, -0.2), (1.0, 30.0, 0.2),
                                                  (1e-3, 1.0, 0.125), (1e7, 1.0, 0.125), (2e-5, 1.0, 1e-6)])
def test_softcap_from_far_below_to_far_above_the_scores(torch, softcap, spread, scale):
    for lens in ([(200, 150)], [(200, 2)]):
        check(torch, make(torch, 31, lens, 4, 2, 64, 64, torch.bfloat16, spread=spread), 64, softcap=softcap, scale=scale)


@pytest.mark.parametrize("max_new", [0, 1, 4, 300, 10**6])
def test_max_new_only_picks_the_kernel(torch, max_new):
    lens = [(300, 120), (64, 1), (200, 7), (33, 33)]
    check(torch, make(torch, 2, lens, 8, 2, 128, 64, torch.bfloat16), 64, max_new=max_new)


@pytest.mark.parametrize("d,dtype,page", [(64, "bfloat16", 16), (128, "float16", 64), (128, "bfloat16", 128)])
@pytest.mark.parametrize("window", [0, 100])
@pytest.mark.parametrize("max_new", [1, 5, 10**6])
def test_hidden_values_that_are_not_finite(torch, d, dtype, page, window, max_new):
    # infinities and NaN among the values: only rows that see the key have them, in its columns alone
    from vvli_b200.paged import PagedAttention
    lens = [(90, 5), (300, 200), (64, 64), (700, 3), (2000, 40), (130, 1)]
    q, k, v, table, cu, seq = make(torch, 21, lens, 8, 2, d, page, getattr(torch, dtype), poison=False)
    g = torch.Generator().manual_seed(5)
    for b, (e, n) in enumerate(lens):
        for i, value in enumerate((math.nan, math.inf, -math.inf, math.inf)):
            key = e - 1 - int(torch.randint(0, min(e, n + 110), (1,), generator=g))
            v[table[b][key // page], i % 2, key % page, int(torch.randint(0, d, (1,), generator=g))] = value
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    att = PagedAttention(8, 2, d, page, dtype=q.dtype, window=window)
    out = att(q.cuda(), k.cuda(), v.cuda(), ints(table), ints(cu), ints(seq), max_new).cpu().double()
    want, _ = ref.attention(q, k, v, table, cu, seq, d**-0.5, window)
    odd = ~torch.isfinite(want)
    assert int(odd.sum()) > 100 and torch.equal(torch.isnan(out), torch.isnan(want))
    assert torch.equal(out[odd & ~torch.isnan(want)], want[odd & ~torch.isnan(want)])
    half = torch.finfo(q.dtype).eps / 2
    assert float((out - want)[~odd].norm() / want[~odd].norm()) < 2 * half  # as in check()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hk", [(8, 2), (7, 1)])
def test_few_rows_over_one_to_many_tiles(torch, d, hq, hk):
    # items of at most 128 rows in the kernel for many: one key tile, two, odd and even counts, whole and split
    lens = [(n, min(n, 1 + i % 9)) for i, n in enumerate([1, 64, 127, 128, 129, 200, 256, 257, 300, 384, 385, 640, 641, 1500])]
    for window in (0, 130):
        check(torch, make(torch, d + hq, lens, hq, hk, d, 64, torch.bfloat16), 64, max_new=1000, window=window)
    check(torch, make(torch, d, [(6000, 5)], hq, hk, d, 32, torch.float16), 32, max_new=1000)


@pytest.mark.parametrize("max_new", [1, 10**6])
def test_nan_rows_stay_apart(torch, max_new):
    # a NaN query gives NaN (whole item or split over CTAs) and leaves the rows beside it alone
    q, k, v, table, cu, seq = make(torch, 11, [(3000, 3), (70, 2)], 4, 2, 64, 16, torch.bfloat16, poison=False)
    q[1, 2], q[4, 0] = math.nan, math.inf
    from vvli_b200.paged import PagedAttention
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    out, lse = PagedAttention(4, 2, 64, 16)(q.cuda(), k.cuda(), v.cuda(), ints(table), ints(cu), ints(seq), max_new, lse=True)
    bad = torch.zeros(5, 4, dtype=torch.bool)
    bad[1, 2] = bad[4, 0] = True
    assert torch.equal(torch.isnan(out.cpu()).all(-1), bad) and torch.equal(torch.isnan(out.cpu()).any(-1), bad)
    assert torch.equal(torch.isnan(lse.cpu()), bad)


@pytest.mark.parametrize("max_new", [1, 10**6])
def test_empty_rows_bad_pages_and_rows_behind(torch, max_new):
    # seq_len 0 (an unserved request), fewer keys than rows, entries outside the cache, lengths past the table
    lens = [(0, 3), (2, 5), (-4, 2), (100, 4), (200, 1), (150, 2)]
    inp = list(make(torch, 3, lens, 4, 2, 64, 16, torch.bfloat16, extra_rows=5,
                    bad_pages=[(3, 1, -1), (4, 0, 10**9), (4, 5, -2**31), (5, 2, 2**31 - 1)], width_slack=0))
    check(torch, tuple(inp), 16, max_new=max_new)
    inp = list(make(torch, 3, lens, 4, 2, 64, 16, torch.bfloat16, poison=False, bad_pages=[(3, 1, -1)], width_slack=0))
    inp[5][3], inp[5][5] = 10**4, 2**31 - 1
    check(torch, tuple(inp), 16, max_new=max_new)
    check(torch, make(torch, 3, [(0, 0), (0, 0)], 4, 2, 64, 16, torch.bfloat16, extra_rows=2), 16, max_new=max_new)


@pytest.mark.parametrize("long", [False, True])
def test_cut_rows(torch, long):
    # cu_new past the rows of q: the rows there are keep their positions
    n = 200 if long else 4
    q, k, v, table, cu, seq = make(torch, 4, [(n + 40, n), (n + 3, n)], 4, 2, 64, 16, torch.float16)
    check(torch, (q[:n + n // 2].contiguous(), k, v, table, cu, seq), 16)
    check(torch, (q[:n - 2].contiguous(), k, v, table, cu, seq), 16)


@pytest.mark.parametrize("long", [False, True])
def test_strides(torch, long):
    from vvli_b200.paged import PagedAttention
    n = 140 if long else 2
    lens = [(200, n), (n, n), (333, n)]
    q, k, v, table, cu, seq = make(torch, 6, lens, 8, 2, 128, 32, torch.bfloat16)
    want = check(torch, (q, k, v, table, cu, seq), 32)
    both = torch.stack([k, v], 1).cuda()  # pages of keys and values side by side
    wide = torch.randn(q.shape[0], 1600).to(q.dtype).cuda()
    wide[:, 8:8 + 1024] = q.cuda().view(-1, 1024)
    res = torch.zeros(q.shape[0], 1040, dtype=q.dtype, device="cuda")
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    PagedAttention(8, 2, 128, 32)(wide[:, 8:8 + 1024].view(-1, 8, 128), both[:, 0], both[:, 1], ints(table), ints(cu),
                                  ints(seq), n, out=res[:, 16:].view(-1, 8, 128))
    assert torch.equal(res[:, 16:].cpu().view(-1, 8, 128), want) and bool((res[:, :16] == 0).all())


@pytest.mark.parametrize("lens", [[(40000, 1)], [(20000, 4), (5, 1)], [(9000, 40)], [(3000, 1500)],
                                  [(100 + 37 * i % 900, 1) for i in range(700)],
                                  [(1 + 7 * i % 50, 1 + 7 * i % 50) for i in range(40)]])
def test_split_over_ctas(torch, lens):
    # one request over all SMs, many over each SM, and items that end inside shares
    check(torch, make(torch, 7, lens, 4, 1, 64, 64, torch.bfloat16, poison=False), 64)


def test_large_scores_and_fully_peaked_rows(torch):
    for lens in ([(500, 2)], [(500, 200)]):
        q, k, v, table, cu, seq = make(torch, 8, lens, 4, 2, 64, 16, torch.float16, spread=20.0)
        check(torch, (q, k, v, table, cu, seq), 16, scale=0.25)
        check(torch, (q, k, v, table, cu, seq), 16, scale=0.0)
        check(torch, (q, k, v, table, cu, seq), 16, scale=-0.125)


def test_infinite_and_nan_keys_in_sight_reach_the_row(torch):
    # what a row sees is not masked: a NaN value gives NaN in its column, a +inf score NaN in the row, as the formula
    from vvli_b200.paged import PagedAttention
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    for new, max_new in ((1, 1), (130, 130)):
        q, k, v, table, cu, seq = make(torch, 9, [(200, new), (150, new)], 4, 2, 64, 16, torch.bfloat16, poison=False)
        v[table[0][1], 0, 3, 5] = math.nan
        out = PagedAttention(4, 2, 64, 16)(q.cuda(), k.cuda(), v.cuda(), ints(table), ints(cu), ints(seq), max_new).cpu()
        nan = torch.isnan(out)
        assert bool(nan[:new, :2, 5].all()) and int(nan.sum()) == 2 * new


def test_offsets_past_32_bits(torch):
    # pages whose element offset passes 2^32, in caches of one request's pages far apart
    from vvli_b200.paged import PagedAttention
    hk, page, d = 2, 16, 128
    stride = 1 << 29
    base = torch.zeros(stride * 9, dtype=torch.bfloat16, device="cuda")
    cache = base.as_strided((9, hk, page, d), (stride, page * d, d, 1))
    k = torch.randn(9, hk, page, d).to(torch.bfloat16)
    cache.copy_(k.cuda())
    table = [[8, 0, 7, 3, 5, 6, 1, 2, 4]]
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    for n in (1, 40):
        q = torch.randn(n, 4, d).to(torch.bfloat16)
        out = PagedAttention(4, hk, d, page)(q.cuda(), cache, cache, ints(table), ints([0, n]), ints([141]), n)
        want, _ = ref.attention(q, k, k, table, [0, n], [141], d**-0.5)
        assert float((out.cpu().double() - want).norm() / want.norm()) < 2.0**-7


@pytest.mark.parametrize("new", [1, 200])
def test_repeats_bit_for_bit_captured_and_on_another_stream(torch, new):
    from vvli_b200.paged import PagedAttention
    r = random.Random(1)
    lens = [(new + r.randint(0, 600), new) for _ in range(6)]
    q, k, v, table, cu, seq = make(torch, 10, lens, 8, 2, 128, 64, torch.bfloat16)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    att = PagedAttention(8, 2, 128, 64)
    args = (q.cuda(), k.cuda(), v.cuda(), ints(table), ints(cu), ints(seq), new)
    first, l1 = att(*args, lse=True)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    second = att(*args, stream=side)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        third, l3 = att(*args, lse=True)
    for _ in range(2):
        third.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(third, first) and torch.equal(l3, l1)
    assert torch.equal(second, first)
    # the captured call serves other lengths of the same batch
    seq2 = [max(new, s - 50) for s in seq]
    args[5].copy_(ints(seq2))
    graph.replay()
    torch.cuda.synchronize()
    want, _ = ref.attention(q, torch.nan_to_num(k, 0.0), torch.nan_to_num(v, 0.0, 0.0, 0.0), table, cu, seq2, 128**-0.5)
    assert float((third.cpu().double() - want).norm() / want.norm()) < 2.0**-7


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("softcap,with_alibi", [(5.0, False), (50.0, True)])
def test_softcap_repeats_bit_for_bit_between_other_calls(torch, d, softcap, with_alibi):
    # what other calls left in shared memory past the last keys must not show, in the last bit either
    from vvli_b200.paged import PagedAttention
    r = random.Random(d)
    lens = [(n + r.randint(0, 200), n) for n in (r.randint(1, 40) for _ in range(120))]
    q, k, v, table, cu, seq = make(torch, 41, lens, 6, 3, d, 16, torch.bfloat16, poison=False)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    att = PagedAttention(6, 3, d, 16, softcap=softcap, alibi=torch.rand(6).cuda() if with_alibi else None)
    args = (ints(table), ints(cu), ints(seq), 10**6)
    mine, other = (q.cuda(), k.cuda(), v.cuda()), (8 * q.cuda(), 30 * k.cuda(), v.cuda())
    first = att(*mine, *args, lse=True)
    for i in range(12):
        att(*other, *args)
        if i % 3 == 0:
            att(q.cuda(), torch.full_like(other[1], math.nan), other[2], *args)
        again = att(*mine, *args, lse=True)
        assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])


def test_wrapper_refusals(torch):
    from vvli_b200.errors import VvliError
    from vvli_b200.paged import PagedAttention
    with pytest.raises(ValueError):
        PagedAttention(4, 2, 96, 16)
    with pytest.raises(ValueError):
        PagedAttention(4, 2, 64, 16, dtype=torch.float32)
    with pytest.raises(ValueError):
        PagedAttention(4, 2, 64, 16, alibi=torch.zeros(3, device="cuda"))
    att = PagedAttention(4, 2, 64, 16)
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    i = torch.zeros(4, dtype=torch.int32, device="cuda")
    q, c, t = z(3, 4, 64), z(5, 2, 16, 64), i.view(2, 2)
    for bad in (lambda: att(q.half(), c, c, t, i[:3], i[:2], 1), lambda: att(z(3, 2, 64), c, c, t, i[:3], i[:2], 1),
                lambda: att(q, z(5, 2, 32, 64), z(5, 2, 32, 64), t, i[:3], i[:2], 1),
                lambda: att(q, c, c[:4], t, i[:3], i[:2], 1), lambda: att(q, c, c, t[:1], i[:3], i[:2], 1),
                lambda: att(q, c, c, t, i[:2], i[:2], 1), lambda: att(q, c, c, t.long(), i[:3], i[:2], 1),
                lambda: att(q, c, c, t, i[:3], i[:2], 1, out=z(2, 4, 64)),
                lambda: att(q, c, c, t, i[:3], i[:2], 1, lse=torch.zeros(3, 3, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(VvliError):
        PagedAttention(5, 2, 64, 16)(z(3, 5, 64), c, c, t, i[:3], i[:2], 1)
    assert att(q[:0], c, c, t, i[:3], i[:2], 1).shape == (0, 4, 64)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("gap", [12.0, 15.0, 18.0])
@pytest.mark.parametrize("new", [1, 3, 40])
def test_dominant_keys_of_no_value_leave_the_others(torch, dtype, gap, new):
    # keys `gap` above some 30,000 others, with values of zero: the output is what the others add up to.  Eight such
    # keys (16 apart) in every 2,048, and as many requests as keep the SMs at work on whole ones, so that the
    # others are summed beside one.
    from vvli_b200.paged import PagedAttention
    g = torch.Generator().manual_seed(17)
    dtype = getattr(torch, dtype)
    q, k, v, table, _, _ = make(torch, 17, [(30000, new)], 4, 2, 64, 64, dtype, poison=False)
    q.fill_(2.0)  # a score is 16 times the key's one number
    k.copy_(0.015 * (2 * torch.rand(k.shape[:3] + (1,), generator=g) - 1))
    v.copy_(64 * (0.5 + torch.rand(v.shape, generator=g)))
    for key in (first + 16 * i for first in range(0, 29900, 2048) for i in range(8)):
        page = table[0][key // 64]
        k[page, :, key % 64], v[page, :, key % 64] = gap / 16, 0.0
    B = 80
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    out, lse = PagedAttention(4, 2, 64, 64, dtype=dtype)(
        q.repeat(B, 1, 1).cuda(), k.cuda(), v.cuda(), ints(table * B), ints([new * b for b in range(B + 1)]),
        ints([30000] * B), new, lse=True)
    want, wlse = ref.attention(q, k, v, table, [0, new], [30000], 64**-0.5)
    # Values of one sign, so the errors of the terms bound that of the sum, relative to it: the output's
    # rounding, that of a probability (half a step; in fp16 e^-18.3 is 2^-26.4, held as 2^-17.4 at least, where a
    # half's spacing is 2^-24, so that a term is off by up to 2^-7.6, but in either direction: spread over some 46
    # spacings, 29,880 of them together by 2^-7.6 / sqrt(3 * 29,880) = 2^-15.8, six times which is well below the
    # 2^-9.6 allowed), 2^-11 for score and exponential as in check(), and 2^-13 for fp32 sums over 30,000 keys,
    # 16 at a time.
    half = torch.finfo(dtype).eps / 2
    off = float(((out.cpu().double().view(B, new, 4, 64) - want).abs() / want).max())
    assert off < half + max(half, 2.0**-9.6) + 2.0**-11 + 2.0**-13
    off = float((lse.cpu().double().view(B, new, 4) - wlse).abs().max())
    assert off < 2.0**-10


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window", [0, 90])
def test_values_that_are_not_finite_before_runs_of_narrow_items(torch, d, window):
    # chunks of two row tiles with infinities and NaN among their values, each followed by many requests of one
    # token (items that one row tile works on), so that every CTA has dozens of items, over 384 requests in all
    from vvli_b200.paged import PagedAttention
    r = random.Random(d)
    lens = [(n + r.randint(0, 60), n) for n in (70 if i % 40 == 3 else 1 for i in range(1600))]
    q, k, v, table, cu, seq = make(torch, 23, lens, 8, 2, d, 16, torch.bfloat16, poison=False)
    for b, (e, n) in enumerate(lens):
        for i, value in enumerate((math.nan, math.inf, -math.inf) if n > 1 else ()):
            key = e - 1 - r.randrange(n)
            v[table[b][key // 16], i % 2, key % 16, r.randrange(d)] = value
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    att = PagedAttention(8, 2, d, 16, window=window)
    args = (q.cuda(), k.cuda(), v.cuda(), ints(table), ints(cu), ints(seq), 10**6)
    want, _ = ref.attention(q, k, v, table, cu, seq, d**-0.5, window)
    odd = ~torch.isfinite(want)
    assert int(odd.sum()) > 1000
    for _ in range(3):
        out = att(*args).cpu().double()
        assert torch.equal(torch.isnan(out), torch.isnan(want))
        assert torch.equal(out[odd & ~torch.isnan(want)], want[odd & ~torch.isnan(want)])
        assert float((out - want)[~odd].norm() / want[~odd].norm()) < 2 * torch.finfo(q.dtype).eps / 2  # as in check()
    assert att.status() == 0


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("max_new", [1, 10**6])
def test_many_short_requests(torch, d, max_new):
    # more requests than threads of either kernel: the shares are worked out in several rounds
    r = random.Random(d)
    lens = [(n + r.randint(0, 90), n) for n in (r.randint(0, 6) for _ in range(900))]
    check(torch, make(torch, 13, lens, 4, 2, d, 16, torch.bfloat16), 16, max_new=max_new)


@pytest.mark.parametrize("d,dtype", [(64, "float16"), (128, "bfloat16")])
@pytest.mark.parametrize("window,softcap", [(0, 0.0), (60, 0.0), (60, 20.0)])
@pytest.mark.parametrize("max_new", [1, 10**6])
def test_keys_that_are_not_finite(torch, d, dtype, window, softcap, max_new):
    # A NaN key makes the rows that see it NaN, an infinite one those that it scores +inf (a score of -inf has no
    # weight, a cap makes either finite); rows that do not, earlier in the block or past the window, have nothing of it.
    from vvli_b200.paged import PagedAttention
    lens = [(90, 5), (300, 200), (64, 64), (700, 3), (500, 40), (130, 1)]
    q, k, v, table, cu, seq = make(torch, 27, lens, 8, 2, d, 16, getattr(torch, dtype), poison=False)
    r = random.Random(3)
    for b, (e, n) in enumerate(lens):
        for h, value in enumerate((math.nan, math.inf)):
            key = e - 1 - r.randrange(min(e, n + 70 if window else n))
            k[table[b][key // 16], h, key % 16, r.randrange(d)] = value
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    att = PagedAttention(8, 2, d, 16, dtype=q.dtype, window=window, softcap=softcap)
    out = att(q.cuda(), k.cuda(), v.cuda(), ints(table), ints(cu), ints(seq), max_new).cpu().double()
    want, _ = ref.attention(q, k, v, table, cu, seq, d**-0.5, window, softcap)
    nan = torch.isnan(want)
    assert int(nan.sum()) > 100 and int((~nan).sum()) > 100 and torch.equal(torch.isnan(out), nan)
    assert float((out - want)[~nan].norm() / want[~nan].norm()) < 2 * torch.finfo(q.dtype).eps / 2  # as in check()


@pytest.mark.parametrize("new", [1, 60])
def test_workspace_on_other_streams(torch, new):
    # The workspace's memory may be on its way from another use, and back to one: neither shows, whatever stream a
    # call is on, and although the object goes away while its call still runs.
    from vvli_b200.paged import PagedAttention
    q, k, v, table, cu, seq = make(torch, 33, [(3000, new), (40 + new, new)], 8, 2, 128, 64, torch.bfloat16, poison=False)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    args = (q.cuda(), k.cuda(), v.cuda(), ints(table), ints(cu), ints(seq), new)
    want = PagedAttention(8, 2, 128, 64)(*args).cpu()
    size = PagedAttention(8, 2, 128, 64)._ws.numel()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for given in (True, False):
        before = torch.empty(size, dtype=torch.uint8, device="cuda")
        torch.cuda._sleep(20_000_000)  # about 10 ms
        before.fill_(255)
        at = before.data_ptr()
        del before
        att = PagedAttention(8, 2, 128, 64)
        assert att._ws.data_ptr() == at  # the same memory, the point of the test
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)
            out = att(*args, stream=side if given else None)
        del att
        after = torch.empty(size, dtype=torch.uint8, device="cuda")
        assert after.data_ptr() != at
        after.fill_(255)
        side.synchronize()
        assert torch.equal(out.cpu(), want)
        torch.cuda.synchronize()
