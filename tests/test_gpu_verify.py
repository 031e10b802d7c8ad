"""vvli_cuda_verify_drafts against a plain implementation in 64 bits.  Needs a B200."""

import math

import pytest

import paged_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    assert torch.cuda.is_available()
    return torch


def make(torch, seed, lengths, V, noise=1.0, sharp=3.0):
    g = torch.Generator().manual_seed(seed)
    T = sum(lengths)
    logits = torch.randn(T, V, generator=g) * sharp
    target = torch.softmax(logits, -1)
    draft = torch.softmax(logits + noise * torch.randn(T, V, generator=g), -1)
    tokens = torch.roll(torch.multinomial(draft, 1, generator=g)[:, 0], 1).to(torch.int32) if T else torch.zeros(0, dtype=torch.int32)
    cu = [sum(lengths[:i]) for i in range(len(lengths) + 1)]
    return target, draft, tokens, cu, torch.rand(T, generator=g), torch.rand(len(lengths), generator=g)


def run(torch, target, draft, tokens, cu, ua, us):
    from vvli_b200.speculative import verify_drafts
    acc, out = verify_drafts(target.cuda(), None if draft is None else draft.cuda(), tokens.cuda(),
                             torch.tensor(cu, dtype=torch.int32, device="cuda"), ua.cuda(), us.cuda())
    return acc.tolist(), out.tolist()


def check(torch, target, draft, tokens, cu, ua, us):
    got, want = run(torch, target, draft, tokens, cu, ua, us), ref.verify(target, draft, tokens, cu, ua, us)
    assert got[0] == want[0]
    assert [g for g, w in zip(got[1], want[1]) if w is not None] == [w for w in want[1] if w is not None]
    return want


@pytest.mark.parametrize("V", [1, 2, 31, 257, 32003, 50304])
@pytest.mark.parametrize("one_hot", [False, True])
def test_verify(torch, V, one_hot):
    lengths = [1, 5, 0, 3, 2, 7, 1, 4, 0, 40]
    target, draft, tokens, cu, ua, us = make(torch, V, lengths, V)
    check(torch, target, None if one_hot else draft, tokens, cu, ua, us)


def test_accepts_all_long_runs_and_rejects_all(torch):
    target, draft, tokens, cu, ua, us = make(torch, 3, [70, 33, 34, 1], 1000)
    assert check(torch, target, target, tokens, cu, ua * 0, us)[0] == [69, 32, 33, 0]
    assert check(torch, target, draft, tokens, cu, ua * 0 + math.inf, us)[0] == [0, 0, 0, 0]
    assert check(torch, target, draft, tokens, cu, ua * math.nan, us)[0] == [0, 0, 0, 0]


@pytest.mark.parametrize("u", [0.0, 0.5, 1.0 - 2.0**-24, 1.0, math.nan])
def test_draw_borders(torch, u):
    V = 5000
    t = torch.zeros(4, V)
    t[0, 17] = 1.0                      # one token has all weight
    t[1, [3, 4999]] = 0.5               # u = 0.5 falls on the border: the later one
    t[2] = 1.0 / 8192                   # flat, sums exact
    t[3, 100:200] = 2.0                 # rows need not sum to 1
    check(torch, t, None, torch.zeros(4, dtype=torch.int32), [0, 1, 2, 3, 4], torch.rand(4), torch.full((4,), u))


def test_nothing_left_bad_drafts_and_nan(torch):
    V = 300
    target, draft, tokens, cu, ua, us = make(torch, 9, [2, 2, 2, 2, 2, 1], V)
    draft[0] = target[0] * 2            # nothing of the target above the draft: drawn from the target
    tokens[3], tokens[5] = -4, V        # drafts outside the vocabulary
    target[6] = 0                       # no weight at all: token 0
    target[8, 5] = math.nan             # counts as 0
    target[10, 7] = -1.0
    ua[:] = 1e30
    check(torch, target, draft, tokens, cu, ua, us)
    check(torch, target, None, tokens, cu, ua, us)


def test_strided_rows_rows_behind_and_cut_rows(torch):
    target, draft, tokens, cu, ua, us = make(torch, 12, [3, 4, 2], 1001)
    wide_t, wide_d = torch.zeros(9, 1030).cuda(), torch.zeros(9, 1111).cuda()
    wide_t[:, :1001], wide_d[:, :1001] = target.cuda(), draft.cuda()
    from vvli_b200.speculative import verify_drafts
    for ends in ([0, 3, 7, 9], [0, 3, 5, 7], [0, 3, 7, 1000], [0, 3, 2, 9]):  # rows behind the last; past the end; decreasing
        acc, out = verify_drafts(wide_t[:, :1001], wide_d[:, :1001], tokens.cuda(),
                                 torch.tensor(ends, dtype=torch.int32, device="cuda"), ua.cuda(), us.cuda())
        if ends == [0, 3, 2, 9]:
            assert acc.tolist()[1] == 0
            continue
        want = ref.verify(target, draft, tokens, ends, ua, us)
        assert acc.tolist() == want[0]
        assert all(w is None or g == w for g, w in zip(out.tolist(), want[1]))


def test_large_batch_repeats_bit_for_bit(torch):
    g = torch.Generator(device="cuda").manual_seed(4)
    lengths = [1 + i % 6 for i in range(200)]
    T, V = sum(lengths), 32003
    target = torch.softmax(3 * torch.randn(T, V, generator=g, device="cuda"), -1)
    draft = torch.softmax(3 * torch.randn(T, V, generator=g, device="cuda"), -1)
    tokens = torch.randint(0, V, (T,), generator=g, device="cuda").to(torch.int32)
    cu = [sum(lengths[:i]) for i in range(len(lengths) + 1)]
    ua, us = torch.rand(T, generator=g, device="cuda") * 1e-3, torch.rand(len(lengths), generator=g, device="cuda")
    want = check(torch, target.cpu(), draft.cpu(), tokens.cpu(), cu, ua.cpu(), us.cpu())
    assert any(0 < a for a in want[0])


def test_emitted_tokens_follow_the_target(torch):
    # 40,000 drafts of one position: the first emitted token is distributed as the target.
    V, N = 6, 40000
    g = torch.Generator().manual_seed(8)
    p = torch.tensor([0.3, 0.05, 0.25, 0.1, 0.2, 0.1])
    q = torch.tensor([0.05, 0.3, 0.25, 0.2, 0.1, 0.1])
    target, draft = p.repeat(2 * N, 1), q.repeat(2 * N, 1)
    tokens = torch.multinomial(q, 2 * N, True, generator=g).to(torch.int32)
    acc, out = run(torch, target, draft, tokens, list(range(0, 2 * N + 1, 2)), torch.rand(2 * N, generator=g),
                   torch.rand(N, generator=g))
    counts = torch.bincount(torch.tensor(out[::2]), minlength=V).double() / N
    # five standard deviations of a share of 40,000 draws, at most sqrt(1/4 / N)
    assert float((counts - p).abs().max()) < 5 * math.sqrt(0.25 / N)


def test_errors(torch):
    from vvli_b200.speculative import verify_drafts
    t = torch.zeros(4, 10, device="cuda")
    i = torch.zeros(4, dtype=torch.int32, device="cuda")
    u = torch.zeros(4, device="cuda")
    for bad in (lambda: verify_drafts(t.half(), None, i, i, u, u[:1]), lambda: verify_drafts(t, t[:3], i, i, u, u[:1]),
                lambda: verify_drafts(t, None, i[:2], i, u, u[:1]), lambda: verify_drafts(t, None, i, i, u, u),
                lambda: verify_drafts(t.T, None, i, i, u, u[:1]), lambda: verify_drafts(t, None, i, i, u.double(), u[:1])):
        with pytest.raises(ValueError):
            bad()
    acc, out = verify_drafts(t[:0], None, i[:0], i, u[:0], u[:3])
    assert acc.tolist() == [0, 0, 0] and out.numel() == 0


@pytest.mark.parametrize("V", [196608, 196609, 256000, 262144])
@pytest.mark.parametrize("one_hot", [False, True])
def test_large_vocabularies(torch, V, one_hot):
    # up to and past the slice whose runs a thread holds in registers
    target, draft, tokens, cu, ua, us = make(torch, V, [1, 3, 2, 4], V)
    check(torch, target, None if one_hot else draft, tokens, cu, ua, us)
    us[:] = torch.tensor([0.0, 1.0 - 2.0**-24, 1.0, 0.999])
    check(torch, target, None if one_hot else draft, tokens, cu, ua + 1e6, us)


def test_repeats(torch):
    lengths = [1 + i % 6 for i in range(100)]
    args = make(torch, 6, lengths, 32003)
    first = run(torch, *args)
    assert all(run(torch, *args) == first for _ in range(3))


def test_rows_behind_the_last_request_are_left(torch):
    from vvli_b200 import _abi
    target, draft, tokens, cu, ua, us = make(torch, 14, [3, 0, 4, 5], 500)
    dev = [x.cuda() for x in (target, draft, tokens, torch.tensor(cu[:-1], dtype=torch.int32), ua, us)]
    acc, out = (torch.full((n,), 77, dtype=torch.int32, device="cuda") for n in (4, 12))
    a = _abi.pack_verify(3, 12, 500, 500, 500, *[x.data_ptr() for x in dev], acc.data_ptr(), out.data_ptr())
    assert _abi.lib().vvli_cuda_verify_drafts(0, a, torch.cuda.current_stream().cuda_stream) == 0
    want = ref.verify(target, draft, tokens, cu[:-1], ua, us)
    assert acc.tolist() == want[0] + [77] and out.tolist() == [77 if w is None else w for w in want[1]]
