"""Struct layouts and argument checks of the paged serving step (all before any CUDA call: no GPU needed)."""

import ctypes

import pytest

from vvli_b200 import _abi
from vvli_b200.errors import CODE_OF

INVALID = CODE_OF["InvalidArgument"]
PTR = 1 << 20  # never read: every case is refused first


def refused(fn, good, changes, text):
    a = type(good).from_buffer_copy(good)
    for name, value in changes.items():
        setattr(a, name, value)
    assert fn(0, ctypes.byref(a), None) == INVALID, changes
    assert text in _abi.lib().vvli_cuda_last_error().decode(), (changes, _abi.lib().vvli_cuda_last_error())


def test_struct_layouts():
    assert ctypes.sizeof(_abi.CPagedPlanArgs) == (5 + 13) * 8
    assert ctypes.sizeof(_abi.CQkRopeArgs) == 12 * 8 + 4 * 4 + 11 * 8 and _abi.CQkRopeArgs.q.offset == 112
    assert ctypes.sizeof(_abi.CVerifyArgs) == (5 + 8) * 8
    assert ctypes.sizeof(_abi.CPagedAttnArgs) == 13 * 8 + 4 * 4 + 11 * 8 and _abi.CPagedAttnArgs.q.offset == 120


def test_plan_refusals():
    fn = _abi.lib().vvli_cuda_paged_plan
    good = _abi.CPagedPlanArgs(4, 64, 100, 8, 16, *[PTR] * 13)
    assert fn(0, None, None) == INVALID
    for changes, text in (
            ({"requests": 0}, "requests"), ({"requests": 8193}, "requests"), ({"page_size": 48}, "page_size"),
            ({"page_size": 256}, "page_size"), ({"free_entries": 0}, "free_entries"), ({"free_entries": 1 << 31}, "free_entries"),
            ({"table_width": 0}, "table_width"), ({"table_width": 1 << 31}, "table_width"),
            ({"max_tokens": 1 << 31}, "max_tokens"), ({"context": None}, "null"), ({"status": None}, "null"),
            ({"slots": None}, "null"), ({"positions": PTR + 2}, "aligned"), ({"cu_new": PTR + 1}, "aligned")):
        refused(fn, good, changes, text)


def test_qk_refusals():
    fn = _abi.lib().vvli_cuda_qk_rope_write
    good = _abi.CQkRopeArgs(5, 8, 2, 64, 32, 16, 10, 2 * 16 * 64, 512, 128, 128, 512, 0, 1, 0, 1e-6, *[PTR] * 11)
    assert fn(0, None, None) == INVALID
    for changes, text in (
            ({"tokens": 1 << 31}, "tokens"), ({"q_heads": 0}, "heads"), ({"kv_heads": 513}, "heads"),
            ({"head_dim": 72}, "head_dim"), ({"head_dim": 272}, "head_dim"), ({"rotary_pairs": 12}, "rotary_pairs"),
            ({"rotary_pairs": 40}, "rotary_pairs"), ({"page_size": 8}, "page_size"), ({"pages": 0}, "pages"),
            ({"page_stride": 2 * 16 * 64 - 8}, "page_stride"), ({"page_stride": 2 * 16 * 64 + 4}, "page_stride"),
            ({"q_stride": 504}, "strides"), ({"k_stride": 132}, "strides"), ({"v_stride": 64}, "strides"),
            ({"out_stride": 0}, "strides"), ({"dtype": 2}, "dtype"), ({"norm": 3}, "norm"), ({"eps": -1.0}, "eps"),
            ({"eps": float("nan")}, "eps"), ({"q": None}, "null"), ({"v_cache": None}, "null"), ({"slots": None}, "null"),
            ({"positions": None}, "null"), ({"inv_freq": None}, "null"), ({"k": PTR + 8}, "aligned"),
            ({"k_weight": PTR + 2}, "aligned"), ({"inv_freq": PTR + 4}, "aligned")):
        refused(fn, good, changes, text)


def test_attention_refusals_and_workspace():
    lib = _abi.lib()
    assert lib.vvli_cuda_paged_attn_workspace_bytes(96) == 0
    small, large = (lib.vvli_cuda_paged_attn_workspace_bytes(d) for d in (64, 128))
    assert 0 < small < large < 64 << 20
    fn = lib.vvli_cuda_paged_attention
    good = _abi.CPagedAttnArgs(4, 9, 14, 2, 64, 16, 10, 2 * 16 * 64, 5, 14 * 64, 14 * 64, 3, 0, 0, 0.125, 0.0, 0,
                               *[PTR] * 10, small)
    assert fn(0, None, None) == INVALID
    for changes, text in (
            ({"requests": 0}, "requests"), ({"requests": 65537}, "requests"), ({"head_dim": 96}, "head_dim"),
            ({"q_heads": 15}, "q_heads"), ({"q_heads": 514}, "q_heads"), ({"kv_heads": 0}, "q_heads"),
            ({"tokens": (1 << 31) // 14 + 1}, "tokens"), ({"page_size": 24}, "page_size"), ({"pages": 0}, "pages"),
            ({"pages": 1 << 27}, "pages"), ({"page_stride": 2 * 16 * 64 + 2}, "page_stride"),
            ({"page_stride": 16 * 64}, "page_stride"), ({"table_width": 0}, "table_width"),
            ({"q_stride": 13 * 64}, "strides"), ({"out_stride": 14 * 64 + 4}, "strides"),
            ({"window": 1 << 31}, "window"), ({"dtype": 2}, "dtype"), ({"scale": float("inf")}, "scale"),
            ({"softcap": -1.0}, "softcap"), ({"softcap": float("nan")}, "softcap"), ({"q": None}, "null"),
            ({"workspace": None}, "null"), ({"seq_len": None}, "null"), ({"v_cache": PTR + 8}, "aligned"),
            ({"lse": PTR + 2}, "aligned"), ({"workspace": PTR + 128}, "workspace"),
            ({"workspace_bytes": small - 1}, "workspace_bytes")):
        refused(fn, good, changes, text)


def test_verify_refusals():
    fn = _abi.lib().vvli_cuda_verify_drafts
    good = _abi.CVerifyArgs(2, 6, 100, 100, 100, *[PTR] * 8)
    assert fn(0, None, None) == INVALID
    for changes, text in (
            ({"requests": 0}, "requests"), ({"requests": 65536}, "requests"), ({"rows": 1 << 31}, "rows"),
            ({"vocab": 0}, "vocab"), ({"vocab": (1 << 30) + 1}, "vocab"), ({"target_stride": 99}, "strides"),
            ({"draft_stride": 99}, "strides"), ({"target": None}, "null"), ({"out_tokens": None}, "null"),
            ({"draft": PTR + 2}, "aligned"), ({"u_sample": PTR + 1}, "aligned")):
        refused(fn, good, changes, text)


def test_wrappers_refuse_host_tensors():
    torch = pytest.importorskip("torch")
    from vvli_b200 import paged, speculative
    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError):
        paged.plan_step(i, i, i, i.view(4, 1), i, i[:1], 16, 4)
    h = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    c = torch.zeros(3, 2, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        paged.qk_norm_rope_write(h, h, h, c, c, i)
    with pytest.raises(ValueError):
        speculative.verify_drafts(torch.zeros(4, 8), None, i, i, torch.zeros(4), torch.zeros(1))


def test_attention_refuses_scores_out_of_range():
    # scale / softcap past fp32 would make a score of 0 NaN, a cap or scale times log2(e) past it an infinity
    lib = _abi.lib()
    good = _abi.CPagedAttnArgs(4, 9, 14, 2, 64, 16, 10, 2 * 16 * 64, 5, 14 * 64, 14 * 64, 3, 0, 0, 0.125, 0.0, 0,
                               *[PTR] * 10, lib.vvli_cuda_paged_attn_workspace_bytes(64))
    for changes in ({"softcap": 1e-40}, {"softcap": 2e-38, "scale": -8.0}, {"softcap": 3e38}, {"scale": 3e38}, {"scale": -3e38}):
        refused(lib.vvli_cuda_paged_attention, good, changes, "fp32")
