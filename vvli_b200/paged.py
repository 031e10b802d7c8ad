"""Host side of the paged serving step (include/vvli_cuda.h: vvli_cuda_paged_plan,
vvli_cuda_qk_rope_write, vvli_cuda_paged_attention).

The reference keeps one contiguous fp32 cache per sequence (KVCache,
src/llm.zig:539-606) and moves one token at a time (src/llm.zig:702-709).
These operators serve many requests, each with any number of new tokens, over
16-bit pages that the caller owns:

    step = plan_step(context, new, owned, block_table, free_pages, free_count, page_size, rows)
    q = qk_norm_rope_write(q, k, v, k_cache, v_cache, step.slots, step.positions, inv_freq, ...)
    out = attention(q, k_cache, v_cache, block_table, step.cu_new, step.seq_len, max_new)

with attention = PagedAttention(q_heads, kv_heads, head_dim, page_size), which
keeps the workspace; vvli_b200.speculative.verify_drafts ends a step of drafts.
A cache is a [pages][kv heads][page_size][head_dim] tensor (pages may be
further apart).  Device memory is handled with torch tensors (plumbing only).
Work is queued on ``stream`` (the current stream of the tensors' device when
None); tensors used on another stream than their own must outlive that work.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _abi
from .errors import check

_DTYPES = {torch.bfloat16: 0, torch.float16: 1}
_NORMS = {"none": 0, None: 0, "head": 1, "row": 2}


def _stream(device: torch.device, stream) -> int:
    return (torch.cuda.current_stream(device) if stream is None else stream).cuda_stream


def _empty(shape, dtype, device, stream):
    """An output, allocated on the stream that writes it."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    with torch.cuda.stream(stream):
        return torch.empty(shape, dtype=dtype, device=device)


def _ints(who: str, name: str, t, device, n=None):
    """t as a contiguous int32 tensor of `device` with at least n entries."""
    if t.dtype != torch.int32 or t.device != device or not t.is_contiguous() or (n is not None and t.numel() < n):
        raise ValueError(f"{who}: {name} must be a contiguous int32 tensor on {device}"
                         + (f" with at least {n} entries" if n is not None else ""))
    return t.data_ptr()


def _cache_layout(who: str, k_cache, v_cache, heads: int, d: int, dtype, device):
    """(pages, page_size, page_stride) of a pair of caches."""
    shape, strides = k_cache.shape, k_cache.stride()
    if k_cache.dim() != 4 or v_cache.shape != shape or v_cache.stride() != strides:
        raise ValueError(f"{who}: k_cache and v_cache must be alike, [pages][kv heads][page_size][head_dim]")
    if shape[1] != heads or shape[3] != d or strides[1:] != (shape[2] * d, d, 1):
        raise ValueError(f"{who}: the caches' pages must be contiguous [{heads}][page_size][{d}]")
    for c in (k_cache, v_cache):
        if c.dtype != dtype or c.device != device:
            raise ValueError(f"{who}: the caches must be {dtype} on {device}")
    return shape[0], shape[2], strides[0] if shape[0] > 1 else shape[1] * shape[2] * d


def _heads(who: str, name: str, x, dtype, device):
    """Row stride of a [tokens][heads][d] tensor whose rows are contiguous."""
    if x.dim() != 3 or x.dtype != dtype or x.device != device:
        raise ValueError(f"{who}: {name} must be a [tokens][heads][head_dim] {dtype} tensor on {device}")
    n, h, d = x.shape
    s = x.stride()
    if (d > 1 and s[2] != 1) or (h > 1 and s[1] != d):
        raise ValueError(f"{who}: the rows of {name} must be contiguous")
    return s[0] if n > 1 else h * d


class StepPlan(NamedTuple):
    """What plan_step gives; all int32 on the device."""
    cu_new: torch.Tensor      # [requests + 1] request b's rows are cu_new[b] .. cu_new[b + 1]
    seq_len: torch.Tensor     # [requests] tokens in the cache after the step, 0 for an unserved request
    positions: torch.Tensor   # [rows]
    slots: torch.Tensor       # [rows] page * page_size + offset, -1: none
    owned: torch.Tensor       # [requests] pages owned after the step
    free_count: torch.Tensor  # [1] pages left on the stack
    status: torch.Tensor      # [requests] 0 planned, 1 pages ran out, 2 table row too short, 3 rows past max_tokens


def plan_step(context, new, owned, block_table, free_pages, free_count, page_size: int, max_tokens: int,
              inplace: bool = False, stream=None) -> StepPlan:
    """Pages, positions and cache slots of one step (vvli_cuda_paged_plan).

    context, new, owned: int32 [requests], each request's cached tokens, new
    tokens and owned pages; block_table: int32 [requests][width], extended in
    place; free_pages: int32, a stack of which the first free_count[0]
    entries are free.  max_tokens: rows of the step (a captured step may have
    more than are used).  With inplace=True, owned and free_count are updated
    themselves (and are the plan's)."""
    who, dev = "plan_step", context.device
    if dev.type != "cuda":
        raise ValueError("plan_step: context must be a CUDA tensor")
    B = context.numel()
    if block_table.dim() != 2 or block_table.shape[0] < B:
        raise ValueError("plan_step: block_table must be [requests][width]")
    max_tokens = int(max_tokens)
    if max_tokens < 0:
        raise ValueError("plan_step: max_tokens must be >= 0")
    sizes = [B + 1, B, max_tokens, max_tokens, B, 1, B]
    buf = _empty((sum(sizes),), torch.int32, dev, stream)
    at = buf.data_ptr()
    ptr = []
    for n in sizes:
        ptr.append(at)
        at += 4 * n
    own_in, free_in = _ints(who, "owned", owned, dev, B), _ints(who, "free_count", free_count, dev, 1)
    a = _abi.CPagedPlanArgs(
        B, int(page_size), free_pages.numel(), block_table.shape[1], max_tokens, _ints(who, "context", context, dev),
        _ints(who, "new", new, dev, B), own_in, _ints(who, "block_table", block_table, dev),
        _ints(who, "free_pages", free_pages, dev), free_in, ptr[0], ptr[1], ptr[2], ptr[3],
        own_in if inplace else ptr[4], free_in if inplace else ptr[5], ptr[6])
    check(_abi.lib().vvli_cuda_paged_plan(dev.index, ctypes.byref(a), _stream(dev, stream)))
    out = buf.split(sizes)
    if inplace:
        out = out[:4] + (owned, free_count, out[6])
    return StepPlan(*out)


def qk_norm_rope_write(q, k, v, k_cache, v_cache, slots, positions=None, inv_freq=None, q_weight=None, k_weight=None,
                       norm: str = "head", eps: float = 1e-6, interleaved: bool = False, out=None, stream=None):
    """RMSNorm of q and k, rotary positions and the cache write (vvli_cuda_qk_rope_write).

    q [tokens][q heads][d], k and v [tokens][kv heads][d]: bf16 or fp16 views
    with contiguous rows (of a fused projection, say).  norm: "head" (weights
    [d]), "row" (OLMoE: over all heads, weights [heads * d]) or "none"; a weight
    of None counts as ones.  inv_freq: float64 radians per position of each
    rotary pair, None for no rotation.  slots and positions: int32 [tokens]; a
    slot of -1 writes no k and v.  Returns the normed, turned q: ``out``
    (which may be q) or a new tensor."""
    who, dev, dtype = "qk_norm_rope_write", q.device, q.dtype
    if dev.type != "cuda" or dtype not in _DTYPES:
        raise ValueError("qk_norm_rope_write: q must be a bf16 or fp16 CUDA tensor")
    if norm not in _NORMS:
        raise ValueError("qk_norm_rope_write: norm must be 'head', 'row' or 'none'")
    qs, ks, vs = (_heads(who, n, x, dtype, dev) for n, x in (("q", q), ("k", k), ("v", v)))
    T, hq, d = q.shape
    hk = k.shape[1]
    if k.shape != (T, hk, d) or v.shape != (T, hk, d):
        raise ValueError("qk_norm_rope_write: k and v must be [tokens][kv heads][head_dim] with q's tokens and head_dim")
    pages, page_size, page_stride = _cache_layout(who, k_cache, v_cache, hk, d, dtype, dev)
    pairs = 0
    if inv_freq is not None:
        pairs = inv_freq.numel()
        if inv_freq.dtype != torch.float64 or inv_freq.device != dev or not inv_freq.is_contiguous():
            raise ValueError(f"qk_norm_rope_write: inv_freq must be a contiguous float64 tensor on {dev}")
        if positions is None:
            raise ValueError("qk_norm_rope_write: a rotation needs positions")
    for name, w, n in (("q_weight", q_weight, hq), ("k_weight", k_weight, hk)):
        n = n * d if norm == "row" else d
        if w is not None and (w.dtype != dtype or w.device != dev or w.numel() != n or not w.is_contiguous()):
            raise ValueError(f"qk_norm_rope_write: {name} must be {n} contiguous {dtype} values on {dev}")
    if out is None:
        out = _empty((T, hq, d), dtype, dev, stream)
    elif out.shape != q.shape:
        raise ValueError("qk_norm_rope_write: out must have q's shape")
    a = _abi.CQkRopeArgs(
        T, hq, hk, d, pairs, page_size, pages, page_stride, qs, ks, vs, _heads(who, "out", out, dtype, dev),
        _DTYPES[dtype], _NORMS[norm], int(bool(interleaved)), float(eps), q.data_ptr(), k.data_ptr(), v.data_ptr(),
        out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), None if q_weight is None else q_weight.data_ptr(),
        None if k_weight is None else k_weight.data_ptr(),
        None if positions is None else _ints(who, "positions", positions, dev, T), _ints(who, "slots", slots, dev, T),
        None if inv_freq is None else inv_freq.data_ptr())
    if T:
        check(_abi.lib().vvli_cuda_qk_rope_write(dev.index, ctypes.byref(a), _stream(dev, stream)))
    return out


class PagedAttention:
    """Attention of the requests' new tokens over their pages (vvli_cuda_paged_attention).

    Row i of request b (q rows cu_new[b] ..) sees the keys up to its position
    seq_len[b] - new[b] + i, with ``window`` > 0 only the last ``window`` of them;
    scores are scale * q.k (1 / sqrt(head_dim) by default), capped by
    softcap * tanh(s / softcap) when softcap > 0, plus alibi[head] * (key
    position - query position) when alibi (float32 [q_heads]) is given.  The
    workspace (its size depends on head_dim alone) is allocated here: calls of
    one object, and graphs captured from them, must not run at the same time.
    """

    def __init__(self, q_heads: int, kv_heads: int, head_dim: int, page_size: int, dtype=torch.bfloat16, scale=None,
                 softcap: float = 0.0, window: int = 0, alibi=None, device: int | torch.device | None = None):
        if dtype not in _DTYPES:
            raise ValueError("PagedAttention: dtype must be bf16 or fp16")
        need = int(_abi.lib().vvli_cuda_paged_attn_workspace_bytes(max(0, int(head_dim))))
        if need == 0:
            raise ValueError("PagedAttention: head_dim must be 64 or 128")
        if device is None:
            device = torch.cuda.current_device()
        self.device = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
        if alibi is not None and (alibi.dtype != torch.float32 or alibi.numel() != q_heads or not alibi.is_contiguous()
                                  or alibi.device != self.device):
            raise ValueError(f"PagedAttention: alibi must be {q_heads} contiguous float32 values on {self.device}")
        self.q_heads, self.kv_heads, self.head_dim, self.page_size = q_heads, kv_heads, head_dim, page_size
        self.dtype, self.alibi = dtype, alibi
        self.scale = float(head_dim) ** -0.5 if scale is None else float(scale)
        self.softcap, self.window = float(softcap), int(window)
        if self.window < 0:
            raise ValueError("PagedAttention: window must be >= 0")
        self._ws = torch.empty(need, dtype=torch.uint8, device=self.device)
        self._ws[:4].zero_()

    def __call__(self, q, k_cache, v_cache, block_table, cu_new, seq_len, max_new: int, out=None, lse=False, stream=None):
        """q: [rows][q_heads][head_dim]; block_table: int32 [requests][width]; cu_new: int32 [requests + 1] and seq_len:
        int32 [requests], as plan_step gives them; max_new: the longest request's new tokens (picks the kernel).
        Returns out ([rows][q_heads][head_dim], new unless given; rows of no request are not written), and with
        lse=True, or a float32 [rows][q_heads] tensor for it, (out, lse)."""
        who, dev, dtype = "PagedAttention", self.device, self.dtype
        qs = _heads(who, "q", q, dtype, dev)
        T, hq, d = q.shape
        if hq != self.q_heads or d != self.head_dim:
            raise ValueError(f"PagedAttention: q must be [rows][{self.q_heads}][{self.head_dim}]")
        pages, page_size, page_stride = _cache_layout(who, k_cache, v_cache, self.kv_heads, d, dtype, dev)
        if page_size != self.page_size:
            raise ValueError(f"PagedAttention: the caches' pages must have {self.page_size} positions")
        B = seq_len.numel()
        if block_table.dim() != 2 or block_table.shape[0] < B:
            raise ValueError("PagedAttention: block_table must be [requests][width]")
        if out is None:
            out = _empty((T, hq, d), dtype, dev, stream)
        elif out.shape != q.shape:
            raise ValueError("PagedAttention: out must have q's shape")
        if lse is True:
            lse = _empty((T, hq), torch.float32, dev, stream)
        elif lse is not False and (lse.dtype != torch.float32 or lse.device != dev or tuple(lse.shape) != (T, hq)
                                   or not lse.is_contiguous()):
            raise ValueError(f"PagedAttention: lse must be a contiguous [{T}][{hq}] float32 tensor on {dev}")
        a = _abi.CPagedAttnArgs(
            B, T, hq, self.kv_heads, d, page_size, pages, page_stride, block_table.shape[1], qs,
            _heads(who, "out", out, dtype, dev), max(0, int(max_new)), self.window, _DTYPES[dtype], self.scale, self.softcap, 0,
            q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(),
            None if lse is False else lse.data_ptr(), None if self.alibi is None else self.alibi.data_ptr(),
            _ints(who, "block_table", block_table, dev), _ints(who, "cu_new", cu_new, dev, B + 1),
            _ints(who, "seq_len", seq_len, dev), self._ws.data_ptr(), self._ws.numel())
        check(_abi.lib().vvli_cuda_paged_attention(dev.index, ctypes.byref(a), _stream(dev, stream)))
        return out if lse is False else (out, lse)

    def status(self) -> int:
        """0, or VVLI_ERR_TIMEOUT (22) once a bounded wait of a call has given up (synchronises)."""
        return int(self._ws[:4].view(torch.int32).item())
