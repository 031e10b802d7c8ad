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

from typing import NamedTuple

import torch

from . import _abi
from .errors import check

_DTYPES = {torch.bfloat16: 0, torch.float16: 1}
_NORMS = {"none": 0, None: 0, "head": 1, "row": 2}


# The wrappers' own time counts beside kernels of a few microseconds: devices are
# compared by index, and the current stream's handle comes straight from torch's
# C module (torch.cuda.current_stream builds an object for it, 2 us).
_current_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _stream(index: int, stream) -> int:
    return _current_stream(index) if stream is None else stream.cuda_stream


def _empty(shape, dtype, device, stream):
    """An output, allocated on the stream that writes it."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    with torch.cuda.stream(stream):
        return torch.empty(shape, dtype=dtype, device=device)


def _empty_like(x, stream):
    """A contiguous output in the shape of x, whose rows are (half the time of torch.empty by shape and type)."""
    if stream is None:
        return torch.empty_like(x)
    with torch.cuda.stream(stream):
        return torch.empty_like(x)


def _ints(who: str, name: str, t, index: int, n: int = 0) -> int:
    """Address of a contiguous int32 tensor of CUDA device `index` with at least n entries."""
    if t.dtype is not torch.int32 or t.get_device() != index or not t.is_contiguous() or t.numel() < n:
        raise ValueError(f"{who}: {name} must be a contiguous int32 tensor on cuda:{index} with at least {n} entries")
    return t.data_ptr()


def _cache_layout(who: str, k_cache, v_cache, heads: int, d: int, dtype, index: int):
    """(pages, page_size, page_stride) of a pair of caches."""
    shape, strides = k_cache.shape, k_cache.stride()
    if len(shape) != 4 or v_cache.shape != shape or v_cache.stride() != strides:
        raise ValueError(f"{who}: k_cache and v_cache must be alike, [pages][kv heads][page_size][head_dim]")
    pages, h, page_size, dc = shape
    apart, s1, s2, s3 = strides
    if h != heads or dc != d or s3 != 1 or s2 != d or (s1 != page_size * d and h > 1):
        raise ValueError(f"{who}: the caches' pages must be contiguous [{heads}][page_size][{d}]")
    if (k_cache.dtype is not dtype or v_cache.dtype is not dtype or k_cache.get_device() != index
            or v_cache.get_device() != index):
        raise ValueError(f"{who}: the caches must be {dtype} on cuda:{index}")
    return pages, page_size, apart if pages > 1 else h * page_size * d


def _heads(who: str, name: str, x, shape, dtype, index: int) -> int:
    """Row stride of a tensor of the given [tokens][heads][d] shape whose rows are contiguous."""
    if x.shape != shape or x.dtype is not dtype or x.get_device() != index:
        raise ValueError(f"{who}: {name} must be a {list(shape)} {dtype} tensor on cuda:{index}")
    apart, sh, sd = x.stride()
    n, h, d = shape
    if (sd != 1 or sh != d) and ((sd != 1 and d > 1) or (sh != d and h > 1)):
        raise ValueError(f"{who}: the rows of {name} must be contiguous")
    return apart if n > 1 else h * d


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
    who, dev = "plan_step", context.get_device()
    if dev < 0:
        raise ValueError("plan_step: context must be a CUDA tensor")
    B = context.numel()
    if block_table.dim() != 2 or block_table.shape[0] < B:
        raise ValueError("plan_step: block_table must be [requests][width]")
    if max_tokens < 0:
        raise ValueError("plan_step: max_tokens must be >= 0")
    sizes = (B + 1, B, max_tokens, max_tokens, B, 1, B)
    if B == 0:
        return _plan_of_nothing(owned, free_pages, free_count, dev, max_tokens, inplace, stream)
    buf = _empty(4 * B + 2 * max_tokens + 2, torch.int32, context.device, stream)
    cu = buf.data_ptr()
    seq = cu + 4 * (B + 1)
    pos = seq + 4 * B
    slots = pos + 4 * max_tokens
    own = slots + 4 * max_tokens
    own_in, free_in = _ints(who, "owned", owned, dev, B), _ints(who, "free_count", free_count, dev, 1)
    a = _abi.pack_paged_plan(
        B, page_size, free_pages.numel(), block_table.shape[1], max_tokens, _ints(who, "context", context, dev),
        _ints(who, "new", new, dev, B), own_in, _ints(who, "block_table", block_table, dev),
        _ints(who, "free_pages", free_pages, dev), free_in, cu, seq, pos, slots, own_in if inplace else own,
        free_in if inplace else own + 4 * B, own + 4 * B + 4)
    check(_abi.lib().vvli_cuda_paged_plan(dev, a, _stream(dev, stream)))
    out = buf.split_with_sizes(sizes)
    if inplace:
        out = (*out[:4], owned, free_count, out[6])
    return StepPlan(*out)


def _plan_of_nothing(owned, free_pages, free_count, dev: int, max_tokens: int, inplace: bool, stream) -> StepPlan:
    """The plan of a step without requests, which the library does not take."""
    _ints("plan_step", "owned", owned, dev), _ints("plan_step", "free_pages", free_pages, dev)
    _ints("plan_step", "free_count", free_count, dev, 1)
    with torch.cuda.device(dev), torch.cuda.stream(stream):  # None: the current one
        left = free_count[:1].clamp(0, free_pages.numel())
        if inplace:
            free_count[:1].copy_(left)
        none, zeros = owned.new_empty(0), owned.new_zeros(1 + max_tokens)
        return StepPlan(zeros[:1], none, zeros[1:], torch.full_like(zeros[1:], -1), owned if inplace else none,
                        free_count if inplace else left, none)


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
    who, dev, dtype = "qk_norm_rope_write", q.get_device(), q.dtype
    if dev < 0 or dtype not in _DTYPES or q.dim() != 3 or k.dim() != 3:
        raise ValueError("qk_norm_rope_write: q and k must be [tokens][heads][head_dim] bf16 or fp16 CUDA tensors")
    if norm not in _NORMS:
        raise ValueError("qk_norm_rope_write: norm must be 'head', 'row' or 'none'")
    T, hq, d = shape = q.shape
    hk = k.shape[1]
    qs = _heads(who, "q", q, shape, dtype, dev)
    ks = _heads(who, "k", k, (T, hk, d), dtype, dev)
    vs = _heads(who, "v", v, (T, hk, d), dtype, dev)
    pages, page_size, page_stride = _cache_layout(who, k_cache, v_cache, hk, d, dtype, dev)
    pairs = freq = pos = qw = kw = 0  # addresses: 0 is null
    if inv_freq is not None:
        if inv_freq.dtype is not torch.float64 or inv_freq.get_device() != dev or not inv_freq.is_contiguous():
            raise ValueError(f"qk_norm_rope_write: inv_freq must be a contiguous float64 tensor on cuda:{dev}")
        if positions is None:
            raise ValueError("qk_norm_rope_write: a rotation needs positions")
        pairs, freq = inv_freq.numel(), inv_freq.data_ptr()
    if positions is not None:
        pos = _ints(who, "positions", positions, dev, T)
    if q_weight is not None:
        qw = _norm_weight("q_weight", q_weight, hq * d if norm == "row" else d, dtype, dev)
    if k_weight is not None:
        kw = _norm_weight("k_weight", k_weight, hk * d if norm == "row" else d, dtype, dev)
    if out is None:
        out, os = _empty_like(q, stream), hq * d
    else:
        os = _heads(who, "out", out, shape, dtype, dev)
    a = _abi.pack_qk_rope(
        T, hq, hk, d, pairs, page_size, pages, page_stride, qs, ks, vs, os, _DTYPES[dtype], _NORMS[norm],
        1 if interleaved else 0, eps, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), k_cache.data_ptr(),
        v_cache.data_ptr(), qw, kw, pos, _ints(who, "slots", slots, dev, T), freq)
    if T:
        check(_abi.lib().vvli_cuda_qk_rope_write(dev, a, _stream(dev, stream)))
    return out


def _norm_weight(name: str, w, n: int, dtype, index: int) -> int:
    if w.dtype is not dtype or w.get_device() != index or w.numel() != n or not w.is_contiguous():
        raise ValueError(f"qk_norm_rope_write: {name} must be {n} contiguous {dtype} values on cuda:{index}")
    return w.data_ptr()


class PagedAttention:
    """Attention of the requests' new tokens over their pages (vvli_cuda_paged_attention).

    Row i of request b (q rows cu_new[b] ..) sees the keys up to its position
    seq_len[b] - new[b] + i, with ``window`` > 0 only the last ``window`` of them;
    scores are scale * q.k (1 / sqrt(head_dim) by default), capped by
    softcap * tanh(s / softcap) when softcap > 0, plus alibi[head] * (key
    position - query position) when alibi (float32 [q_heads]) is given.  The
    workspace (its size depends on head_dim alone) is allocated here: calls of
    one object, and graphs captured from them, must not run at the same time.
    Calls may be on any streams, which have to outlive the object; a graph of
    its calls must not be replayed once it is gone.
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
        if self.device.type != "cuda":
            raise ValueError("PagedAttention: device must be a CUDA device")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        if alibi is not None and (alibi.dtype != torch.float32 or alibi.numel() != q_heads or not alibi.is_contiguous()
                                  or alibi.device != self.device):
            raise ValueError(f"PagedAttention: alibi must be {q_heads} contiguous float32 values on {self.device}")
        self.q_heads, self.kv_heads, self.head_dim, self.page_size = q_heads, kv_heads, head_dim, page_size
        self.dtype, self.alibi = dtype, alibi
        self.scale = float(head_dim) ** -0.5 if scale is None else float(scale)
        self.softcap, self.window = float(softcap), int(window)
        if self.window < 0:
            raise ValueError("PagedAttention: window must be >= 0")
        self._type, self._alibi = _DTYPES[dtype], 0 if alibi is None else alibi.data_ptr()
        with torch.cuda.device(self.device):
            self._ws = torch.empty(need, dtype=torch.uint8, device=self.device)
            self._ws[:4].zero_()
            home = torch.cuda.current_stream()
            if not torch.cuda.is_current_stream_capturing():
                home.synchronize()  # calls may be on any stream: what the memory was used for before is over
        self._ws_at, self._ws_bytes, self._streams = self._ws.data_ptr(), need, {home.cuda_stream}

    def __call__(self, q, k_cache, v_cache, block_table, cu_new, seq_len, max_new: int, out=None, lse=False, stream=None):
        """q: [rows][q_heads][head_dim]; block_table: int32 [requests][width]; cu_new: int32 [requests + 1] and seq_len:
        int32 [requests], as plan_step gives them; max_new: the longest request's new tokens (picks the kernel).
        Returns out ([rows][q_heads][head_dim], new unless given; rows of no request are not written), and with
        lse=True, or a float32 [rows][q_heads] tensor for it, (out, lse)."""
        who, dev, dtype = "PagedAttention", self.device.index, self.dtype
        T, hq, d = shape = (q.shape[0], self.q_heads, self.head_dim)
        qs = _heads(who, "q", q, shape, dtype, dev)
        pages, page_size, page_stride = _cache_layout(who, k_cache, v_cache, self.kv_heads, d, dtype, dev)
        if page_size != self.page_size:
            raise ValueError(f"PagedAttention: the caches' pages must have {self.page_size} positions")
        B = seq_len.numel()
        if block_table.dim() != 2 or block_table.shape[0] < B:
            raise ValueError("PagedAttention: block_table must be [requests][width]")
        if out is None:
            out, os = _empty_like(q, stream), hq * d
        else:
            os = _heads(who, "out", out, shape, dtype, dev)
        lp = 0
        if lse is True:
            lse = _empty((T, hq), torch.float32, self.device, stream)
            lp = lse.data_ptr()
        elif lse is not False:
            if lse.dtype is not torch.float32 or lse.get_device() != dev or lse.shape != (T, hq) or not lse.is_contiguous():
                raise ValueError(f"PagedAttention: lse must be a contiguous [{T}][{hq}] float32 tensor on cuda:{dev}")
            lp = lse.data_ptr()
        a = _abi.pack_paged_attn(
            B, T, hq, self.kv_heads, d, page_size, pages, page_stride, block_table.shape[1], qs, os, max(0, max_new),
            self.window, self._type, self.scale, self.softcap, 0, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
            out.data_ptr(), lp, self._alibi, _ints(who, "block_table", block_table, dev),
            _ints(who, "cu_new", cu_new, dev, B + 1), _ints(who, "seq_len", seq_len, dev), self._ws_at, self._ws_bytes)
        s = _stream(dev, stream)
        if s not in self._streams:  # the workspace goes back to the allocator when that stream is done with it, too
            self._ws.record_stream(torch.cuda.current_stream(dev) if stream is None else stream)
            self._streams.add(s)
        if B:  # a step without requests writes nothing
            check(_abi.lib().vvli_cuda_paged_attention(dev, a, s))
        return out if lse is False else (out, lse)

    def status(self) -> int:
        """0, or VVLI_ERR_TIMEOUT (22) once a bounded wait of a call has given up (synchronises)."""
        return int(self._ws[:4].view(torch.int32).item())
