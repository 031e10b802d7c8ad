"""Verification of drafted tokens (vvli_cuda_verify_drafts, include/vvli_cuda.h).

The reference samples one token per forward (Sampler.next,
src/generator.zig:97-126); this is the sampling step of a decoder that feeds
several drafted tokens at once and keeps those the target model agrees with,
so that the emitted tokens are distributed as the target's.
"""

from __future__ import annotations

import torch

from . import _abi
from .errors import check
from .paged import _empty, _ints, _stream


def _rows_of(name: str, x, index: int, shape=None) -> int:
    if x.dtype is not torch.float32 or x.get_device() != index or x.dim() != 2 or (
            x.stride(1) != 1 and x.shape[1] > 1) or (shape is not None and x.shape != shape):
        raise ValueError(f"verify_drafts: {name} must be a [rows][vocab] float32 tensor on cuda:{index} with contiguous rows")
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _uniform(name: str, u, n: int, index: int) -> int:
    if u.dtype is not torch.float32 or u.get_device() != index or u.numel() < n or not u.is_contiguous():
        raise ValueError(f"verify_drafts: {name} must be {n} contiguous float32 values on cuda:{index}")
    return u.data_ptr()


def verify_drafts(target, draft, tokens, cu_rows, u_accept, u_sample, stream=None):
    """Accepts drafts against the target's probabilities and draws the next token of every request.

    target [rows][vocab]: float32 probabilities after each fed token; draft:
    the drafter's, row r for the draft fed at row r + 1, or None for a drafter
    that does not sample; tokens [rows] int32: the fed tokens (request b's rows
    are cu_rows[b] .. cu_rows[b + 1], the first one not a draft, all others
    drafts: of a prompt only the rows from its last token on, of a request that
    plan_step did not serve none; a step's cu_new is such a cu_rows only where
    every request was served and fed one known token and drafts); u_accept
    [rows] and u_sample [requests]: float32 uniform numbers in [0, 1).
    Returns (accepted [requests], out [rows]) int32: out holds the accepted
    drafts from cu_rows[b] on, then the drawn token, then -1; rows of no
    request are not written."""
    dev = target.get_device()
    if dev < 0:
        raise ValueError("verify_drafts: target must be a CUDA tensor")
    ts = _rows_of("target", target, dev)
    ds = 0 if draft is None else _rows_of("draft", draft, dev, target.shape)
    T, V = target.shape
    B = u_sample.numel()
    ua, us = _uniform("u_accept", u_accept, T, dev), _uniform("u_sample", u_sample, B, dev)
    tok, cu = _ints("verify_drafts", "tokens", tokens, dev, T), _ints("verify_drafts", "cu_rows", cu_rows, dev, B + 1)
    buf = _empty(B + T, torch.int32, target.device, stream)
    if T == 0 or B == 0:  # no request has a row
        with torch.cuda.stream(stream):  # None: the current one
            buf.zero_()
    else:
        at = buf.data_ptr()
        a = _abi.pack_verify(B, T, V, ts, ds, target.data_ptr(), 0 if draft is None else draft.data_ptr(), tok, cu, ua, us,
                             at, at + 4 * B)
        check(_abi.lib().vvli_cuda_verify_drafts(dev, a, _stream(dev, stream)))
    return buf.split_with_sizes((B, T))
