"""Plain implementations of the paged serving step in 64 bits, on host lists and torch CPU tensors."""

import math

import torch


def plan(context, new, owned, table, free_pages, free_count, page, max_tokens):
    """What vvli_cuda_paged_plan documents, request by request; table is changed in place."""
    cu, seq, own, status, pos, slot = [0], [], [], [], [0] * max_tokens, [-1] * max_tokens
    lacking = taken = 0
    free = min(max(0, free_count), len(free_pages))
    for b, (c, n, o) in enumerate(zip(context, new, owned)):
        c, n, o = max(0, c), max(0, n), max(0, o)
        row = cu[-1]
        cu.append(row + n)
        st = 3 if n > 0 and 0 < max_tokens < row + n else 2 if -(-(c + n) // page) > len(table[b]) else 0
        need = 0 if st else max(0, -(-(c + n) // page) - o)
        lacking += need
        if need and lacking > free:
            st, need = 1, 0
        for i in range(need):
            table[b][o + i] = free_pages[free - 1 - taken]
            taken += 1
        for i in range(n):
            if row + i < max_tokens:
                pos[row + i] = c + i
                if st == 0:
                    at = table[b][(c + i) // page]
                    slot[row + i] = at * page + (c + i) % page if 0 <= at <= (2**31 - page) // page else -1
        seq.append(0 if st else c + n)
        own.append(o + need)
        status.append(st)
    return cu, seq, pos, slot, own, [free - taken], status


def qk_rows(x, weight, norm, eps, positions, inv_freq, interleaved):
    """Normed and turned rows [T][h][d] in float64."""
    y = x.double()
    if norm != "none":
        dims = (1, 2) if norm == "row" else (2,)
        y = y / torch.sqrt((y * y).mean(dim=dims, keepdim=True) + eps)
        if weight is not None:
            y = y * weight.double().view(*((x.shape[1], x.shape[2]) if norm == "row" else (x.shape[2],)))
    out = y.clone()
    if inv_freq is not None:
        m = inv_freq.numel()
        a = positions.double()[:, None, None] * inv_freq
        i, j = (slice(0, 2 * m, 2), slice(1, 2 * m, 2)) if interleaved else (slice(0, m), slice(m, 2 * m))
        out[..., i] = y[..., i] * a.cos() - y[..., j] * a.sin()
        out[..., j] = y[..., j] * a.cos() + y[..., i] * a.sin()
    return out


def attention(q, k_cache, v_cache, table, cu_new, seq_len, scale, window=0, softcap=0.0, alibi=None):
    """Rows of every request in float64: (out, lse), untouched rows NaN. Keys of pages outside the cache are zeros."""
    T, hq, d = q.shape
    pages, hk, page, _ = k_cache.shape
    out = torch.full((T, hq, d), math.nan, dtype=torch.float64)
    lse = torch.full((T, hq), math.nan, dtype=torch.float64)
    for b, end in enumerate(seq_len):
        end = min(end, len(table[b]) * page)
        r0, r1 = min(cu_new[b], T), min(max(cu_new[b], cu_new[b + 1]), T)
        n = cu_new[b + 1] - cu_new[b]
        k = torch.zeros(hk, max(end, 0), d, dtype=torch.float64)
        v = torch.zeros_like(k)
        for j in range(-(-max(end, 0) // page)):
            at = int(table[b][j])
            if 0 <= at < pages:
                m = min(page, end - j * page)
                k[:, j * page:j * page + m] = k_cache[at, :, :m].double()
                v[:, j * page:j * page + m] = v_cache[at, :, :m].double()
        for r in range(r0, r1):
            p = end - n + r - r0
            lo = max(0, p - window + 1) if window else 0
            if p < 0 or lo > p:
                out[r], lse[r] = 0.0, -math.inf
                continue
            kk, vv = (x[:, lo:p + 1].repeat_interleave(hq // hk, 0) for x in (k, v))
            s = torch.einsum("hd,hjd->hj", q[r].double(), kk) * scale
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            if alibi is not None:
                s = s + alibi.double()[:, None] * (torch.arange(lo, p + 1) - p)
            lse[r] = torch.logsumexp(s, -1)
            out[r] = torch.einsum("hj,hjd->hd", torch.exp(s - lse[r][:, None]), vv)
    return out, lse


def verify(target, draft, tokens, cu, u_accept, u_sample):
    """(accepted, out) lists; rows of no request stay None."""
    T, V = target.shape
    accepted, out = [], [None] * T
    for b in range(len(cu) - 1):
        r0, r1 = min(cu[b], T), min(cu[b + 1], T)
        if r0 >= r1:
            accepted.append(0)
            continue
        n = 0
        while r0 + n < r1 - 1:
            x, r = int(tokens[r0 + n + 1]), r0 + n
            if not 0 <= x < V:
                break
            q = 1.0 if draft is None else float(draft[r, x])
            if not float(u_accept[r]) * q < float(target[r, x]):
                break
            n += 1
        row = r0 + n
        w = target[row].double().clone()
        if row < r1 - 1:
            if draft is None:
                if 0 <= int(tokens[row + 1]) < V:
                    w[int(tokens[row + 1])] = 0
            else:
                w = w - draft[row].double()
            w = torch.where(w > 0, w, torch.zeros_like(w))
            if not w.sum() > 0:
                w = target[row].double()
        w = torch.where(w > 0, w, torch.zeros_like(w))
        c = torch.cumsum(w, 0)
        hit = (c > float(u_sample[b]) * c[-1]) & (w > 0)
        some = torch.nonzero(hit if hit.any() else w > 0)
        token = 0 if not len(some) else int(some[0] if hit.any() else some[-1])
        accepted.append(n)
        for r in range(r0, r1):
            out[r] = int(tokens[r + 1]) if r < row else token if r == row else -1
    return accepted, out
