"""Oracles of the packed serving step: batch layout, rotary positions, packed and tree attention, draft verification, in
64 bits and one sequence at a time.  Test infrastructure only (see oracle/__init__.py)."""

from __future__ import annotations

import math

import torch

from .paged_decode import gather_kv


def half_step(dtype: torch.dtype) -> float:
    """The largest relative error of one rounding to `dtype`."""
    return torch.finfo(dtype).eps / 2


def batch_layout_ref(block_table, context_lens, new_lens, free_pages, page, num_tokens):
    """(block_table, seq_lens, cu_new, positions, seq_ids, slots, pages_needed) as lists and a new table."""
    table, free = block_table.clone(), free_pages.tolist()
    W = table.shape[1]
    seq_lens, cu, pos, ids, slots, needed = [], [0], [], [], [], 0
    for s, (c, n) in enumerate(zip(context_lens.tolist(), new_lens.tolist())):
        c = max(c, 0)
        n = min(max(n, 0), num_tokens - cu[-1])
        for p in range(min(-(-c // page), W), min(-(-(c + n) // page), W)):
            table[s, p] = free[needed] if needed < len(free) else -1
            needed += 1
        for t in range(c, c + n):
            entry = int(table[s, t // page]) if t // page < W else -1
            pos.append(t)
            ids.append(s)
            slots.append(entry * page + t % page if entry >= 0 else -1)
        seq_lens.append(c + n)
        cu.append(cu[-1] + n)
    pad = num_tokens - len(pos)
    return table, seq_lens, cu, pos + [0] * pad, ids + [-1] * pad, slots + [-1] * pad, [needed]


def rope_ref(x, positions, inv_freq, interleaved: bool, inverse: bool = False, scale: float = 1.0):
    """(result, bound) in float64: the rotation, and how far a 32-bit computation rounded once to x's type may be off.

    The bound: the angle's remainder in turns is rounded once below 1/2 (2^-26), 2 pi times that in the angle; sine and
    cosine are good to 4 half steps of 32 bits, each product and the sum to one more; then half a step of x's type."""
    half = inv_freq.numel()
    xd = x.double()
    t = positions.double()[:, None, None] * inv_freq.double()
    c, s = torch.cos(t) * scale, torch.sin(t) * (-scale if inverse else scale)
    if interleaved:
        a, b = xd[..., 0 : 2 * half : 2], xd[..., 1 : 2 * half : 2]
    else:
        a, b = xd[..., :half], xd[..., half : 2 * half]
    out, slack = xd.clone(), torch.zeros_like(xd)
    y0, y1 = a * c - b * s, a * s + b * c
    err = (a.abs() + b.abs()) * abs(scale) * (2 * math.pi * 2.0**-26 + 8 * 2.0**-24)
    for buf, u, v in ((out, y0, y1), (slack, err, err)):
        if interleaved:
            buf[..., 0 : 2 * half : 2], buf[..., 1 : 2 * half : 2] = u, v
        else:
            buf[..., :half], buf[..., half : 2 * half] = u, v
    rounding = half_step(x.dtype) * out.abs() + (2.0**-25 if x.dtype == torch.float16 else 0.0)  # fp16: half the smallest step
    rounding[..., 2 * half :] = 0
    return out, slack + rounding


def attention_ref(q, k, v, visible, scale: float | None = None):
    """(result, bound) in float64 for q [n, Hq, D], k, v [m, Hkv, D], visible bool [n, m]; a query that sees nothing: zeros.

    The bound, with h = half a step of the 16-bit type and f = 2^-24: a score of D products summed in 32 bits is off by
    at most D f (scale |q| . |k|), its product with the scale and the subtraction of the maximum by 4 f (|s| + |max|); with
    d the largest of these, weights move by a factor e^(2 d) at most; each weight is rounded to 16 bits once (h) and again where its sum is taken from the
    rounded ones (h); the accumulation over m keys adds (m + 64) f; the result is rounded once (h).

    fp16 weights below 2^-14 are off by up to t = 2^-25 instead, in the result and in the weights' sum: t (sum |v| + n |out|) over that
    sum, n the visible keys.  A weight is exp(score - r) with r a maximum of scores seen so far, which the true maximum is never below, and is only ever scaled
    down afterwards, so that the weights' sum is at least that of exp(score - true maximum), but for e^d."""
    n, hq, D = q.shape
    m, hkv = k.shape[0], k.shape[1]
    scale = 1 / math.sqrt(D) if scale is None else scale
    h, f = half_step(q.dtype), 2.0**-24
    out = torch.zeros(n, hq, D, dtype=torch.float64)
    bound = torch.zeros_like(out)
    if m == 0:
        return out, bound
    tiny = 2.0**-25 if q.dtype == torch.float16 else 0.0
    for j in range(hq):
        kk, vv, qq = k[:, j // (hq // hkv)].double(), v[:, j // (hq // hkv)].double(), q[:, j].double()
        s = (qq @ kk.t()) * scale
        s = torch.where(visible, s, -math.inf)
        mag = torch.where(visible, (qq.abs() @ kk.abs().t()) * scale, 0.0)
        top = s.amax(-1, keepdim=True)
        off = mag * D * f + 4 * f * torch.where(visible, s.abs() + top.abs(), 0.0)
        d = off.amax(-1, keepdim=True)
        w = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
        total = w.sum(-1, keepdim=True)
        total = torch.where(total > 0, total, 1.0)
        w = w / total
        out[:, j] = w @ vv
        seen = visible.double()
        small = tiny * torch.exp(2 * d) / total * (seen @ vv.abs() + seen.sum(-1, keepdim=True) * out[:, j].abs())
        bound[:, j] = (torch.expm1(2 * d) + 2 * h + (m + 64) * f) * (w @ vv.abs()) + h * out[:, j].abs() + small + tiny
    return out, bound


def varlen_ref(q, k, v, cu_q, cu_k, is_causal: bool, scale: float | None = None):
    out = torch.zeros(q.shape, dtype=torch.float64)
    bound = torch.zeros_like(out)
    cq, ck = [x.tolist() for x in (cu_q, cu_k)]
    for a, b, c, d in zip(cq, cq[1:], ck, ck[1:]):
        if b <= a:
            continue
        visible = torch.ones(b - a, max(d - c, 0), dtype=torch.bool)
        if is_causal:
            visible = visible.tril(d - c - (b - a))
        out[a:b], bound[a:b] = attention_ref(q[a:b], k[c:d], v[c:d], visible, scale)
    return out, bound


def ancestors_ref(parents: list[int]) -> torch.Tensor:
    """bool [N, N]: j is i or an ancestor of i; a parent outside [0, i) is none."""
    N = len(parents)
    see = torch.eye(N, dtype=torch.bool)
    for i in range(N):
        if 0 <= parents[i] < i:
            see[i] |= see[parents[i]]
    return see


def tree_ref(q, k_cache, v_cache, block_table, seq_lens, parents, scale: float | None = None):
    """q [S, N, Hq, D]; tokens whose page id is outside the cache are dropped."""
    S, N = q.shape[:2]
    P, page = k_cache.shape[:2]
    out = torch.zeros(q.shape, dtype=torch.float64)
    bound = torch.zeros_like(out)
    for s in range(S):
        L = min(max(int(seq_lens[s]), 0), block_table.shape[1] * page)
        ids = block_table[s, : -(-L // page)]
        ok = ((ids >= 0) & (ids < P)).repeat_interleave(page)[:L]
        row = torch.where((ids >= 0) & (ids < P), ids, 0)
        k, v = gather_kv(k_cache, row, L), gather_kv(v_cache, row, L)
        see = ancestors_ref(parents[s].tolist())
        at = torch.arange(L) - (L - N)
        visible = torch.where(at[None] < 0, True, see[:, at.clamp(0, N - 1)]) & ok[None]
        keep = visible.any(0)
        out[s], bound[s] = attention_ref(q[s], k[keep], v[keep], visible[:, keep], scale)
    return out, bound


def verify_ref(target, draft, tokens, parents, uniforms):
    """(path, num_accepted, next_token) as int32 tensors."""
    S, N, V = target.shape
    path = torch.full((S, N), -1, dtype=torch.int32)
    count, last = torch.zeros(S, dtype=torch.int32), torch.full((S,), -1, dtype=torch.int32)
    for s in range(S):
        cur, r, M = 0, target[s, 0].double(), 1.0
        for i in range(1, N):
            t, par = int(tokens[s, i]), int(parents[s, i])
            if par != cur or par >= i or not 0 <= t < V:
                continue
            if draft is None:
                q = torch.zeros(V, dtype=torch.float64)
                q[t] = 1.0
            else:
                q = draft[s, cur].double()
            if float(uniforms[s, i]) * (float(q[t]) * M) < float(r[t]):
                path[s, count[s]] = i
                count[s] += 1
                cur, r, M = i, target[s, i].double(), 1.0
            else:
                left = (r - q * M).clamp(min=0)
                if float(left.sum()) > 0:
                    r, M = left, float(left.sum())
        run = torch.cumsum(r, 0)
        if float(run[-1]) > 0:
            hit = ((run > max(float(uniforms[s, 0]), 0.0) * run[-1]) & (r > 0)).nonzero()
            last[s] = int(hit[0]) if len(hit) else int((r > 0).nonzero()[-1])
    return path, count, last
