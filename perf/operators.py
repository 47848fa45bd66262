"""The serving operators around the paged KV cache as measured cases: batch layout, rotary positions (alone, with its
gradient, and fused with the cache append), attention over packed prompts, attention of drafted token trees over the
cache, and the verification of drafted tokens.

`run` computes them from elementary torch operations while `own` is false and through `torch.ops.mi355.*` where it is
true; `exact` restates the definitions in 64 bits, one sequence at a time.
"""

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}


# ---- the cases -------------------------------------------------------------------------------------------------------


def listed():
    return [
        # One decode step of a running batch: every sequence adds one token, few of them cross into a new page.
        {"name": "layout_decode_64", "op": "layout", "seqs": 64, "page": 16, "ctx_min": 512, "ctx_max": 8192, "new_min": 1, "new_max": 1, "spare": 0, "shape": 1},
        # A scheduler step that admits many prompts of very different lengths, padded to a fixed number of token rows.
        {"name": "layout_prompts_1000", "op": "layout", "seqs": 1000, "page": 32, "ctx_min": 0, "ctx_max": 2000, "new_min": 0, "new_max": 130, "spare": 77, "shape": 2},
        # The same decode step's queries and keys: rotated, keys and values put into their slots.
        {"name": "rope_append_decode_64", "op": "rope_append", "tokens": 64, "hq": 32, "hkv": 8, "rotary": 128, "interleaved": False, "far": 8192, "factor": 1.0, "page": 16, "pad": 0, "dtype": "bfloat16", "shape": 3},
        # A packed prompt batch far into a stretched context; adjacent pairs, half of the head; the last rows are padding.
        {"name": "rope_append_prompts_8000", "op": "rope_append", "tokens": 8000, "hq": 32, "hkv": 8, "rotary": 64, "interleaved": True, "far": 131072, "factor": 16.0, "page": 64, "pad": 55, "dtype": "float16", "shape": 4},
        # Training: rotation of a query projection and the gradient that goes back through it.
        {"name": "rope_train_16384", "op": "rope_train", "tokens": 16384, "heads": 32, "dim": 128, "rotary": 128, "interleaved": False, "far": 16384, "factor": 1.0, "dtype": "bfloat16", "shape": 5},
        # Short prompts of a chat batch, one-token ones among them, packed without padding.
        {"name": "prompts_short_32", "op": "prompts", "seqs": 32, "len_min": 1, "len_max": 300, "prefix_max": 0, "hq": 32, "hkv": 8, "causal": True, "dtype": "bfloat16", "shape": 6},
        # Chunks of prompts whose earlier part is packed in front of them: more keys than queries, one head of keys for 16.
        {"name": "prompts_chunked_12", "op": "prompts", "seqs": 12, "len_min": 100, "len_max": 700, "prefix_max": 1500, "hq": 16, "hkv": 1, "causal": True, "dtype": "float16", "shape": 7},
        # Long documents packed into one call.
        {"name": "prompts_long_4", "op": "prompts", "seqs": 4, "len_min": 1500, "len_max": 8192, "prefix_max": 0, "hq": 32, "hkv": 8, "causal": True, "dtype": "float16", "shape": 8},
        # One user, a long conversation, a small tree of drafts.
        {"name": "tree_1x32768", "op": "tree", "seqs": 1, "nodes": 7, "branch": 3, "ctx_min": 32768, "ctx_max": 32768, "hq": 32, "hkv": 8, "page": 64, "dtype": "float16", "shape": 9},
        # The decode benchmark's batch with trees of sixteen drafts.
        {"name": "tree_64x8192", "op": "tree", "seqs": 64, "nodes": 16, "branch": 3, "ctx_min": 512, "ctx_max": 8192, "hq": 32, "hkv": 8, "page": 16, "dtype": "bfloat16", "shape": 10},
        # A chain of drafts for a few users, sampled from a draft model.
        {"name": "verify_chain_8", "op": "verify", "seqs": 8, "nodes": 5, "branch": 1, "vocab": 32000, "sampled": True, "shape": 11},
        # Trees whose siblings are drawn from the draft model, over a large vocabulary.
        {"name": "verify_tree_64", "op": "verify", "seqs": 64, "nodes": 13, "branch": 3, "vocab": 131072, "sampled": True, "shape": 12},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["layout", "rope_append", "rope_train", "prompts", "tree", "verify"])
    shape = rng.randrange(1 << 30)
    half = rng.choice(["float16", "bfloat16"])
    page = rng.choice([16, 32, 64, 128, 256])
    if op == "layout":
        ctx = _spread(rng, 16, 8192)
        new = _spread(rng, 1, 512)
        return {"op": op, "seqs": min(_spread(rng, 1, 2000), 200000 // new + 1), "page": page, "ctx_min": rng.choice([0, ctx // 2]), "ctx_max": ctx,
                "new_min": rng.choice([0, 1, new]), "new_max": new, "spare": rng.choice([0, rng.randrange(1, 500)]), "shape": shape}
    if op == "rope_append":
        hkv = rng.choice([1, 2, 4, 8])
        return {"op": op, "tokens": _spread(rng, 1, 8000), "hq": hkv * rng.choice([1, 2, 4]), "hkv": hkv, "rotary": rng.choice([32, 64, 96, 128]),
                "interleaved": rng.random() < 0.5, "far": _spread(rng, 8192, 1 << 20), "factor": rng.choice([1.0, 4.0, 16.0]), "page": page,
                "pad": rng.choice([0, rng.randrange(0, 64)]), "dtype": half, "shape": shape}
    if op == "rope_train":
        dim = rng.choice([64, 80, 96, 128, 256])
        return {"op": op, "tokens": _spread(rng, 1, 8192), "heads": rng.randrange(1, 33), "dim": dim, "rotary": dim if rng.random() < 0.5 else dim // 4 * 2,
                "interleaved": rng.random() < 0.5, "far": _spread(rng, 8192, 1 << 20), "factor": rng.choice([1.0, 4.0]),
                "dtype": rng.choice(["float16", "bfloat16", "float32"]), "shape": shape}
    if op == "prompts":
        longest = _spread(rng, 1, 4096)
        hkv = rng.choice([1, 2, 4, 8])
        hq = hkv * rng.choice([1, 2, 4])
        seqs = max(1, min(_spread(rng, 1, 48), (1 << 31) // (hq * longest * longest)))
        return {"op": op, "seqs": seqs, "len_min": rng.choice([0, 1, longest]), "len_max": longest, "prefix_max": rng.choice([0, 0, longest // 2]),
                "hq": hq, "hkv": hkv, "causal": rng.random() < 0.8, "dtype": half, "shape": shape}
    if op == "tree":
        ctx = _spread(rng, 64, 16384)
        hkv = rng.choice([1, 2, 4, 8])
        return {"op": op, "seqs": max(1, min(_spread(rng, 1, 64), 400000 // ctx)), "nodes": rng.randrange(1, 65), "branch": rng.randrange(1, 5),
                "ctx_min": rng.choice([0, ctx // 8, ctx]), "ctx_max": ctx, "hq": hkv * rng.choice([1, 2, 4, 8]), "hkv": hkv, "page": page, "dtype": half, "shape": shape}
    vocab = _spread(rng, 1000, 131072)
    nodes = rng.randrange(1, 17)
    return {"op": op, "seqs": max(1, min(_spread(rng, 1, 64), 100000000 // (vocab * nodes))), "nodes": nodes, "branch": rng.randrange(1, 4), "vocab": vocab,
            "sampled": rng.random() < 0.7, "shape": shape}


# ---- what a case's sizes are -----------------------------------------------------------------------------------------


def _between(case, lo, hi, salt):
    """One length per sequence: from the case alone, even over the logarithm, the largest among them."""
    rng = random.Random(case["shape"] * 31 + salt)
    got = [lo if hi <= lo else min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo + 1), math.log(hi + 1.999)))) - 1)) for _ in range(case["seqs"])]
    got[rng.randrange(case["seqs"])] = hi
    return got


def _lens(case):
    """(tokens in front, new tokens) of every sequence."""
    if case["op"] == "layout":
        return _between(case, case["ctx_min"], case["ctx_max"], 1), _between(case, case["new_min"], case["new_max"], 2)
    if case["op"] == "prompts":
        return _between(case, 0, case["prefix_max"], 1), _between(case, case["len_min"], case["len_max"], 2)
    return _between(case, case["ctx_min"], case["ctx_max"], 1), [case["nodes"]] * case["seqs"]


def _tree(case):
    """The parents of every sequence's nodes: node 0 is the root, and up to `branch` nodes share a parent."""
    rng = random.Random(case["shape"] * 17 + 3)
    rows = []
    for _ in range(case["seqs"]):
        parents, kids = [-1], [0]
        for i in range(1, case["nodes"]):
            free = [j for j in range(max(0, i - 2 * case["branch"]), i) if kids[j] < case["branch"]]
            p = rng.choice(free) if case["branch"] > 1 else i - 1
            parents.append(p)
            kids[p] += 1
            kids.append(0)
        rows.append(parents)
    return rows


def _inv_freq(rotary, factor, base=10000.0, trained=4096):
    """Rotary frequencies in 64 bits; factor > 1 stretches the slow ones for contexts `factor` times the trained length
    (blended between 1 and 32 turns within it) and scales the result by 0.1 ln(factor) + 1."""
    f = [base ** (-2.0 * i / rotary) for i in range(rotary // 2)]
    if factor > 1:
        keep = [min(1.0, max(0.0, (trained * x / (2 * math.pi) - 1) / 31)) for x in f]
        f = [x * k + x / factor * (1 - k) for x, k in zip(f, keep)]
    return f, 0.1 * math.log(factor) + 1


def work(case):
    op = case["op"]
    if op == "layout":
        ctx, new = _lens(case)
        rows = sum(new) + case["spare"]
        return {"bytes": 16 * case["seqs"] + 16 * rows + 8 * sum(-(-(c + n) // case["page"]) + (-c // case["page"]) for c, n in zip(ctx, new)), "flops": 0}
    if op == "rope_append":
        row = 128 * 2 * (case["hq"] + 2 * case["hkv"])
        return {"bytes": 2 * case["tokens"] * row + 12 * case["tokens"], "flops": 3 * case["tokens"] * (case["hq"] + case["hkv"]) * case["rotary"]}
    if op == "rope_train":
        n = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 4 * n * DTYPES[case["dtype"]].itemsize, "flops": 6 * n}
    if op == "prompts":
        before, new = _lens(case)
        pairs = sum(n * b + (n * (n + 1) // 2 if case["causal"] else n * n) for b, n in zip(before, new))
        return {"bytes": 256 * (2 * case["hq"] * sum(new) + 2 * case["hkv"] * (sum(new) + sum(before))), "flops": 512 * case["hq"] * pairs}
    if op == "tree":
        ctx, new = _lens(case)
        return {"bytes": 512 * case["hkv"] * (sum(ctx) + sum(new)) + 512 * case["hq"] * sum(new) + 4 * sum(-(-(c + n) // case["page"]) for c, n in zip(ctx, new)),
                "flops": 512 * case["hq"] * case["nodes"] * (sum(ctx) + sum(new))}
    return {"bytes": case["seqs"] * (4 * case["vocab"] * (2 if case["sampled"] else 1) + 16 * case["nodes"]), "flops": 3 * case["seqs"] * case["vocab"]}


# ---- inputs ----------------------------------------------------------------------------------------------------------


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 11)
    normal = lambda *size, dtype=torch.float32: torch.randn(*size, generator=g, device=DEV).to(dtype)  # noqa: E731
    op = case["op"]
    s = {"case": case}
    if op == "layout":
        ctx, new = _lens(case)
        page = case["page"]
        have = [-(-c // page) for c in ctx]
        width = max(-(-(c + n) // page) for c, n in zip(ctx, new)) + 3
        need = sum(-(-(c + n) // page) - h for c, n, h in zip(ctx, new, have))
        ids = torch.randperm(sum(have) + need + 100, generator=g, device=DEV).int()
        table = torch.full((case["seqs"], width), -1, dtype=torch.int32, device=DEV)
        table[torch.arange(width, device=DEV)[None] < _i32(have)[:, None]] = ids[: sum(have)]
        return {**s, "table": table, "ctx": _i32(ctx), "new": _i32(new), "free": ids[sum(have):].clone(), "page": page, "rows": max(1, sum(new) + case["spare"])}
    if op in ("rope_append", "rope_train"):
        f, s["scale"] = _inv_freq(case["rotary"], case["factor"])
        s["freq"] = torch.tensor(f, dtype=torch.float64, device=DEV)
        T, dt = case["tokens"], DTYPES[case["dtype"]]
        s["pos"] = torch.randint(0, case["far"], (T,), generator=g, device=DEV, dtype=torch.int32)
        if op == "rope_train":
            s["x"] = normal(T, case["heads"], case["dim"], dtype=dt).requires_grad_()
            s["dy"] = normal(T, case["heads"], case["dim"], dtype=dt)
            return s
        qkv = normal(T, case["hq"] + 2 * case["hkv"], 128, dtype=dt)  # the projection's output, its parts read in place
        s["q"], s["k"], s["v"] = qkv.split([case["hq"], case["hkv"], case["hkv"]], dim=1)
        pages = -(-T // case["page"]) + 3
        s["kc"], s["vc"] = (normal(pages, case["page"], case["hkv"], 128, dtype=dt) for _ in range(2))
        s["slots"] = torch.randperm(pages * case["page"], generator=g, device=DEV)[:T].clone()
        s["slots"][T - min(case["pad"], T - 1):] = -1
        return s
    dt = DTYPES[case.get("dtype", "float32")]
    if op == "prompts":
        before, new = _lens(case)
        lk = [b + n for b, n in zip(before, new)]
        s["q"], s["k"], s["v"] = (normal(max(1, sum(n)), h, 128, dtype=dt) for n, h in ((new, case["hq"]), (lk, case["hkv"]), (lk, case["hkv"])))
        for name, n in (("q", new), ("k", lk)):
            s["cu_" + name] = torch.cat([_i32([0]), torch.cumsum(_i32(n), 0, dtype=torch.int32)])
            s["max_" + name] = max(n)
        return s
    if op == "tree":
        ctx, new = _lens(case)
        lens = [c + n for c, n in zip(ctx, new)]
        page, hkv = case["page"], case["hkv"]
        need = [-(-n // page) for n in lens]
        width = max(need) + 1
        pages = sum(need) + 5
        s["table"] = torch.full((case["seqs"], width), -1, dtype=torch.int32, device=DEV)
        s["table"][torch.arange(width, device=DEV)[None] < _i32(need)[:, None]] = torch.randperm(pages, generator=g, device=DEV)[: sum(need)].int()
        s["kc"], s["vc"] = (normal(pages, page, hkv, 128, dtype=dt) for _ in range(2))
        s["q"] = normal(case["seqs"], case["nodes"], case["hq"], 128, dtype=dt)
        s["lens"], s["parents"] = _i32(lens), _i32(_tree(case))
        return s
    S, N, V = case["seqs"], case["nodes"], case["vocab"]
    logits = 3 * normal(S, N, V)
    s["parents"] = _i32(_tree(case))
    up = s["parents"].clamp(min=0).long()
    if case["sampled"]:  # the draft model is near the target; a node's token is drawn from its parent's row
        s["draft"] = torch.softmax(logits + 0.7 * normal(S, N, V), -1)
        rows = torch.gather(s["draft"], 1, up[..., None].expand(S, N, V))
    else:  # drafts without probabilities: some of the target's likely tokens
        s["draft"] = None
        rows = torch.softmax(2 * torch.gather(logits, 1, up[..., None].expand(S, N, V)), -1)
    s["target"] = torch.softmax(logits, -1)
    noise = -torch.log(torch.rand(S, N, V, generator=g, device=DEV).clamp_(min=1e-30))
    s["tokens"] = (rows / noise).argmax(-1).int()
    s["u"] = torch.rand(S, N, generator=g, device=DEV)
    return s


# ---- the framework's own calls ---------------------------------------------------------------------------------------


def _own(s):
    import iree_turbine_amd  # noqa: F401

    ops, case = torch.ops.mi355, s["case"]
    op = case["op"]
    if op == "layout":
        return (s["table"], *ops.paged_batch_layout(s["table"], s["ctx"], s["new"], s["free"], s["page"], s["rows"]))
    if op == "rope_append":
        q = ops.rope_kv_append(s["q"], s["k"], s["v"], s["pos"], s["freq"], s["kc"], s["vc"], s["slots"], case["interleaved"], s["scale"])
        return q, s["kc"], s["vc"]
    if op == "rope_train":
        y = ops.rope(s["x"], s["pos"], s["freq"], case["interleaved"], False, s["scale"])
        return y.detach(), torch.autograd.grad(y, s["x"], s["dy"])[0]
    if op == "prompts":
        return ops.flash_attn_varlen_fwd(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], case["causal"], 0.0)
    if op == "tree":
        return ops.paged_tree_attn(s["q"], s["kc"], s["vc"], s["table"], s["lens"], s["parents"], 0.0, 0)
    return ops.verify_draft(s["target"], s["draft"], s["tokens"], s["parents"], s["u"])


# ---- the plain forms -------------------------------------------------------------------------------------------------


def _plain_layout(s):
    """Pages for the new tokens from the front of the free list, and every new token's sequence, position and slot."""
    table, free, page, rows = s["table"], s["free"], s["page"], s["rows"]
    S, W = table.shape
    ctx, new = s["ctx"].long(), s["new"].long()
    have, want = -(-ctx // page), -(-(ctx + new) // page)
    need = want.clamp(max=W) - have.clamp(max=W)
    first = torch.cumsum(need, 0) - need
    col = torch.arange(W, device=DEV)[None]
    which = first[:, None] + col - have[:, None]
    ids = torch.where(which < free.numel(), free[which.clamp(0, free.numel() - 1)], -1)
    table.copy_(torch.where((col >= have[:, None]) & (col < want[:, None]), ids, table))
    ends = torch.cumsum(new, 0)
    tok = torch.arange(rows, device=DEV)
    seq = torch.searchsorted(ends, tok, right=True)
    live = seq < S
    at = seq.clamp(max=S - 1)
    pos = ctx[at] + tok - (ends - new)[at]
    entry = torch.where(pos // page < W, table[at, (pos // page).clamp(max=W - 1)], -1).long()
    slot = torch.where(live & (entry >= 0), entry * page + pos % page, -1)
    cu = torch.cat([torch.zeros_like(ends[:1]), ends]).clamp(max=rows)
    return (table, (ctx + new).int(), cu.int(), torch.where(live, pos, 0).int(), torch.where(live, seq, -1).int(), slot, need.sum()[None].int())


def _turn(x, pos, freq, interleaved, scale, sign=1.0):
    """The pairs of the first 2 len(freq) elements turned by pos * freq, angles in 64 bits, products in 32."""
    half = freq.numel()
    angle = pos.double()[:, None, None] * freq
    c, n = (torch.cos(angle) * scale).float(), (torch.sin(angle) * (scale * sign)).float()
    f = x.float()
    head, rest = f[..., : 2 * half], f[..., 2 * half:]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        out = torch.stack([a * c - b * n, a * n + b * c], -1).flatten(-2)
    else:
        a, b = head[..., :half], head[..., half:]
        out = torch.cat([a * c - b * n, a * n + b * c], -1)
    return torch.cat([out, rest], -1).to(x.dtype)


def _plain_rope_append(s):
    case = s["case"]
    q, k = (_turn(s[n], s["pos"], s["freq"], case["interleaved"], s["scale"]) for n in "qk")
    kc, vc = s["kc"].view(-1, case["hkv"], 128), s["vc"].view(-1, case["hkv"], 128)
    keep = (s["slots"] >= 0)[:, None, None]  # a padded token writes back what its (clamped) slot already holds
    at = torch.where(s["slots"] >= 0, s["slots"], s["slots"][0])
    kc[at] = torch.where(keep, k, k[:1])
    vc[at] = torch.where(keep, s["v"], s["v"][:1])
    return q, s["kc"], s["vc"]


def _plain_rope_train(s):
    case, x = s["case"], s["x"].detach()
    return (_turn(x, s["pos"], s["freq"], case["interleaved"], s["scale"]), _turn(s["dy"], s["pos"], s["freq"], case["interleaved"], s["scale"], -1.0))


def _softmax_rows(scores, hidden):
    """exp(x - max) / sum over the last axis without the hidden places; rows without any place give zeros."""
    scores = scores.masked_fill_(hidden, -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores = scores.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = scores.sum(-1, keepdim=True)
    return scores.div_(torch.where(total > 0, total, 1.0))


def _plain_prompts(s):
    """Sequences laid out on a common grid of rows, masked products and softmax in 32 bits, rows gathered back."""
    case, q, k, v = s["case"], s["q"], s["k"], s["v"]
    hq, hkv = case["hq"], case["hkv"]
    lq, lk = s["cu_q"].diff().long(), s["cu_k"].diff().long()
    i, j = torch.arange(s["max_q"], device=DEV), torch.arange(s["max_k"], device=DEV)
    at_q = (s["cu_q"][:-1, None] + i).clamp(max=q.shape[0] - 1)
    at_k = (s["cu_k"][:-1, None] + j).clamp(max=k.shape[0] - 1)
    S = at_q.shape[0]
    Q = q[at_q].float().view(S, -1, hkv, hq // hkv, 128).permute(0, 2, 3, 1, 4).reshape(S * hkv, -1, 128)
    K, V = (x[at_k].float().transpose(1, 2).reshape(S * hkv, -1, 128) for x in (k, v))
    hidden = (j >= lk[:, None])[:, None, None, None, :]
    if case["causal"]:
        hidden = hidden | (j[None, None] > i[None, :, None] + (lk - lq)[:, None, None])[:, None, None]
    scores = torch.matmul(Q, K.transpose(1, 2).contiguous()).mul_(128 ** -0.5).view(S, hkv, hq // hkv, -1, j.numel())
    P = _softmax_rows(scores, hidden)
    O = torch.matmul(P.view(S * hkv, -1, j.numel()), V).view(S, hq, -1, 128).transpose(1, 2)
    row = torch.arange(q.shape[0], device=DEV)
    seq = torch.searchsorted(s["cu_q"][1:].contiguous(), row, right=True).clamp(max=S - 1)
    live = (row < s["cu_q"][-1])[:, None, None]
    return torch.where(live, O[seq, (row - s["cu_q"][seq]).clamp(max=s["max_q"] - 1)], 0.0).to(q.dtype)


def _reach(parents):
    """reach[s, i, j]: node j is node i or one of its ancestors."""
    N = parents.shape[1]
    step = torch.arange(N, device=DEV) == parents[..., None]
    reach = (step | torch.eye(N, dtype=torch.bool, device=DEV)).float()
    for _ in range(max(0, N - 1).bit_length()):
        reach = (torch.matmul(reach, reach.contiguous()) > 0).float()
    return reach > 0


def _plain_tree(s):
    case, q = s["case"], s["q"]
    S, N, hq, D = q.shape
    hkv, page = case["hkv"], case["page"]
    L = s["table"].shape[1] * page
    rows = s["table"].clamp(min=0).long()
    K, V = (c[rows].view(S, L, hkv, D).float().transpose(1, 2).reshape(S * hkv, L, D) for c in (s["kc"], s["vc"]))
    Q = q.float().view(S, N, hkv, hq // hkv, D).permute(0, 2, 1, 3, 4).reshape(S * hkv, -1, D)
    at = torch.arange(L, device=DEV)[None] - (s["lens"].long() - N)[:, None]  # negative in front of the drafts, then the node
    seen = torch.gather(_reach(s["parents"]), 2, at.clamp(0, N - 1)[:, None].expand(S, N, L)) & (at < N)[:, None]
    hidden = ~(seen | (at < 0)[:, None])
    scores = torch.matmul(Q, K.transpose(1, 2).contiguous()).mul_(D ** -0.5).view(S, hkv, N, hq // hkv, L)
    P = _softmax_rows(scores, hidden[:, None, :, None, :])
    V = V * (s["table"] >= 0).repeat_interleave(page, 1).repeat_interleave(hkv, 0)[..., None]
    O = torch.matmul(P.view(S * hkv, -1, L), V).view(S, hkv, N, hq // hkv, D)
    return O.transpose(1, 2).reshape(S, N, hq, D).to(q.dtype)


def _plain_verify(s):
    """The nodes in order: a child of the present node is accepted where u q < r, and otherwise leaves max(r - q, 0).
    r is the target's row with its mass beside it, in 64 bits: a comparison must not depend on how a sum was rounded."""
    p, q, tokens, parents, u = s["target"], s["draft"], s["tokens"].long(), s["parents"].long(), s["u"].double()
    S, N, V = p.shape
    row = torch.arange(S, device=DEV)
    cur, count = torch.zeros_like(row), torch.zeros_like(row)
    r, mass = p[:, 0].double(), torch.ones(S, dtype=torch.float64, device=DEV)
    path = torch.full((S, N + 1), -1, dtype=torch.long, device=DEV)
    for i in range(1, N):
        t = tokens[:, i]
        child = parents[:, i] == cur
        qi = q[row, cur].double() if q is not None else (torch.arange(V, device=DEV) == t[:, None]).double()
        qi = qi * mass[:, None]
        take = child & (u[:, i] * qi[row, t] < r[row, t])
        drop = child & ~take
        left = (r - qi).clamp_(min=0)
        total = left.sum(-1)
        drop = drop & (total > 0)
        r = torch.where(take[:, None], p[:, i].double(), torch.where(drop[:, None], left, r))
        mass = torch.where(take, 1.0, torch.where(drop, total, mass))
        path[row, torch.where(take, count, N)] = i
        cur, count = torch.where(take, i, cur), count + take
    path[:, N] = -1
    sums = torch.cumsum(r, -1)
    hit = (sums > (u[:, 0] * sums[:, -1])[:, None]) & (r > 0)
    return path[:, :N].int(), count.int(), hit.int().argmax(-1).int()


PLAIN = {"layout": _plain_layout, "rope_append": _plain_rope_append, "rope_train": _plain_rope_train, "prompts": _plain_prompts, "tree": _plain_tree, "verify": _plain_verify}


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return PLAIN[state["case"]["op"]](state)


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------


def _exact_layout(s):
    table, free, page, rows = s["table"].cpu().numpy().copy(), s["free"].cpu().numpy(), s["page"], s["rows"]
    ctx, new = s["ctx"].cpu().tolist(), s["new"].cpu().tolist()
    W = table.shape[1]
    taken, cu, pos, seq, slot = 0, [0], [], [], []
    for i, (c, n) in enumerate(zip(ctx, new)):
        for col in range(min(W, (c + page - 1) // page), min(W, (c + n + page - 1) // page)):
            table[i, col] = free[taken] if taken < len(free) else -1
            taken += 1
        for t in range(c, c + n):
            pos.append(t)
            seq.append(i)
            e = int(table[i, t // page]) if t // page < W else -1
            slot.append(e * page + t % page if e >= 0 else -1)
        cu.append(min(rows, cu[-1] + n))
    fill = lambda v, x, dt: np.array((v + [x] * rows)[:rows], dtype=dt)  # noqa: E731
    return (table, np.array([c + n for c, n in zip(ctx, new)], np.int32), np.array(cu, np.int32), fill(pos, 0, np.int32), fill(seq, -1, np.int32), fill(slot, -1, np.int64), np.array([taken], np.int32))


def _exact_turn(x, s, sign):
    """Each pair as a complex number, times scale * exp(i * sign * pos * freq)."""
    case = s["case"]
    half = s["freq"].numel()
    x = x.detach().double()
    pairs = x[..., : 2 * half].unflatten(-1, (half, 2) if case["interleaved"] else (2, half))
    if not case["interleaved"]:
        pairs = pairs.transpose(-1, -2)
    by = torch.polar(torch.full_like(s["freq"], s["scale"]).expand(x.shape[0], half).contiguous(), sign * torch.outer(s["pos"].double(), s["freq"]))
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * by[:, None])
    z = z.flatten(-2) if case["interleaved"] else z.transpose(-1, -2).flatten(-2)
    return torch.cat([z, x[..., 2 * half:]], -1)


def _exact_attention(q, k, v, visible):
    """q [n, hq, d] over k, v [m, hkv, d], one head at a time; visible [n, m]."""
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    group = q.shape[1] // k.shape[1]
    for h in range(q.shape[1]):
        a = torch.mm(q[:, h].double(), k[:, h // group].double().t().contiguous()) / math.sqrt(q.shape[2])
        a = torch.where(visible, a, -math.inf)
        w = torch.nan_to_num(torch.softmax(a, -1))
        out[:, h] = torch.mm(w, v[:, h // group].double())
    return out


def _exact_prompts(s):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    cq, ck = s["cu_q"].tolist(), s["cu_k"].tolist()
    for a, b, c, d in zip(cq, cq[1:], ck, ck[1:]):
        if b > a and d > c:
            visible = torch.ones(b - a, d - c, dtype=torch.bool, device=DEV)
            if s["case"]["causal"]:
                visible = visible.tril(d - c - (b - a))
            out[a:b] = _exact_attention(s["q"][a:b], s["k"][c:d], s["v"][c:d], visible)
    return out


def _exact_tree(s):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    N, page = s["q"].shape[1], s["case"]["page"]
    for i, L in enumerate(s["lens"].tolist()):
        pages = s["table"][i, : -(-L // page)].long()
        k, v = (c[pages].flatten(0, 1)[:L] for c in (s["kc"], s["vc"]))
        par = s["parents"][i].tolist()
        visible = torch.zeros(N, L, dtype=torch.bool)
        for n in range(N):
            visible[n, : L - N] = True
            a = n
            while a >= 0:
                visible[n, L - N + a] = True
                a = par[a]
        out[i] = _exact_attention(s["q"][i], k, v, visible.to(DEV))
    return out


def _exact_verify(s):
    tokens, parents, u = s["tokens"].cpu().tolist(), s["parents"].cpu().tolist(), s["u"].cpu().double().numpy()
    S, N = len(tokens), len(tokens[0])
    path, count, last = np.full((S, N), -1, np.int32), np.zeros(S, np.int32), np.zeros(S, np.int32)
    for b in range(S):
        cur, r, mass = 0, s["target"][b, 0].double().cpu().numpy(), 1.0
        for i in range(1, N):
            if parents[b][i] != cur:
                continue
            t = tokens[b][i]
            if s["draft"] is None:
                q = np.zeros_like(r)
                q[t] = 1.0
            else:
                q = s["draft"][b, cur].double().cpu().numpy()
            if u[b, i] * (q[t] * mass) < r[t]:
                cur, r, mass = i, s["target"][b, i].double().cpu().numpy(), 1.0
                path[b, count[b]] = i
                count[b] += 1
            else:
                left = np.maximum(r - q * mass, 0.0)
                if left.sum() > 0:
                    r, mass = left, left.sum()
        sums = np.cumsum(r)
        last[b] = int(np.nonzero((sums > u[b, 0] * sums[-1]) & (r > 0))[0][0])
    return path, count, last


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "rope_append":
            kc, vc = s["kc"].double(), s["vc"].double()
            rows = (s["slots"] >= 0).nonzero()[:, 0]
            kc.view(-1, case["hkv"], 128)[s["slots"][rows]] = _exact_turn(s["k"], s, 1.0)[rows]
            vc.view(-1, case["hkv"], 128)[s["slots"][rows]] = s["v"].double()[rows]
            return _exact_turn(s["q"], s, 1.0), kc, vc
        if case["op"] == "rope_train":
            return _exact_turn(s["x"], s, 1.0), _exact_turn(s["dy"], s, -1.0)
        return {"layout": _exact_layout, "prompts": _exact_prompts, "tree": _exact_tree, "verify": _exact_verify}[case["op"]](s)
