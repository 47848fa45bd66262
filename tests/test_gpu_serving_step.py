"""The serving operators together, as a server would run them: a packed prompt step, then rounds of drafting and verification over
the paged cache, against the same steps in 64 bits without pages."""

import pytest
import torch

import iree_turbine_amd as ita
from conftest import announce

pytestmark = pytest.mark.gpu

HQ, HKV, PAGE, V = 8, 2, 16, 600


class Cache:
    """What the server keeps on the device: pages, their table, the free list, lengths."""

    def __init__(self, dev, S, pages, width, dtype):
        self.dev, self.S = dev, S
        self.k, self.v = (torch.full((pages, PAGE, HKV, 128), float("nan"), dtype=dtype, device=dev) for _ in range(2))
        self.table = torch.full((S, width), -1, dtype=torch.int32, device=dev)
        self.free = torch.randperm(pages, device=dev).int()
        self.len = torch.zeros(S, dtype=torch.int32, device=dev)

    def step(self, new_lens, rows):
        """Layout of a step; the pages it takes leave the free list."""
        out = torch.ops.mi355.paged_batch_layout(self.table, self.len, new_lens, self.free, PAGE, rows)
        taken = int(out[5])
        assert taken <= self.free.numel()
        self.free = self.free[taken:]
        return out


def _tokens_of(cache, s, n):
    rows = cache.table[s, : -(-n // PAGE)].long()
    return [c[rows].flatten(0, 1)[:n].cpu() for c in (cache.k, cache.v)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prompt_then_draft_rounds(dev, dtype):
    from oracle import serving

    announce(f"serving step {dtype}")
    torch.manual_seed(11)
    lens = [37, 1, 100, 0, 16]
    S, T, pad = len(lens), sum(lens), 6
    freq, scale = ita.rope_inv_freq(128, scaling="yarn", factor=4.0)
    fd = freq.to(dev)
    cache = Cache(dev, S, 64, 20, dtype)

    # -- the prompts: layout, rotation and append, packed attention
    new = torch.tensor(lens, dtype=torch.int32, device=dev)
    seq_lens, cu, pos, seq_ids, slots, _ = cache.step(new, T + pad)
    qkv = torch.randn(T + pad, HQ + 2 * HKV, 128).to(dtype)
    q, k, v = qkv.to(dev).split([HQ, HKV, HKV], 1)
    q = torch.ops.mi355.rope_kv_append(q, k, v, pos, fd, cache.k, cache.v, slots, False, scale)
    kr = torch.ops.mi355.rope(k, pos, fd, False, False, scale)
    out = torch.ops.mi355.flash_attn_varlen_fwd(q, kr, v, cu, cu, True, 0.0)
    cache.len = seq_lens
    assert seq_lens.tolist() == lens and slots[T:].tolist() == [-1] * pad
    want_k, bound_k = serving.rope_ref(qkv[:, HQ:HQ + HKV], pos.cpu(), freq, False, scale=scale)
    for s in range(S):
        a, b = int(cu[s]), int(cu[s + 1])
        ks, vs = _tokens_of(cache, s, lens[s])
        assert bool(((ks.double() - want_k[a:b]).abs() <= bound_k[a:b]).all())
        assert torch.equal(vs, qkv[a:b, HQ + HKV:]) and torch.equal(ks, kr[a:b].cpu())
    want, bound = serving.varlen_ref(q.cpu(), kr.cpu(), v.cpu(), cu.cpu(), cu.cpu(), True)
    assert bool(((out.double().cpu() - want).abs() <= bound).all())
    # the paged prefill of one sequence gives the same numbers
    one = torch.ops.mi355.paged_prefill_attn(q[38:138][None].contiguous(), cache.k, cache.v, cache.table[2:3].contiguous(), seq_lens[2:3].contiguous(), 0.0)
    torch.testing.assert_close(one[0], out[38:138], rtol=2e-2, atol=2e-2)

    # -- rounds of drafts: a tree of six nodes per sequence, attention, verification, the accepted path kept
    N = 6
    parents = torch.tensor([[-1, 0, 0, 1, 1, 2]] * S, dtype=torch.int32, device=dev)
    depth = torch.tensor([0, 1, 1, 2, 2, 2], dtype=torch.int32, device=dev)
    for rnd in range(3):
        before = cache.len.clone()
        seq_lens, cu, pos, _, slots, _ = cache.step(torch.full((S,), N, dtype=torch.int32, device=dev), S * N)
        qkv = torch.randn(S * N, HQ + 2 * HKV, 128).to(dtype).to(dev)
        at = (before[:, None] + depth).flatten()  # a node's position is its depth in the tree, its slot its number
        q = torch.ops.mi355.rope_kv_append(*qkv.split([HQ, HKV, HKV], 1), at, fd, cache.k, cache.v, slots, False, scale)
        out = torch.ops.mi355.paged_tree_attn(q.view(S, N, HQ, 128), cache.k, cache.v, cache.table, seq_lens, parents, 0.0, 0)
        args = [t.cpu() for t in (q.view(S, N, HQ, 128), cache.k, cache.v, cache.table, seq_lens, parents)]
        args[1:3] = [torch.nan_to_num(c, 0.0) for c in args[1:3]]
        want, bound = serving.tree_ref(*args)
        assert torch.isfinite(out).all() and bool(((out.double().cpu() - want).abs() <= bound).all())

        logits = 2 * torch.randn(S, N, V)
        target, draft = torch.softmax(logits, -1), torch.softmax(logits + torch.randn(S, N, V), -1)
        tokens = torch.stack([torch.multinomial(draft[:, max(0, int(p))], 1)[:, 0] for p in parents[0]], 1).int()
        u = torch.rand(S, N)
        path, count, last = torch.ops.mi355.verify_draft(target.to(dev), draft.to(dev), tokens.to(dev), parents, u.to(dev))
        for g, w in zip((path, count, last), serving.verify_ref(target, draft, tokens, parents.cpu(), u)):
            assert torch.equal(g.cpu(), w)

        # keep node 0 and the accepted path: their rows move to the places behind the old end
        flat_k, flat_v = cache.k.view(-1, HKV, 128), cache.v.view(-1, HKV, 128)
        for s in range(S):
            kept = [0] + [n for n in path[s].tolist() if n >= 0]
            src = slots.view(S, N)[s, kept]
            dst = slots.view(S, N)[s, : len(kept)]
            flat_k[dst], flat_v[dst] = flat_k[src], flat_v[src]
        cache.len = before + 1 + count
        # pages behind the new end go back to the free list
        for s in range(S):
            first, end = -(-int(cache.len[s]) // PAGE), -(-int(seq_lens[s]) // PAGE)
            cache.free = torch.cat([cache.table[s, first:end], cache.free])
            cache.table[s, first:end] = -1
    held = cache.table[cache.table >= 0].tolist()
    assert sorted(held + cache.free.tolist()) == list(range(64))


def test_training_step_with_packed_rotation_captured(dev):
    """The rotation's gradient inside a captured training step, replayed with new data, against the eager one."""
    announce("captured rotation gradient")
    f = ita.rope_inv_freq(64, device=dev)[0]
    pos = torch.arange(33, dtype=torch.int32, device=dev) * 50
    w = torch.randn(64, 4 * 96, device=dev, requires_grad=True)
    x = torch.randn(33, 64, device=dev)

    def step():
        y = torch.ops.mi355.rope((x @ w).view(33, 4, 96), pos, f, True, False, 1.0)
        return torch.autograd.grad((y * y * 0.5 + y).sum(), w)[0]

    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream(dev).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        g = step()
    for _ in range(3):
        x.copy_(torch.randn(33, 64))
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        # The same kernels on the same data; the library's products may differ in the order of their sums.  An entry of the
        # gradient is 33 products of x with the turned (y + 1), y itself the turned sum of 64 products: each of them is off
        # by 2^-24 per product and turn (a turn adds two products) against the sum of magnitudes.
        with torch.no_grad():
            mag = (x.abs() @ w.abs()).view(33, 4, 96)
            for _ in range(2):  # a turn's magnitude: the pair's sum
                mag = torch.cat([mag[..., :64].unflatten(-1, (32, 2)).sum(-1, keepdim=True).expand(-1, -1, -1, 2).flatten(-2), mag[..., 64:]], -1) + 1
            bound = (33 + 64 + 2 * 4) * 2.0**-24 * (x.abs().t() @ mag.view(33, -1))
            assert bool(((g - eager).abs() <= 2 * bound).all())
    h = (x @ w).detach().view(33, 4, 96)
    y = torch.ops.mi355.rope(h, pos, f, True, False, 1.0)
    dx = torch.ops.mi355.rope(y + 1, pos, f, True, True, 1.0).view(33, -1)
    torch.testing.assert_close(eager, x.t() @ dx, rtol=1e-4, atol=1e-3)
