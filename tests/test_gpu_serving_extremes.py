"""GPU parity: the serving operators at the ends of their ranges -- the widest trees and groups, the most sequences, rows laid
out head by head, one-element pairs over many heads."""

import random

import pytest
import torch

import iree_turbine_amd as ita
from conftest import announce

pytestmark = pytest.mark.gpu
OPS = torch.ops.mi355


def _inside(got, want, bound):
    off = (got.double().cpu() - want).abs()
    assert torch.isfinite(got).all()
    worst = (off - bound).max().item()
    assert worst <= 0, f"off by {off.max().item():.3g}, {worst:.3g} more than the bound allows"


def _cu(lens):
    return torch.cumsum(torch.tensor([0] + list(lens)), 0).int()


@pytest.mark.parametrize("splits", [1, 0, 1024])
@pytest.mark.parametrize("N,hq", [(64, 128), (1, 128), (63, 127)])
def test_widest_trees_and_groups(dev, N, hq, splits):
    """Up to 64 nodes and 128 query heads on one K/V head: 8192 rows that share one pass."""
    from oracle import serving

    announce(f"tree N={N} hq={hq} hkv=1 splits={splits}")
    lens = [N + 300, N - 1]
    g = torch.Generator().manual_seed(N)
    kc, vc = (torch.randn(30, 16, 1, 128, generator=g).bfloat16() for _ in range(2))
    table = torch.randperm(30, generator=g).int()[: 2 * 15].view(2, 15)
    table = torch.cat([table, torch.full((2, 9), -1, dtype=torch.int32)], 1)
    lens = [min(n, 15 * 16) for n in lens]
    q = torch.randn(2, N, hq, 128, generator=g).bfloat16()
    rng = random.Random(N)
    par = torch.tensor([[-1] + [rng.randrange(max(0, i - 5), i) for i in range(1, N)] for _ in range(2)], dtype=torch.int32)
    sl = torch.tensor(lens, dtype=torch.int32)
    got = OPS.paged_tree_attn(*(t.to(dev) for t in (q, kc, vc, table, sl, par)), 0.0, splits)
    heads = [0, 1, hq // 2, hq - 1]  # the oracle takes a head at a time
    _inside(got[:, :, heads], *serving.tree_ref(q[:, :, heads], kc, vc, table, sl, par))


@pytest.mark.parametrize("causal", [True, False])
def test_packed_rows_laid_out_head_by_head(dev, causal):
    """[heads, tokens, 128] tensors seen as [tokens, heads, 128]: rows 128 elements apart, heads far; and the result's view too."""
    from iree_turbine_amd import launch
    from oracle import serving

    announce(f"varlen head by head causal={causal}")
    lens = [70, 1, 200, 33]
    T, cu = sum(lens), _cu(lens)
    q, k, v = (torch.randn(h, T, 128).half() for h in (8, 2, 2))
    views = [t.transpose(0, 1) for t in (q, k, v)]
    on = [t.to(dev).transpose(0, 1) for t in (q, k, v)]
    assert on[0].stride() == (128, T * 128, 1)
    want, bound = serving.varlen_ref(*views, cu, cu, causal)
    got = OPS.flash_attn_varlen_fwd(*on, cu.to(dev), cu.to(dev), causal, 0.0)
    _inside(got, want, bound)
    o = torch.empty(8, T, 128, dtype=torch.float16, device=dev).transpose(0, 1)
    launch.flash_attn_varlen_fwd_out(*on, cu.to(dev), cu.to(dev), o, causal, 0.0)
    assert torch.equal(o, got)


def test_packed_attention_of_very_many_sequences(dev):
    """65535 sequences, most of them empty; single tokens among them, some without keys."""
    from oracle import serving

    announce("varlen 65535 sequences")
    S = 65535
    rng = random.Random(4)
    lq, lk = [0] * S, [0] * S
    for s in sorted(rng.sample(range(S), 60) + [0, S - 1]):
        lq[s], lk[s] = rng.choice([1, 1, 2, 70]), rng.choice([0, 1, 5, 130])
    lk[100] += 40  # keys that no query has
    cq, ck = _cu(lq), _cu(lk)
    q, k, v = (torch.randn(n, h, 128).bfloat16() for n, h in ((sum(lq), 4), (sum(lk), 2), (sum(lk), 2)))
    for causal in (True, False):
        got = OPS.flash_attn_varlen_fwd(*(t.to(dev) for t in (q, k, v, cq, ck)), causal, 0.0)
        _inside(got, *serving.varlen_ref(q, k, v, cq, ck, causal))


def test_layout_of_the_most_sequences(dev):
    from oracle import serving

    announce("layout 65535 sequences")
    S, W, page = 65535, 3, 16
    g = torch.Generator().manual_seed(2)
    ctx, new = torch.randint(0, 30, (S,), generator=g).int(), torch.randint(0, 3, (S,), generator=g).int()
    new[7], new[S - 1] = 5000, 9  # far behind its table; the last
    table, free = torch.randint(0, 1 << 20, (S, W), generator=g).int(), torch.randperm(60000, generator=g).int()
    T = int(new.sum()) - 4  # the last tokens find no row
    want = serving.batch_layout_ref(table, ctx, new, free, page, T)
    on = table.to(dev)
    got = OPS.paged_batch_layout(on, ctx.to(dev), new.to(dev), free.to(dev), page, T)
    assert torch.equal(on.cpu(), want[0])
    for a, b in zip(got, want[1:]):
        assert a.tolist() == b


@pytest.mark.parametrize("T,H,D,R,inter", [(3, 65535, 2, 2, False), (2, 3001, 64, 6, True), (1, 1, 65536, 1024, False), (2100, 1, 4, 2, True)])
def test_rope_of_odd_proportions(dev, T, H, D, R, inter):
    from oracle import serving

    announce(f"rope T={T} H={H} D={D} R={R}")
    x, pos, (f, _) = torch.randn(T, H, D).half(), torch.randint(-5, 1 << 20, (T,), dtype=torch.int32), ita.rope_inv_freq(R)
    _inside(OPS.rope(x.to(dev), pos.to(dev), f.to(dev), inter, False, 1.0), *serving.rope_ref(x, pos, f, inter))


def test_append_with_more_key_heads_than_query_heads(dev):
    from oracle import serving

    announce("append 1 query head, 65 key heads")
    T, hkv = 2050, 65
    q, k, v = (torch.randn(T, h, 128).bfloat16() for h in (1, hkv, hkv))
    kc, vc = (torch.zeros(10, 256, hkv, 128, dtype=torch.bfloat16, device=dev) for _ in range(2))
    pos, slots, (f, _) = torch.arange(T, dtype=torch.int32), torch.randperm(2560)[:T], ita.rope_inv_freq(32)
    got = OPS.rope_kv_append(q.to(dev), k.to(dev), v.to(dev), pos.to(dev), f.to(dev), kc, vc, slots.to(dev), False, 1.0)
    _inside(got, *serving.rope_ref(q, pos, f, False))
    _inside(kc.view(-1, hkv, 128)[slots.to(dev)], *serving.rope_ref(k, pos, f, False))
    assert torch.equal(vc.view(-1, hkv, 128)[slots.to(dev)].cpu(), v)
    rest = torch.ones(2560, dtype=torch.bool)
    rest[slots] = False
    assert not kc.view(-1, hkv, 128).cpu()[rest].any() and not vc.view(-1, hkv, 128).cpu()[rest].any()


def test_verify_largest_vocabulary_and_batch(dev):
    """2^24 entries (64 blocks a piece); 65535 sequences of one and two nodes."""
    from oracle import serving

    announce("verify 2^24 entries")
    V = 1 << 24
    g = torch.Generator().manual_seed(8)
    target = torch.rand(1, 3, V, generator=g)
    target /= target.sum(-1, keepdim=True)
    draft = target.flip(-1).contiguous()
    tokens, par = torch.tensor([[0, 5, V - 1]], dtype=torch.int32), torch.tensor([[-1, 0, 0]], dtype=torch.int32)
    for u in ([0.3, 0.99999, 0.99999], [1 - 2**-24, 0.99999, 0.0], [0.0, 0.0, 0.5]):
        ins = (target, draft, tokens, par, torch.tensor([u]))
        for a, b in zip(OPS.verify_draft(*(t.to(dev) for t in ins)), serving.verify_ref(*ins)):
            assert torch.equal(a.cpu(), b)
    announce("verify 65535 sequences")
    S, V = 65535, 5
    target, draft = (torch.softmax(torch.randn(S, 2, V, generator=g), -1) for _ in range(2))
    tokens, par = torch.randint(0, V, (S, 2), generator=g).int(), torch.tensor([[-1, 0]], dtype=torch.int32).repeat(S, 1)
    ins = (target, draft, tokens, par, torch.rand(S, 2, generator=g))
    got = OPS.verify_draft(*(t.to(dev) for t in ins))
    some = torch.arange(0, S, 97)
    for a, b in zip(got, serving.verify_ref(*(t[some] for t in ins))):
        assert torch.equal(a.cpu()[some], b)
