"""GPU parity: verification of drafted tokens; whole numbers, equal to the 64-bit oracle's."""

import random

import pytest
import torch

import iree_turbine_amd  # noqa: F401  (registers torch.ops.mi355)
from conftest import announce

pytestmark = pytest.mark.gpu


def _parents(seed, S, N, branch):
    rng = random.Random(seed)
    return torch.tensor([[-1] + [rng.randrange(max(0, i - branch), i) if branch > 1 else i - 1 for i in range(1, N)] for _ in range(S)], dtype=torch.int32)


def _inputs(seed, S, N, V, branch, sampled, near=0.7):
    g = torch.Generator().manual_seed(seed)
    logits = 2 * torch.randn(S, N, V, generator=g)
    target = torch.softmax(logits, -1)
    parents = _parents(seed, S, N, branch)
    up = parents.clamp(min=0).long()[..., None].expand(S, N, V)
    draft = torch.softmax(logits + near * torch.randn(S, N, V, generator=g), -1)
    tokens = torch.multinomial(torch.gather(draft, 1, up).reshape(S * N, V), 1, generator=g).view(S, N).int()
    return target, draft if sampled else None, tokens, parents, torch.rand(S, N, generator=g)


def _check(dev, ins):
    from oracle import serving

    want = serving.verify_ref(*ins)
    got = torch.ops.mi355.verify_draft(*(t.to(dev) if t is not None else None for t in ins))
    for name, a, b in zip(("path", "num_accepted", "next_token"), got, want):
        assert torch.equal(a.cpu(), b), name
    return got


@pytest.mark.parametrize("sampled", [True, False])
@pytest.mark.parametrize("S,N,V,branch", [(1, 1, 50, 1), (1, 1, 1, 1), (3, 2, 7, 1), (4, 5, 1000, 1), (6, 9, 4096, 3), (5, 64, 300, 6), (3, 12, 4097, 4), (2, 6, 20001, 5), (70, 4, 33, 2)])
def test_verify(dev, S, N, V, branch, sampled):
    announce(f"verify S={S} N={N} V={V} branch={branch} sampled={sampled}")
    for seed in range(4):
        _check(dev, _inputs(seed, S, N, V, branch, sampled))


@pytest.mark.parametrize("sampled", [True, False])
def test_verify_siblings_rejected_in_a_row(dev, sampled):
    """A far draft: every child of the root is rejected, one after the other, over many chunks of the vocabulary."""
    announce(f"verify many rejections sampled={sampled}")
    target, draft, tokens, _, u = _inputs(1, 4, 12, 9000, 1, sampled, near=6.0)
    star = torch.tensor([[-1] + [0] * 11] * 4, dtype=torch.int32)
    u[:, 1:] = 0.9999
    tokens[1, 3:] = tokens[1, 2]  # the same token again and again
    got = _check(dev, (target, draft, tokens, star, u))
    assert int(got[1].sum()) <= 4
    u[2, 0], u[3, 0] = 0.0, 1 - 2**-24
    _check(dev, (target, draft, tokens, star, u))


def test_verify_borders(dev):
    """Drafts equal to the target are always accepted; zero probabilities never; tokens and parents that are none take no
    part; a row without mass gives no token; random numbers outside their range stay in bounds."""
    announce("verify borders")
    target, draft, tokens, parents, u = _inputs(2, 6, 5, 500, 1, True)
    got = _check(dev, (target, target.clone(), tokens, parents, u))
    assert got[1].tolist() == [4] * 6 and got[0][:, :4].tolist() == [[1, 2, 3, 4]] * 6 and got[0][:, 4].tolist() == [-1] * 6
    none = target.clone()
    none.scatter_(2, torch.gather(tokens, 1, torch.tensor([1, 2, 3, 4, 0]).expand(6, 5)).long()[..., None], 0.0)
    got = _check(dev, (none, draft, tokens, parents, u.clamp(min=1e-3)))
    assert got[1].tolist() == [0] * 6
    odd_tokens, odd_parents = tokens.clone(), parents.clone()
    odd_tokens[0, 1], odd_tokens[1, 2], odd_parents[2, 3], odd_parents[3, 1] = -1, 500, 3, 9
    got = _check(dev, (target, target.clone(), odd_tokens, odd_parents, u))
    assert got[1].tolist() == [0, 1, 2, 0, 4, 4]
    empty = target.clone()
    empty[4] = 0
    got = _check(dev, (empty, draft, tokens, parents, u))
    assert int(got[2][4]) == -1
    wild = u.clone()
    wild[:, 0] = torch.tensor([-1.0, 1.0, 5.0, float("nan"), float("inf"), 0.0])
    got = torch.ops.mi355.verify_draft(*(t.to(dev) for t in (target, draft, tokens, parents, wild)))
    assert all(0 <= t < 500 for t in got[2].tolist())


def test_verify_one_entry_holds_all(dev):
    """Greedy targets: rows with a single one, in the first, a middle and the last chunk."""
    announce("verify greedy")
    S, N, V = 3, 3, 10000
    target = torch.zeros(S, N, V)
    best = torch.tensor([[5, 0, 9999], [4095, 4096, 7], [8191, 8192, 3]])
    target.scatter_(2, best[..., None], 1.0)
    tokens = torch.tensor([[0, 5, 0], [0, 4095, 4096], [0, 8191, 1]], dtype=torch.int32)
    parents = torch.tensor([[-1, 0, 1]] * 3, dtype=torch.int32)
    got = _check(dev, (target, None, tokens, parents, torch.full((S, N), 0.5)))
    assert got[1].tolist() == [2, 2, 1] and got[2].tolist() == [9999, 7, 8192]


def test_verify_keeps_the_target_distribution(dev):
    """First tokens of many sequences follow the target whatever the draft: within 5 standard deviations."""
    announce("verify distribution")
    S, V = 30000, 6
    torch.manual_seed(5)
    p, q = (torch.softmax(torch.randn(V), 0) for _ in range(2))
    for parents in ([-1, 0], [-1, 0, 0, 0]):
        N = len(parents)
        tokens = torch.multinomial(q, S * N, replacement=True).view(S, N).int().to(dev)
        path, count, last = torch.ops.mi355.verify_draft(p.expand(S, N, V).contiguous().to(dev), q.expand(S, N, V).contiguous().to(dev), tokens,
                                                         torch.tensor(parents, dtype=torch.int32).expand(S, N).contiguous().to(dev), torch.rand(S, N).to(dev))
        first = torch.where(count > 0, tokens.gather(1, path[:, :1].clamp(min=0).long())[:, 0], last)
        share = torch.bincount(first.long(), minlength=V).double().cpu() / S
        assert float(((share - p).abs() / (p * (1 - p) / S).sqrt()).max()) < 5


def test_verify_rows_past_32_bits(dev):
    """Rows more than 2^32 bytes into the probabilities, and the largest tree."""
    from oracle import serving

    announce("verify far rows")
    S, N, V = 10, 64, 2000000  # 5.1 GB
    target = torch.zeros(S, N, V, device=dev)
    target[..., 1000:1100] = torch.rand(S, N, 100, device=dev) / 100
    tokens = torch.randint(1000, 1100, (S, N), dtype=torch.int32)
    parents, u = _parents(3, S, N, 4), torch.rand(S, N)
    got = torch.ops.mi355.verify_draft(target, None, tokens.to(dev), parents.to(dev), u.to(dev))
    want = serving.verify_ref(target[..., 1000:1100].cpu(), None, tokens - 1000, parents, u)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1]) and torch.equal(got[2].cpu() - 1000, want[2])


def test_verify_captured_twice(dev):
    """Two captured calls replayed on two streams at once, with new random numbers between the replays."""
    announce("verify captured")
    ins = [t.to(dev) for t in _inputs(6, 8, 9, 5000, 3, True)]
    torch.ops.mi355.verify_draft(*ins)
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    graphs = []
    for _ in streams:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = torch.ops.mi355.verify_draft(*ins)
        graphs.append((g, outs))
    for k in range(4):
        ins[4].copy_(torch.rand(8, 9))
        torch.cuda.synchronize()
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        want = torch.ops.mi355.verify_draft(*ins)
        for _, outs in graphs:
            assert all(torch.equal(a, b) for a, b in zip(outs, want))
