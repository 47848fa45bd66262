"""GPU parity: the forms of the packed attention and of the draft verification that only large calls are dispatched to, on
the smallest such calls."""

import pytest
import torch

import iree_turbine_amd  # noqa: F401  (registers torch.ops.mi355)
from conftest import announce

pytestmark = pytest.mark.gpu


def _cu(lens, first=0):
    return torch.cumsum(torch.tensor([first] + list(lens)), 0).int()


def _inside(got, want, bound):
    off = (got.double().cpu() - want).abs()
    assert torch.isfinite(got).all()
    worst = (off - bound).max().item()
    assert worst <= 0, f"off by {off.max().item():.3g}, {worst:.3g} more than the bound allows"


def _rows_of(n, group):
    """Tokens of a sequence of n: the first, the last, those at the borders of blocks of 128 rows, and some between."""
    per = max(1, 128 // group)
    picked = {0, 1, n // 2, n - 2, n - 1}
    for b in range(0, n, per):
        if b // per < 3 or b + 3 * per >= n:
            picked |= {b - 1, b, b + per // 2}
    return sorted(t for t in picked if 0 <= t < n)


def _check_rows(got, q, k, v, cq, ck, causal):
    from oracle import serving

    group = q.shape[1] // k.shape[1]
    for a, b, c, d in zip(cq.tolist(), cq.tolist()[1:], ck.tolist(), ck.tolist()[1:]):
        rows = torch.tensor(_rows_of(b - a, group), dtype=torch.long)
        if len(rows) == 0:
            continue
        visible = torch.ones(len(rows), d - c, dtype=torch.bool)
        if causal:
            visible = torch.arange(d - c)[None] <= (rows + (d - c) - (b - a))[:, None]
        _inside(got[a + rows], *serving.attention_ref(q[a + rows], k[c:d], v[c:d], visible))


# 128-row blocks from 512 of them on (per K/V head, all heads), the masked ones in pairs from 2048 on; heads instead of
# tokens make them many.  Odd and even numbers of blocks in a sequence, groups of 1, 3, 8 and 9 heads, K/V heads that divide over
# eight and that do not.
LARGE = {
    "single, 8 a group": ([513, 0, 1, 300, 300], [513, 0, 1, 300, 300], 64, 8, False),
    "single, 9 a group, prefixes": ([60, 400, 1, 400], [500, 400, 700, 30], 81, 9, False),
    "single, 3 a group": ([129, 740, 2, 400], [129, 740, 2, 400], 54, 18, False),
    "pairs, 8 a group": ([300, 17, 1, 0, 650, 140], [300, 17, 1, 0, 650, 140], 256, 32, True),
    "pairs, 1 a group": ([129, 128, 1, 400, 385], [129, 128, 1, 400, 385], 260, 260, True),
    "pairs, 3 a group, prefixes": ([43, 300, 85, 2, 86, 600], [500, 300, 20, 900, 0, 640], 240, 80, True),
}


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("name", LARGE)
def test_packed_attention_of_many_blocks(dev, name, dtype, causal):
    lq, lk, hq, hkv, pairs = LARGE[name]
    announce(f"varlen many blocks {name} {dtype} causal={causal}")
    blocks = sum(lq) * (hq // hkv) // 128 * hkv
    assert blocks >= 512 and (blocks >= 2048) == pairs
    q, k, v = (torch.randn(sum(n), h, 128).to(dtype) for n, h in ((lq, hq), (lk, hkv), (lk, hkv)))
    cq, ck = _cu(lq), _cu(lk)
    args = [t.to(dev) for t in (q, k, v, cq, ck)]
    got = torch.ops.mi355.flash_attn_varlen_fwd(*args, causal, 0.0)
    _check_rows(got.cpu(), q, k, v, cq, ck, causal)
    assert torch.equal(got, torch.ops.mi355.flash_attn_varlen_fwd(*args, causal, 0.0))


@pytest.mark.parametrize("name", ["single, 8 a group", "pairs, 8 a group", "pairs, 1 a group"])
def test_later_tokens_do_not_leak_in_many_blocks(dev, name):
    """Non-finite keys and values change nothing for the queries in front of them, in either block of a pair."""
    lq, _, hq, hkv, _ = LARGE[name]
    announce(f"varlen later tokens {name}")
    cu = _cu(lq)
    q, k, v = (torch.randn(sum(lq), h, 128).bfloat16() for h in (hq, hkv, hkv))
    clean = torch.ops.mi355.flash_attn_varlen_fwd(*(t.to(dev) for t in (q, k, v, cu, cu)), True, 0.0).cpu()
    kb, vb, front = k.clone(), v.clone(), torch.ones(sum(lq), dtype=torch.bool)
    for a, b in zip(cu.tolist(), cu.tolist()[1:]):
        if b - a > 20:
            at = a + (b - a) // 3  # an infinite value in the sequence's first half, a NaN key near its end
            vb[at, :, 7], kb[b - 3], vb[b - 3] = float("inf"), float("nan"), float("-inf")
            front[at:b] = False
            got_inf = (at, b - 3)
    got = torch.ops.mi355.flash_attn_varlen_fwd(*(t.to(dev) for t in (q, kb, vb, cu, cu)), True, 0.0).cpu()
    _check_rows(clean, q, k, v, cu, cu, True)
    assert torch.equal(got[front], clean[front])
    seen = got[got_inf[0] : got_inf[1]]
    assert bool((seen[..., 7] == float("inf")).all()) and bool(torch.isfinite(seen[..., [0, 6, 8, 127]]).all())
    assert bool(got[got_inf[1] : got_inf[1] + 3].isnan().all())


def test_falling_offsets(dev):
    """A sequence that ends before it begins is empty: the rows that one sequence alone claims are that one's."""
    from oracle import serving

    announce("varlen falling offsets")
    for S, T, H in ((4, 60, 2), (4, 60, 16)):
        q, k, v = (torch.randn(T, H, 128).half() for _ in range(3))
        # sequence 1 falls, 2 claims rows 20 .. 49 (without keys) of which 20 .. 29 belong to sequence 0 as well
        cq, ck = torch.tensor([0, 30, 20, 50, 60], dtype=torch.int32), torch.tensor([0, 30, 30, 30, 60], dtype=torch.int32)
        got = torch.ops.mi355.flash_attn_varlen_fwd(*(t.to(dev) for t in (q, k, v, cq, ck)), True, 0.0).cpu()
        _inside(got[:20], *(t[:20] for t in serving.varlen_ref(q[:30], k[:30], v[:30], cq[:2], ck[:2], True)))
        assert torch.equal(got[30:50], torch.zeros(20, H, 128).half())
        _inside(got[50:], *serving.varlen_ref(q[50:], k[30:], v[30:], torch.tensor([0, 10]), torch.tensor([0, 30]), True))


def _rejecting(S, N, V, seed):
    """Stars of N - 1 siblings with draft probabilities; sequence s rejects its first s % N of them and takes the next."""
    g = torch.Generator().manual_seed(seed)
    target = torch.softmax(2 * torch.randn(S, N, V, generator=g), -1)
    draft = torch.softmax(2 * torch.randn(S, N, V, generator=g), -1)
    parents = torch.tensor([[-1] + [0] * (N - 1)] * S, dtype=torch.int32)
    ratio = draft[:, 0] / target[:, 0]
    refused, taken = ratio.topk(N, -1)[1], (-ratio).topk(N, -1)[1]
    tokens, u = torch.zeros(S, N, dtype=torch.int32), torch.rand(S, N, generator=g)
    for s in range(S):
        k = s % N
        tokens[s, 1:] = refused[s, 1:]
        u[s, 1:] = 0.9999
        if 1 + k < N:
            tokens[s, 1 + k], u[s, 1 + k] = taken[s, 0], 0.0
    return target, draft, tokens, parents, u


@pytest.mark.parametrize("S,N,V", [(7, 7, 65537), (3, 3, 65536), (64, 6, 65537), (6, 6, 262145), (8, 8, 300001), (4, 4, 30000)],
                         ids=["one past a launch each", "two launches", "several batches a wave", "two blocks a piece", "more rejections than launches", "one launch"])
def test_verify_siblings_rejected_with_draft_probabilities(dev, S, N, V):
    """Every number of rejections from none to all, over rows whose sums several launches make."""
    from oracle import serving

    announce(f"verify rejections S={S} N={N} V={V}")
    ins = _rejecting(S, N, V, S * N)
    want = serving.verify_ref(*ins)
    assert want[0][:, 0].tolist() == [1 + s % N if 1 + s % N < N else -1 for s in range(S)]
    on = [t.to(dev) for t in ins]
    for _ in range(2):
        for name, a, b in zip(("path", "num_accepted", "next_token"), torch.ops.mi355.verify_draft(*on), want):
            assert torch.equal(a.cpu(), b), name
    # certain drafts over the same rows
    none = (ins[0], None, *ins[2:])
    for a, b in zip(torch.ops.mi355.verify_draft(on[0], None, *on[2:]), serving.verify_ref(*none)):
        assert torch.equal(a.cpu(), b)
    # deeper walks: the same tokens as a chain that ends in a rejection at another depth each
    chain = torch.arange(-1, N - 1, dtype=torch.int32).expand(S, N).contiguous()
    u = torch.where(torch.arange(N)[None] <= torch.arange(S)[:, None] % N, 1e-6, 0.9999)
    u[:, 0] = ins[4][:, 0]
    deep = (ins[0], ins[0].clone(), ins[2], chain, u)
    deep[1][torch.arange(S), (torch.arange(S) % N).clamp(max=N - 1)] = ins[1][:, 0]
    for a, b in zip(torch.ops.mi355.verify_draft(*(t.to(dev) for t in deep)), serving.verify_ref(*deep)):
        assert torch.equal(a.cpu(), b)
