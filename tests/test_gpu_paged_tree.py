"""GPU parity: tree attention over the paged cache against the 64-bit oracle, within the bound that it derives."""

import random

import pytest
import torch

import iree_turbine_amd  # noqa: F401  (registers torch.ops.mi355)
from conftest import announce

pytestmark = pytest.mark.gpu


def _inside(got, want, bound):
    off = (got.double().cpu() - want).abs()
    assert torch.isfinite(got).all()
    worst = (off - bound).max().item()
    assert worst <= 0, f"off by {off.max().item():.3g}, {worst:.3g} more than the bound allows"


def _inputs(seed, lens, N, hq, hkv, page, dtype, poison=True):
    """Pages in random order; places behind a sequence's end and unused pages hold NaN, unused table entries wild ids."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-max(0, n) // page) for n in lens]
    P = sum(need) + 2
    kc, vc = (torch.full((P, page, hkv, 128), float("nan") if poison else 0.0).to(dtype) for _ in range(2))
    table = torch.full((len(lens), max(need) + 2), 2**30, dtype=torch.int32)
    order = torch.randperm(P, generator=g).tolist()
    for s, n in enumerate(lens):
        for p in range(need[s]):
            table[s, p] = order.pop()
            fill = min(page, n - p * page)
            for c in (kc, vc):
                c[table[s, p], :fill] = torch.randn(fill, hkv, 128, generator=g).to(dtype)
    q = torch.randn(len(lens), N, hq, 128, generator=g).to(dtype)
    return q, kc, vc, table, torch.tensor(lens, dtype=torch.int32)


def _parents(seed, S, N, branch):
    rng = random.Random(seed)
    return torch.tensor([[-1] + [rng.randrange(max(0, i - branch), i) for i in range(1, N)] for _ in range(S)], dtype=torch.int32)


def _check(dev, ins, parents, splits, scale=0.0):
    from oracle import serving

    q, kc, vc, table, lens = ins
    got = torch.ops.mi355.paged_tree_attn(*(t.to(dev) for t in (*ins, parents)), scale, splits)
    clean = [torch.nan_to_num(c, 0.0) for c in (kc, vc)]
    want, bound = serving.tree_ref(q, *clean, table, lens, parents, scale or None)
    _inside(got, want, bound)
    return got


@pytest.mark.parametrize("splits", [1, 2, 5, 0])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("N,hq,hkv,page", [(1, 4, 4, 16), (1, 8, 2, 16), (4, 8, 2, 32), (7, 32, 8, 16), (8, 16, 1, 64), (16, 8, 2, 256), (33, 3, 1, 16), (64, 8, 2, 128), (5, 14, 2, 16)])
def test_tree(dev, N, hq, hkv, page, dtype, splits):
    announce(f"tree N={N} hq={hq} hkv={hkv} page={page} {dtype} splits={splits}")
    lens = [N, N + 1, 200 + N, 31 + N, 515]
    _check(dev, _inputs(N, lens, N, hq, hkv, page, dtype), _parents(N, 5, N, 4), splits)


@pytest.mark.parametrize("splits", [1, 3, 0])
@pytest.mark.parametrize("S,N,hq", [(64, 3, 4), (65, 3, 4), (70, 12, 8), (64, 12, 8)])
def test_many_sequences(dev, S, N, hq, splits):
    """Up to 64 sequences are handed out by falling size, more chunk by chunk; lengths from none to several chunks."""
    announce(f"tree sequences={S} N={N} hq={hq} splits={splits}")
    rng = random.Random(S + N)
    lens = [rng.choice([0, 1, N, 31, 32, 33, rng.randrange(N, 700)]) for _ in range(S)]
    _check(dev, _inputs(S, lens, N, hq, 2, 16, torch.bfloat16), _parents(S, S, N, 3), splits)


@pytest.mark.parametrize("splits", [1, 3])
def test_tree_lengths_on_the_borders(dev, splits):
    """Drafts that start inside a 16-token block, across pages, sequences shorter than their drafts, empty and wild lengths."""
    announce(f"tree borders splits={splits}")
    lens = [5, 0, 3, 1, 15, 16, 17, 31, 32, 33, 36, 37, 64, 127, 128, 129, 133]
    ins = _inputs(3, lens, 5, 4, 2, 16, torch.float16)
    got = _check(dev, ins, _parents(9, len(lens), 5, 3), splits)
    assert torch.equal(got[1].cpu(), torch.zeros(5, 4, 128).half())
    q, kc, vc, table, sl = ins
    wild, tame = sl.clone(), sl.clone()
    wild[1], wild[16] = -9, 10**9
    tame[16] = table.shape[1] * 16
    par = _parents(9, len(lens), 5, 3)
    a, b = (torch.ops.mi355.paged_tree_attn(*(t.to(dev) for t in (q, torch.nan_to_num(kc, 0.0), torch.nan_to_num(vc, 0.0), table, s, par)), 0.0, splits) for s in (wild, tame))
    assert torch.equal(a, b)


@pytest.mark.parametrize("splits", [1, 4])
def test_bad_pages_are_dropped(dev, splits):
    announce(f"tree bad pages splits={splits}")
    ins = _inputs(5, [300, 200, 90], 6, 8, 2, 16, torch.bfloat16)
    table = ins[3]
    table[0, 0], table[0, 7], table[1, 3], table[1, 12] = -1, ins[1].shape[0], 2**30, -(2**31)
    table[2, :6] = -5
    got = _check(dev, ins, _parents(2, 3, 6, 2), splits)
    assert torch.equal(got[2].cpu(), torch.zeros(6, 8, 128).bfloat16())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("N,hq,hkv", [(4, 4, 2), (7, 8, 2), (12, 8, 2), (40, 8, 2)], ids=["16 rows", "32 rows", "64 rows", "160 rows"])
@pytest.mark.parametrize("splits", [1, 3])
def test_other_branches_do_not_leak(dev, splits, N, hq, hkv, dtype):
    """A draft that was never written (NaN and infinities in its place) changes nothing for nodes of other branches; its
    descendants see it: infinity where its value is infinite, NaN where its key is NaN."""
    from oracle import serving

    announce(f"tree other branches N={N} hq={hq} {dtype} splits={splits}")
    lens = [150 + N, N, 64 + N]
    q, kc, vc, table, sl = _inputs(3, lens, N, hq, hkv, 16, dtype)
    par = torch.tensor([[-1, 0, 0, 1] + [1] * (N - 4)] * 3, dtype=torch.int32)  # node 2 has no children, node 3 is node 1's
    place = lambda s, n: (int(table[s, (lens[s] - N + n) // 16]), (lens[s] - N + n) % 16)
    want, bound = serving.tree_ref(q, torch.nan_to_num(kc, 0.0), torch.nan_to_num(vc, 0.0), table, sl, par)
    for s in range(3):
        p, at = place(s, 2)
        kc[p, at], vc[p, at] = float("nan"), float("inf")
        p, at = place(s, 3)
        vc[p, at, 0, 9], vc[p, at, hkv - 1, 100] = float("-inf"), float("nan")
    got = torch.ops.mi355.paged_tree_attn(*(t.to(dev) for t in (q, kc, vc, table, sl, par)), 0.0, splits).cpu()
    others = [n for n in range(N) if n not in (2, 3)]
    off = (got[:, others].double() - want[:, others]).abs() - bound[:, others]
    assert torch.isfinite(got[:, others]).all() and float(off.max()) <= 0
    assert bool(got[:, 2].isnan().all())
    g = hq // hkv
    assert bool((got[:, 3, :g, 9] == float("-inf")).all()) and bool(got[:, 3, hq - g:, 100].isnan().all())
    clear = torch.ones(128, dtype=torch.bool)
    clear[[9, 100]] = False
    assert float(((got[:, 3].double() - want[:, 3]).abs() - bound[:, 3])[..., clear].max()) <= 0


def test_chain_is_paged_prefill(dev):
    """A chain is the causal mask: the prefill op's result within the two kernels' rounding; single nodes are decode."""
    announce("tree chain against prefill and decode")
    ins = _inputs(7, [400, 90, 33, 1000], 8, 16, 4, 16, torch.float16, poison=False)
    chain = (torch.arange(8, dtype=torch.int32) - 1).expand(4, 8).contiguous()
    d = [t.to(dev) for t in ins]
    a = torch.ops.mi355.paged_tree_attn(*d, chain.to(dev), 0.0, 2)
    b = torch.ops.mi355.paged_prefill_attn(*d, 0.0)
    torch.testing.assert_close(a, b, rtol=1e-2, atol=2e-3)
    q1 = d[0][:, :1].contiguous()
    a = torch.ops.mi355.paged_tree_attn(q1, *d[1:], chain[:, :1].contiguous().to(dev), 0.0, 3)
    b = torch.ops.mi355.paged_decode_attn(q1[:, 0].contiguous(), *d[1:], 0.0, 3)
    torch.testing.assert_close(a[:, 0], b, rtol=1e-2, atol=2e-3)


def test_parents_out_of_order_are_roots(dev):
    announce("tree parents")
    ins = _inputs(8, [50, 60, 70], 6, 4, 1, 16, torch.float16)
    par = torch.tensor([[5, 1, 1, 9, -7, 2], [0, 0, 1, 2, 3, 4], [-1, 2, 3, 4, 5, 0]], dtype=torch.int32)
    _check(dev, ins, par, 2)
    deep = (torch.arange(64, dtype=torch.int32) - 1).expand(3, 64).contiguous()
    _check(dev, _inputs(9, [64, 100, 500], 64, 2, 2, 16, torch.bfloat16), deep, 0)


def test_splits_and_placement_do_not_matter(dev):
    """Any number of chunks agrees with the oracle; the same call gives the same bits; wide scores and a scale of one's own."""
    announce("tree splits")
    ins = _inputs(11, [1500, 700], 9, 8, 2, 32, torch.bfloat16)
    par = _parents(4, 2, 9, 3)
    for splits in (1, 2, 7, 24, 1024):
        a, b = (_check(dev, ins, par, splits) for _ in range(2))
        assert torch.equal(a, b)
    _check(dev, (ins[0] * 8, *ins[1:]), par, 3)
    _check(dev, ins, par, 3, scale=0.4)


def test_caches_past_32_bit_offsets(dev):
    """Pages that lie more than 2^32 bytes into the cache."""
    from oracle import serving

    announce("tree far pages")
    page, hkv, P = 256, 8, 9000  # 9000 x 512 KiB = 4.7 GB each
    kc, vc = (torch.zeros(P, page, hkv, 128, dtype=torch.float16, device=dev) for _ in range(2))
    ids = [P - 1, 0, P - 2]
    for c in (kc, vc):
        for i in ids:
            c[i] = torch.randn(page, hkv, 128, device=dev).half()
    table, lens, par = torch.tensor([ids], dtype=torch.int32), torch.tensor([700], dtype=torch.int32), _parents(1, 1, 4, 2)
    q = torch.randn(1, 4, 16, 128).half()
    got = torch.ops.mi355.paged_tree_attn(q.to(dev), kc, vc, table.to(dev), lens.to(dev), par.to(dev), 0.0, 2)
    small = torch.tensor([[0, 1, 2]], dtype=torch.int32)
    want, bound = serving.tree_ref(q, kc[ids].cpu(), vc[ids].cpu(), small, lens, par)
    _inside(got, want, bound)


def test_two_streams_and_a_capture(dev):
    announce("tree streams and capture")
    ins = [t.to(dev) for t in _inputs(12, [900, 300, 60], 6, 8, 2, 16, torch.float16, poison=False)]
    par = _parents(5, 3, 6, 3).to(dev)
    want = torch.ops.mi355.paged_tree_attn(*ins, par, 0.0, 4)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    outs = []
    for s in streams:
        with torch.cuda.stream(s):
            outs.append([torch.ops.mi355.paged_tree_attn(*ins, par, 0.0, 4) for _ in range(5)])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for per in outs for o in per)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = torch.ops.mi355.paged_tree_attn(*ins, par, 0.0, 4)
        graphs.append((g, out))
    for k in range(3):
        ins[4].copy_(torch.tensor([900 - 100 * k, 300, 60 - k], dtype=torch.int32))
        torch.cuda.synchronize()
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        eager = torch.ops.mi355.paged_tree_attn(*ins, par, 0.0, 4)
        assert all(torch.equal(out, eager) for _, out in graphs)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("N,hq,hkv", [(4, 4, 1), (7, 8, 2), (12, 8, 2), (40, 8, 2)], ids=["16 rows", "32 rows", "64 rows", "160 rows"])
@pytest.mark.parametrize("splits", [1, 2])
def test_weights_add_up_to_one(dev, splits, N, hq, hkv, dtype):
    """Equal values come out as they went in, whatever the weights' rounding to 16 bits loses: one key of weight 1 and the
    others just below the middle between 1/2 and the next 16-bit number, all of which round down."""
    announce(f"tree equal values N={N} hq={hq} {dtype} splits={splits}")
    eps = torch.finfo(dtype).eps
    L = max(32, N + 20)
    k = torch.zeros(64, hkv, 128, dtype=dtype)
    k[1:, :, 0], k[1:, :, 1] = -1.0, 0.95 * eps / 2 / 0.6931  # 2^(-1 + d), about 1/2 (1 + 0.95 eps / 2)
    v = torch.full((64, hkv, 128), 2 - eps, dtype=dtype)
    q = torch.zeros(1, N, hq, 128, dtype=dtype)
    q[..., :2] = 1.0
    table, lens, par = torch.tensor([[0]], dtype=torch.int32), torch.tensor([L], dtype=torch.int32), _parents(1, 1, N, 3)
    weights = torch.exp2((k[:L, 0, 0] + k[:L, 0, 1]).double())
    lost = 1 - weights.to(dtype).double().sum() / weights.sum()
    assert float(lost) > eps / 4  # more than half a step of a value next to 2
    got = torch.ops.mi355.paged_tree_attn(*(t.to(dev) for t in (q, k[None], v[None], table, lens, par)), 0.6931471805599453, splits)
    assert torch.equal(got.cpu(), torch.full((1, N, hq, 128), 2 - eps, dtype=dtype))


@pytest.mark.parametrize("N,hq,hkv", [(4, 4, 2), (7, 8, 2), (12, 8, 2), (40, 8, 2)], ids=["16 rows", "32 rows", "64 rows", "160 rows"])
@pytest.mark.parametrize("lens", [[1300], [700, 0, 64, 1200, 33], [100, 900] + [70] * 68], ids=["one", "five", "seventy"])
def test_spare_columns_change_nothing(dev, lens, N, hq, hkv):
    """Keys are cut by the longest sequence: a block table with room for far longer ones gives the same bits, for any number of
    chunks, and cuts as finely."""
    announce(f"tree wide table N={N} hq={hq} sequences={len(lens)}")
    ins = _inputs(N, lens, N, hq, hkv, 16, torch.bfloat16)
    par = _parents(N, len(lens), N, 3)
    wide = torch.full((len(lens), 3000), -1, dtype=torch.int32)
    wide[:, : ins[3].shape[1]] = ins[3]
    whole = _check(dev, ins, par, 1)
    for splits in (2, 3, 16):
        a = _check(dev, ins, par, splits)
        assert torch.equal(a, _check(dev, (*ins[:3], wide, ins[4]), par, splits))
        assert not torch.equal(a, whole)
    # lengths wilder than either table's reach are cut to it
    wild = torch.where(ins[4] == max(lens), torch.tensor(2**31 - 1, dtype=torch.int32), ins[4])
    tame = torch.where(ins[4] == max(lens), torch.tensor(ins[3].shape[1] * 16, dtype=torch.int32), ins[4])
    clean = [torch.nan_to_num(c, 0.0).to(dev) for c in ins[1:3]]
    a, b = (torch.ops.mi355.paged_tree_attn(ins[0].to(dev), *clean, ins[3].to(dev), s.to(dev), par.to(dev), 0.0, 4) for s in (wild, tame))
    assert torch.equal(a, b)


def test_more_sequences_than_lengths_are_looked_at(dev):
    """From 513 sequences on the table's width is cut."""
    announce("tree 513 and 512 sequences")
    rng = random.Random(1)
    for S in (512, 513):
        lens = [rng.choice([0, 1, 5, 40, rng.randrange(200)]) for _ in range(S)]
        lens[7] = 300
        _check(dev, _inputs(S, lens, 3, 2, 1, 16, torch.float16), _parents(S, S, 3, 2), 3)
