"""GPU parity: block tables and slot maps built on the device; whole numbers, equal to the oracle's."""

import random

import pytest
import torch

import iree_turbine_amd  # noqa: F401  (registers torch.ops.mi355)
from conftest import announce

pytestmark = pytest.mark.gpu


def _case(seed, S, page, ctx_max, new_max, spare_pages=3, width_off=0):
    rng = random.Random(seed)
    ctx = [rng.randrange(0, ctx_max + 1) for _ in range(S)]
    new = [rng.randrange(0, new_max + 1) for _ in range(S)]
    have = [-(-c // page) for c in ctx]
    need = [-(-(c + n) // page) - h for c, n, h in zip(ctx, new, have)]
    width = max(1, max(h + n for h, n in zip(have, need)) + width_off)
    ids = list(range(sum(have) + sum(need) + spare_pages))
    rng.shuffle(ids)
    table = torch.full((S, width), -1, dtype=torch.int32)
    at = 0
    for s, h in enumerate(have):
        h = min(h, width)
        table[s, :h] = torch.tensor(ids[at:at + h], dtype=torch.int32)
        at += h
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)
    return table, i32(ctx), i32(new), i32(ids[at:]), sum(new)


def _check(dev, table, ctx, new, free, page, rows, what):
    from oracle import serving

    announce(what)
    want = serving.batch_layout_ref(table, ctx, new, free, page, rows)
    td = table.to(dev)
    got = torch.ops.mi355.paged_batch_layout(td, ctx.to(dev), new.to(dev), free.to(dev), page, rows)
    assert torch.equal(td.cpu(), want[0])
    for name, g, w in zip(("seq_lens", "cu_new", "positions", "seq_ids", "slots", "pages_needed"), got, want[1:]):
        assert g.tolist() == w, name
    again = torch.ops.mi355.paged_batch_layout(td, ctx.to(dev), new.to(dev), free.to(dev), page, rows)
    assert torch.equal(td.cpu(), want[0]) and all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("S,page,ctx_max,new_max", [(1, 16, 0, 1), (1, 16, 100, 3000), (3, 32, 50, 5), (64, 16, 900, 1), (100, 256, 700, 90), (1023, 16, 40, 3),
                                                    (1024, 64, 40, 3), (1025, 16, 60, 3), (2500, 32, 30, 4)])
def test_layout(dev, S, page, ctx_max, new_max):
    table, ctx, new, free, total = _case(S + page, S, page, ctx_max, new_max)
    _check(dev, table, ctx, new, free, page, max(1, total), f"layout S={S} page={page}")
    _check(dev, table, ctx, new, free, page, total + 1500, f"layout S={S} page={page}, padded rows")


def test_layout_borders(dev):
    """Lengths on page borders, empty sequences in front, between and behind, negative lengths."""
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)
    ctx = i32(0, 16, 15, 17, 0, -3, 32, 31, 5, 0)
    new = i32(0, 16, 1, 15, 16, 17, 0, 2, -4, 0)
    table = torch.arange(40, dtype=torch.int32).reshape(10, 4) + 100
    free = torch.arange(50, dtype=torch.int32)
    for rows in (67, 68, 1, 16, 17, 200):
        _check(dev, table, ctx, new, free, 16, rows, f"layout borders rows={rows}")


def test_layout_runs_out_of_pages_and_table(dev):
    """Too short a free list leaves -1 behind its end, a table too narrow leaves its tokens without a slot, and stale or
    missing ids of cached pages give no slot."""
    table, ctx, new, free, total = _case(5, 20, 16, 100, 60)
    _check(dev, table, ctx, new, free[:7], 16, total, "layout with 7 free pages")
    _check(dev, table, ctx, new, free[:0], 16, total, "layout without free pages")
    narrow = table[:, :4].contiguous()
    _check(dev, narrow, ctx, new, free, 16, total, "layout with a narrow table")
    holes = table.clone()
    holes[::2] = -7
    _check(dev, holes, ctx, new, free, 16, total, "layout with missing pages")


def test_layout_large_lengths(dev):
    """Sums past 32 bits are cut to the rows there are; positions far out have no slot."""
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)
    from oracle import serving  # noqa: F401

    announce("layout large lengths")
    big = 2**31 - 1
    table = torch.full((3, 4), 9, dtype=torch.int32)
    td = table.to(dev)
    got = torch.ops.mi355.paged_batch_layout(td, i32(big, 60, 0).to(dev), i32(5, big, big).to(dev), i32(1, 2, 3).to(dev), 16, 12)
    assert got[0].tolist() == [big, 67, 0] and got[1].tolist() == [0, 5, 12, 12]
    assert got[2].tolist() == [big] * 5 + [60, 61, 62, 63, 64, 65, 66]
    assert got[3].tolist() == [0] * 5 + [1] * 7
    assert got[4].tolist() == [-1] * 5 + [9 * 16 + i for i in range(12, 16)] + [-1] * 3 and got[5].tolist() == [0]


def test_layout_captured(dev):
    announce("layout captured")
    table, ctx, new, free, total = _case(9, 40, 16, 300, 20)
    td, cd, nd, fd = (t.to(dev) for t in (table, ctx, new, free))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = torch.ops.mi355.paged_batch_layout(td, cd, nd, fd, 16, total + 5)
    for k in range(3):
        nd.copy_((new - k).to(dev))
        td.copy_(table.to(dev))
        graph.replay()
        torch.cuda.synchronize()
        t2 = table.to(dev)
        want = torch.ops.mi355.paged_batch_layout(t2, cd, nd, fd, 16, total + 5)
        assert torch.equal(td, t2) and all(torch.equal(a, b) for a, b in zip(outs, want))
