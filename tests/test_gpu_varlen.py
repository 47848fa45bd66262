"""GPU parity: attention over packed sequences against the 64-bit oracle, within the bound that it derives."""

import ctypes

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


def _run(dev, lq, lk, hq, hkv, causal, dtype, scale=0.0, spread=1.0, pad=0):
    from oracle import serving

    q = (torch.randn(sum(lq) + pad, hq, 128) * spread).to(dtype)
    k, v = ((torch.randn(max(1, sum(lk) + pad), hkv, 128)).to(dtype) for _ in range(2))
    cq, ck = _cu(lq), _cu(lk)
    got = torch.ops.mi355.flash_attn_varlen_fwd(q.to(dev), k.to(dev), v.to(dev), cq.to(dev), ck.to(dev), causal, scale)
    want, bound = serving.varlen_ref(q, k, v, cq, ck, causal, scale or None)
    _inside(got, want, bound)
    return got


LENGTHS = [[1], [1, 1, 1], [5, 0, 130, 1, 64], [127, 128, 129], [63, 65, 300, 2], [0, 0, 17], [257]]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens", LENGTHS, ids=str)
def test_self_attention(dev, lens, causal):
    announce(f"varlen lens={lens} causal={causal}")
    _run(dev, lens, lens, 4, 2, causal, torch.bfloat16)
    _run(dev, lens, lens, 3, 3, causal, torch.float16, pad=3)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_keys_in_front_and_missing(dev, dtype, causal):
    """More keys than queries (an earlier part of the prompt), fewer (the first queries see nothing under the mask), none."""
    announce(f"varlen unequal lengths {dtype} causal={causal}")
    got = _run(dev, [3, 70, 129, 200, 5, 1], [90, 70, 1, 60, 0, 500], 8, 2, causal, dtype)
    assert torch.equal(got[402:407].cpu(), torch.zeros(5, 8, 128, dtype=dtype))
    if causal:
        assert torch.equal(got[73:73 + 128].cpu(), torch.zeros(128, 8, 128, dtype=dtype))


@pytest.mark.parametrize("hq,hkv", [(1, 1), (16, 1), (8, 8), (32, 8), (24, 8), (16, 16), (5, 1)])
def test_head_layouts(dev, hq, hkv):
    announce(f"varlen hq={hq} hkv={hkv}")
    _run(dev, [100, 1, 40, 190], [100, 1, 40, 190], hq, hkv, True, torch.float16)


CUT = [([1], [4000], 4, 1), ([1, 1, 1], [1500, 2, 2600], 16, 2), ([33, 0, 7, 64], [1900, 300, 0, 1300], 16, 1), ([130], [2500], 8, 8),
       ([5, 16, 2, 40, 9], [900, 1033, 1024, 1088, 640], 5, 1), ([1100, 3], [1100, 1600], 8, 2), ([300], [200], 2, 2), ([700, 600], [700, 600], 3, 3), ([20] * 64, [600] * 64, 4, 1)]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lq,lk,hq,hkv", CUT, ids=lambda x: str(x)[:30])
def test_keys_cut_into_chunks(dev, lq, lk, hq, hkv, dtype, causal):
    """Few query rows and many keys: every block's keys in up to 16 chunks, joined; the same bits on every call, rows outside
    left alone, and without a workspace the uncut call within the rounding."""
    from iree_turbine_amd import _lib, launch
    from oracle import serving

    announce(f"varlen chunks lq={lq[:5]} lk={lk[:5]} hq={hq} {dtype} causal={causal}")
    T, Tk = sum(lq) + 5, sum(lk) + 3
    lib = _lib.load()
    assert (lib.mi355_flash_attn_varlen_workspace_bytes(len(lq), T, Tk, hq, hkv, causal) > 0) == (lk not in ([200], [700, 600], [600] * 64))
    q, k, v = (torch.randn(t, h, 128).to(dtype) for t, h in ((T, hq), (Tk, hkv), (Tk, hkv)))
    cq, ck = _cu(lq, first=2), _cu(lk, first=1)
    k[int(ck[-1]):], v[int(ck[-1]):], k[0], v[0] = float("nan"), float("inf"), float("inf"), float("nan")
    args = [t.to(dev) for t in (q, k, v, cq, ck)]
    want, bound = serving.varlen_ref(q, torch.nan_to_num(k, 0.0, 0.0, 0.0), torch.nan_to_num(v, 0.0, 0.0, 0.0), cq, ck, causal)
    got = torch.ops.mi355.flash_attn_varlen_fwd(*args, causal, 0.0)
    _inside(got, want, bound)
    o = torch.full((T, 2 * hq, 128), 7.0, dtype=dtype, device=dev)
    launch.flash_attn_varlen_fwd_out(*args, o[:, hq:], causal, 0.0)
    inside = slice(int(cq[0]), int(cq[-1]))
    assert torch.equal(o[inside, hq:], got[inside])
    o[inside, hq:] = 7.0
    assert torch.equal(o, torch.full_like(o, 7.0))
    st = lambda t: (ctypes.c_int64 * 2)(t.stride(0), t.stride(1))
    plain = torch.zeros_like(got)
    rc = lib.mi355_flash_attn_varlen_fwd(*(t.data_ptr() for t in (*args[:3], plain, *args[3:])), len(lq), T, Tk, hq, hkv, 128, *(st(t) for t in (*args[:3], plain)),
                                         128**-0.5, causal, 0, _lib.dtype_code(dtype), None, 0, _lib.raw_stream(dev))
    assert rc == 0
    _inside(plain, want, bound)


def test_chunks_on_two_streams_and_captured(dev):
    """Calls at once and two captured ones keep scratch of their own."""
    announce("varlen chunks streams and capture")
    q, k, v = (torch.randn(t, h, 128).half().to(dev) for t, h in ((40, 8), (6000, 2), (6000, 2)))
    cq, ck = _cu([30, 2, 8]).to(dev), _cu([3000, 2000, 1000]).to(dev)
    call = lambda: torch.ops.mi355.flash_attn_varlen_fwd(q, k, v, cq, ck, True, 0.0)
    want = call()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    outs, graphs = [], []
    for s in streams:
        with torch.cuda.stream(s):
            outs += [call() for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        graphs.append((g, out))
    for lens in ([3000, 2000, 1000], [0, 4000, 2000], [100, 5000, 64]):
        ck.copy_(_cu(lens))
        torch.cuda.synchronize()
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        eager = call()
        assert all(torch.equal(out, eager) for _, out in graphs)


@pytest.mark.parametrize("S", [63, 64, 65, 130, 300])
def test_many_sequences(dev, S):
    announce(f"varlen {S} sequences")
    lens = [(7 * s * s + 3) % 23 if s % 5 else 0 for s in range(S)]
    lens[S // 2], lens[-1] = 180, 150
    _run(dev, lens, lens, 2, 1, True, torch.bfloat16)


def test_scores_far_apart(dev):
    """Large scores (a softmax that picks single keys), and a scale of one's own."""
    announce("varlen far scores")
    _run(dev, [150, 33], [150, 33], 2, 2, True, torch.float16, spread=12.0)
    _run(dev, [150, 33], [150, 33], 2, 2, True, torch.bfloat16, scale=0.5)


@pytest.mark.parametrize("causal", [True, False])
def test_neighbours_do_not_leak(dev, causal):
    """Keys and values of other sequences and behind the last one hold NaN and infinities: nobody else sees them, and the
    rows behind the last sequence are zeros from the op and left alone by the launcher."""
    from iree_turbine_amd import launch
    from oracle import serving

    announce(f"varlen neighbours causal={causal}")
    lens = [70, 33, 129, 5]
    cu = _cu(lens, first=6)
    T = int(cu[-1]) + 9
    q, k, v = (torch.randn(T, h, 128).half() for h in (4, 2, 2))
    for rows in (slice(0, 6), slice(76, 109), slice(int(cu[-1]), T)):
        k[rows], v[rows] = float("nan"), float("inf")
    got = torch.ops.mi355.flash_attn_varlen_fwd(q.to(dev), k.to(dev), v.to(dev), cu.to(dev), cu.to(dev), causal, 0.0)
    clean = torch.ones(T, dtype=torch.bool)
    clean[76:109] = False
    want, bound = serving.varlen_ref(q, torch.nan_to_num(k, 0.0, 0.0), torch.nan_to_num(v, 0.0, 0.0, 0.0), cu, cu, causal)
    _inside(got.cpu()[clean], want[clean], bound[clean])
    outside = torch.ones(T, dtype=torch.bool)
    outside[6:int(cu[-1])] = False
    assert torch.equal(got.cpu()[outside], torch.zeros(15, 4, 128).half())
    o = torch.full((T, 4, 128), 7.0, dtype=torch.float16, device=dev)
    launch.flash_attn_varlen_fwd_out(q.to(dev), k.to(dev), v.to(dev), cu.to(dev), cu.to(dev), o, causal, 0.0)
    assert torch.equal(o.cpu()[outside], torch.full((15, 4, 128), 7.0).half())
    assert torch.equal(o.cpu()[~outside & clean], got.cpu()[~outside & clean])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,hq,hkv", [([150, 40, 5], 4, 2), ([700], 8, 8), ([2048, 300], 32, 8)], ids=["64 rows", "one", "128 rows"])
def test_later_tokens_do_not_leak(dev, lens, hq, hkv, dtype):
    """A token whose key and value hold NaN or infinities changes nothing for the queries in front of it, also in the tile
    that both lie in; queries that see an infinite value get an infinity in its column, one that sees a NaN gets NaN."""
    from oracle import serving

    announce(f"varlen later tokens lens={lens} {dtype}")
    cu = _cu(lens)
    q, k, v = (torch.randn(sum(lens), h, 128).to(dtype) for h in (hq, hkv, hkv))
    bad = [min(9, lens[0] - 1), lens[0] - 1]
    kb, vb = k.clone(), v.clone()
    kb[bad[1]] = float("nan")
    vb[bad[1]] = float("inf")
    vb[bad[0], 0, 5], vb[bad[0], 0, 77], vb[bad[0], hkv - 1, 127] = float("inf"), float("-inf"), float("nan")
    args = [t.to(dev) for t in (q, kb, vb, cu, cu)]
    got = torch.ops.mi355.flash_attn_varlen_fwd(*args, True, 0.0).cpu()
    want, bound = serving.varlen_ref(q[:300], k[:300], v[:300], torch.tensor([0, min(300, lens[0])]), torch.tensor([0, min(300, lens[0])]), True)
    front = got[: bad[0]].double()
    assert torch.isfinite(front).all() and bool(((front - want[: bad[0]]).abs() <= bound[: bad[0]]).all())
    seen = got[bad[0] : bad[1]]
    g = hq // hkv
    if len(seen):
        assert bool((seen[:, :g, 5] == float("inf")).all()) and bool((seen[:, :g, 77] == float("-inf")).all()) and bool(seen[:, hq - g :, 127].isnan().all())
        clear = torch.ones(128, dtype=torch.bool)
        clear[[5, 77, 127]] = False
        n = min(bad[1], len(want))
        off = (got[bad[0] : n].double() - want[bad[0] : n]).abs() - bound[bad[0] : n]
        assert float(off[..., clear].max()) <= 0
    assert bool(got[bad[1]].isnan().all())
    other = torch.ops.mi355.flash_attn_varlen_fwd(*(t.to(dev) for t in (q, k, v, cu, cu)), True, 0.0).cpu()
    assert torch.equal(got[lens[0]:], other[lens[0]:])


def test_offsets_outside_the_stream(dev):
    """Wild offsets are cut to the stream; a sequence that ends before it begins is empty."""
    announce("varlen wild offsets")
    q, k, v = (torch.randn(50, 2, 128).half() for _ in range(3))
    wild = torch.tensor([-9, 20, 2**31 - 1], dtype=torch.int32)
    tame = torch.tensor([0, 20, 50], dtype=torch.int32)
    a, b = (torch.ops.mi355.flash_attn_varlen_fwd(q.to(dev), k.to(dev), v.to(dev), c.to(dev), c.to(dev), True, 0.0) for c in (wild, tame))
    assert torch.equal(a, b)
    back = torch.tensor([0, 30, 10, 50], dtype=torch.int32)
    got = torch.ops.mi355.flash_attn_varlen_fwd(q.to(dev), k.to(dev), v.to(dev), back.to(dev), torch.tensor([0, 30, 30, 30], dtype=torch.int32).to(dev), True, 0.0)
    assert got.shape == q.shape


def test_offsets_outside_the_stream_in_chunks(dev):
    """The same where the keys are cut into chunks."""
    announce("varlen wild offsets, chunks")
    q, k, v = (torch.randn(t, 2, 128).half().to(dev) for t in (50, 4000, 4000))
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)
    a = torch.ops.mi355.flash_attn_varlen_fwd(q, k, v, i(-9, 20, 2**31 - 1), i(-5, 1500, 2**31 - 1), True, 0.0)
    b = torch.ops.mi355.flash_attn_varlen_fwd(q, k, v, i(0, 20, 50), i(0, 1500, 4000), True, 0.0)
    assert torch.equal(a, b) and torch.isfinite(a).all()
    got = torch.ops.mi355.flash_attn_varlen_fwd(q, k, v, i(0, 30, 10, 50), i(0, 3000, 10, 4000), True, 0.0)
    torch.cuda.synchronize()
    assert got.shape == q.shape
    # a sequence whose keys begin behind its end, one without keys, one without queries
    c = torch.ops.mi355.flash_attn_varlen_fwd(q, k, v, i(0, 20, 40, 40, 50), i(3000, 3000, 3000, 3500, 4000), False, 0.0)
    assert torch.equal(c[:40], torch.zeros_like(c[:40])) and bool((c[40:] != 0).any(-1).all())


def test_agrees_with_the_rectangular_op_and_reads_slices(dev):
    """Equal lengths: the rectangular op's result within the two kernels' rounding; slices of a packed projection are read
    in place and give the same bits as copies; so do rows off the 16-byte borders, which are copied."""
    announce("varlen against flash_attn_fwd")
    B, L, hq, hkv = 3, 200, 8, 2
    qkv = torch.randn(B * L, hq + 2 * hkv, 128).bfloat16().to(dev)
    q, k, v = qkv.split([hq, hkv, hkv], 1)
    cu = _cu([L] * B).to(dev)
    got = torch.ops.mi355.flash_attn_varlen_fwd(q, k, v, cu, cu, True, 0.0)
    rect = torch.ops.mi355.flash_attn_fwd(*(t.unflatten(0, (B, L)).transpose(1, 2) for t in (q, k, v)), True, 0.0)
    torch.testing.assert_close(got, rect.transpose(1, 2).reshape(B * L, hq, 128), rtol=2e-2, atol=2e-2)
    copies = torch.ops.mi355.flash_attn_varlen_fwd(q.contiguous(), k.contiguous(), v.contiguous(), cu, cu, True, 0.0)
    assert torch.equal(got, copies)
    odd = torch.empty(B * L * 12 * 128 + 1, dtype=torch.bfloat16, device=dev)[1:].view(B * L, 12, 128).copy_(qkv)
    assert odd.data_ptr() % 16
    assert torch.equal(got, torch.ops.mi355.flash_attn_varlen_fwd(*odd.split([hq, hkv, hkv], 1), cu, cu, True, 0.0))
    one = torch.ops.mi355.flash_attn_varlen_fwd(q, k[:, :1].expand(-1, hkv, -1), v, cu, cu, True, 0.0)
    same = torch.ops.mi355.flash_attn_varlen_fwd(q, k[:, :1].repeat(1, hkv, 1), v, cu, cu, True, 0.0)
    assert torch.equal(one, same)


def test_captured_for_any_lengths(dev):
    """One captured call serves other lengths in the same buffers: offsets are read on the device."""
    announce("varlen captured")
    T = 300
    q, k, v = (torch.randn(T, h, 128).half().to(dev) for h in (4, 2, 2))
    cu = _cu([100, 50, 150]).to(dev)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        torch.ops.mi355.flash_attn_varlen_fwd(q, k, v, cu, cu, True, 0.0)
    torch.cuda.current_stream(dev).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = torch.ops.mi355.flash_attn_varlen_fwd(q, k, v, cu, cu, True, 0.0)
    for lens in ([100, 50, 150], [1, 298, 1], [0, 300, 0], [20, 20, 20]):
        cu.copy_(_cu(lens))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, torch.ops.mi355.flash_attn_varlen_fwd(q, k, v, cu, cu, True, 0.0))


@pytest.mark.parametrize("lens", [[2300, 1], [2, 4, 2400]], ids=["chunks", "last"])
def test_rows_past_32_bit_offsets(dev, lens):
    """Rows a mebi-element apart: the last ones lie more than 2^32 bytes behind the first."""
    from oracle import serving

    announce(f"varlen far rows {lens}")
    T, pitch = sum(lens), 1 << 20
    far = torch.empty(T * pitch, dtype=torch.bfloat16, device=dev).view(T, pitch)
    assert far.numel() * 2 > 2**32
    q, k, v, o = (far[:, 256 * i : 256 * i + 256].view(T, 2, 128) for i in range(4))
    host = [torch.randn(T, 2, 128).bfloat16() for _ in range(3)]
    for t, h in zip((q, k, v), host):
        t.copy_(h)
    cu = _cu(lens)
    want, bound = serving.varlen_ref(*host, cu, cu, True)
    _inside(torch.ops.mi355.flash_attn_varlen_fwd(q, k, v, cu.to(dev), cu.to(dev), True, 0.0), want, bound)
    from iree_turbine_amd import launch

    launch.flash_attn_varlen_fwd_out(q, k, v, cu.to(dev), cu.to(dev), o, True, 0.0)
    _inside(o, want, bound)
