"""GPU parity: rotary positions, their gradient, and the rotation fused with the cache append, against the 64-bit oracle
within the bound that it derives."""

import pytest
import torch

import iree_turbine_amd  # noqa: F401  (registers torch.ops.mi355)
from conftest import announce

pytestmark = pytest.mark.gpu


def _inside(got, want, bound, extra=0.0):
    off = (got.double().cpu() - want).abs()
    worst = (off - bound).max().item()
    assert worst <= extra, f"off by {off.max().item():.3g}, {worst:.3g} more than the bound allows"


def _freq(R, **kw):
    import iree_turbine_amd as ita

    return ita.rope_inv_freq(R, **kw)


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,H,D,R", [(1, 1, 128, 128), (5, 3, 128, 64), (33, 7, 96, 96), (4, 2, 80, 48), (3, 5, 66, 22), (7, 1, 2, 2), (2, 2, 1100, 1024), (9, 32, 64, 10), (70, 2, 80, 40), (3000, 1, 8, 8), (5000, 2, 72, 24)])
def test_rope(dev, T, H, D, R, dtype, inter):
    from oracle import serving

    announce(f"rope T={T} H={H} D={D} R={R} {dtype} interleaved={inter}")
    x = torch.randn(T, H, D).to(dtype)
    pos = torch.randint(0, 1 << 20, (T,), dtype=torch.int32)
    pos[0] = 0
    f, _ = _freq(R)
    for inverse in (False, True):
        got = torch.ops.mi355.rope(x.to(dev), pos.to(dev), f.to(dev), inter, inverse, 1.25)
        want, bound = serving.rope_ref(x, pos, f, inter, inverse, 1.25)
        _inside(got, want, bound)
        assert torch.equal(got.cpu()[..., R:], x[..., R:])


def test_rope_far_positions_and_32_bit_frequencies(dev):
    """The angle of the largest position is formed in 64 bits from either type of frequencies; negative positions turn back."""
    from oracle import serving

    announce("rope far positions")
    x = torch.randn(4, 2, 128)
    pos = torch.tensor([2**31 - 1, -(2**31), -5, 16777217], dtype=torch.int32)
    f, _ = _freq(128)
    for freq in (f, f.float()):
        got = torch.ops.mi355.rope(x.to(dev), pos.to(dev), freq.to(dev), False, False, 1.0)
        want, bound = serving.rope_ref(x, pos, freq, False)
        # the product of 2^31 rad, rounded once to 64 bits in the oracle and three times in the kernel (2^-22 each), on both of a pair
        _inside(got, want, bound + 8 * 2.0**-22 * x.abs().max())


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_rope_reads_strided_operands(dev, dtype):
    """Slices of a packed projection, rows off the 16-byte borders, transposed and broadcast operands, elements apart."""
    from oracle import serving

    announce(f"rope strided {dtype}")
    f, _ = _freq(64)
    pos = torch.arange(6, dtype=torch.int32) * 1000
    packed = torch.randn(6, 9, 128).to(dtype)
    odd = torch.randn(6, 4 * 131).to(dtype)
    cases = {
        "slice": packed[:, 2:5],
        "off the border": odd[:, 3:3 + 4 * 128].unflatten(1, (4, 128)),
        "odd row pitch": odd.as_strided((6, 4, 128), (4 * 131, 131, 1)),
        "transposed": torch.randn(4, 6, 128).to(dtype).transpose(0, 1),
        "heads broadcast": torch.randn(6, 1, 128).to(dtype).expand(6, 4, 128),
        "elements apart": torch.randn(6, 4, 256).to(dtype)[..., ::2],
    }
    for name, x in cases.items():
        base = x.to(dev) if name in ("transposed",) else None
        xd = torch.empty_strided(x.shape, x.stride(), dtype=dtype, device=dev).copy_(x) if 0 not in x.stride() else x[:, :1].to(dev).expand(x.shape)
        if name == "off the border":
            xd = odd.to(dev)[:, 3:3 + 4 * 128].unflatten(1, (4, 128))
        assert xd.stride() == x.stride(), name
        for inter in (False, True):
            got = torch.ops.mi355.rope(xd, pos.to(dev), f.to(dev), inter, False, 1.0)
            want, bound = serving.rope_ref(x, pos, f, inter)
            _inside(got, want, bound)


def test_rope_gradient(dev):
    """Autograd's gradient against the formula's and against differences; a leaf that is broadcast over heads sums its heads'."""
    from oracle import serving

    announce("rope gradient")
    f, scale = _freq(32, scaling="yarn", factor=8.0)
    pos = torch.tensor([0, 3, 900, 40000], dtype=torch.int32)
    for inter in (False, True):
        x = torch.randn(4, 3, 48)
        dy = torch.randn(4, 3, 48)
        leaf = x.to(dev).requires_grad_()
        y = torch.ops.mi355.rope(leaf, pos.to(dev), f.to(dev), inter, False, scale)
        got, = torch.autograd.grad(y, leaf, dy.to(dev), create_graph=False)
        want, bound = serving.rope_ref(dy, pos, f, inter, inverse=True, scale=scale)
        _inside(got, want, bound)
        # differences of the forward pass: it is linear, so a step of 1 has no truncation error
        d = torch.randn(4, 3, 48)
        up = torch.ops.mi355.rope((x + d).to(dev), pos.to(dev), f.to(dev), inter, False, scale).double().cpu()
        diff = ((up - y.detach().double().cpu()) * dy.double()).sum().item()
        # 2 x 576 results, each off by 2^-19 of its size (about 4) at most, times dy
        assert abs(diff - (got.double().cpu() * d.double()).sum().item()) < 2 * 576 * 2.0**-19 * 4 * dy.abs().max().item()
        shared = torch.randn(4, 1, 48, device=dev).requires_grad_()
        y = torch.ops.mi355.rope(shared.expand(4, 3, 48), pos.to(dev), f.to(dev), inter, False, scale)
        got, = torch.autograd.grad(y, shared, dy.to(dev))
        torch.testing.assert_close(got.double().cpu(), want.sum(1, keepdim=True), rtol=0, atol=3 * bound.max().item() + 2.0**-20)
        # the gradient of the gradient is the forward rotation
        g = dy.to(dev).requires_grad_()
        back = torch.ops.mi355.rope(g, pos.to(dev), f.to(dev), inter, True, scale)
        twice, = torch.autograd.grad(back, g, x.to(dev))
        _inside(twice, *serving.rope_ref(x, pos, f, inter, scale=scale))


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,hq,hkv,R,page", [(1, 4, 4, 128, 16), (19, 8, 2, 64, 32), (70, 32, 8, 128, 16), (5, 3, 1, 96, 256), (6, 2, 2, 6, 16)])
def test_rope_kv_append(dev, T, hq, hkv, R, page, dtype, inter):
    """Rows that no slot names keep what they held, dropped tokens go nowhere, values move bit for bit."""
    from oracle import serving

    announce(f"rope_kv_append T={T} hq={hq} hkv={hkv} R={R} page={page} {dtype} interleaved={inter}")
    P = -(-T // page) + 2
    qkv = torch.randn(T, hq + 2 * hkv, 128).to(dtype)
    kc, vc = (torch.randn(P, page, hkv, 128).to(dtype) for _ in range(2))
    pos = torch.randint(0, 100000, (T,), dtype=torch.int32)
    slots = torch.randperm(P * page)[:T]
    if T > 4:
        slots[1], slots[3], slots[4] = -1, P * page, -(2**40)
    f, scale = _freq(R, scaling="yarn", factor=4.0)
    q, k, v = qkv.to(dev).split([hq, hkv, hkv], 1)
    kd, vd = kc.to(dev), vc.to(dev)
    got = torch.ops.mi355.rope_kv_append(q, k, v, pos.to(dev), f.to(dev), kd, vd, slots.to(dev), inter, scale)
    qw, kw = (serving.rope_ref(x, pos, f, inter, scale=scale) for x in (qkv[:, :hq], qkv[:, hq:hq + hkv]))
    _inside(got, *qw)
    want_k, bound_k, want_v = kc.double(), torch.zeros(kc.shape, dtype=torch.float64), vc.clone()
    for t in range(T):
        s = int(slots[t])
        if 0 <= s < P * page:
            want_k.view(-1, hkv, 128)[s], bound_k.view(-1, hkv, 128)[s] = kw[0][t], kw[1][t]
            want_v.view(-1, hkv, 128)[s] = qkv[t, hq + hkv:]
    _inside(kd, want_k, bound_k)
    assert torch.equal(vd.cpu(), want_v)
    # the same as the rotation alone, bit for bit
    assert torch.equal(got, torch.ops.mi355.rope(q, pos.to(dev), f.to(dev), inter, False, scale))


def test_append_rows_off_the_16_byte_borders(dev):
    from oracle import serving

    announce("rope_kv_append off the borders")
    T, hq, hkv = 7, 4, 2
    flat = torch.randn(T, 8 * 128 + 5).half()
    part = lambda t, a, h: t[:, 3 + a * 128: 3 + (a + h) * 128].unflatten(1, (h, 128))
    f, _ = _freq(128)
    pos, slots = torch.arange(T, dtype=torch.int32), torch.arange(T)
    kc, vc = (torch.zeros(1, 16, hkv, 128).half().to(dev) for _ in range(2))
    fd = flat.to(dev)
    got = torch.ops.mi355.rope_kv_append(part(fd, 0, hq), part(fd, 4, hkv), part(fd, 6, hkv), pos.to(dev), f.to(dev), kc, vc, slots.to(dev), True, 1.0)
    _inside(got, *serving.rope_ref(part(flat, 0, hq), pos, f, True))
    _inside(kc[0, :T], *serving.rope_ref(part(flat, 4, hkv), pos, f, True))
    assert torch.equal(vc[0, :T].cpu(), part(flat, 6, hkv))


def test_rope_in_place_on_a_stream_and_captured(dev):
    from iree_turbine_amd import launch
    from oracle import serving

    announce("rope in place, other stream, captured")
    f, _ = _freq(128)
    x = torch.randn(40, 8, 128).bfloat16()
    pos = torch.arange(40, dtype=torch.int32) * 700
    want, bound = serving.rope_ref(x, pos, f, False)
    xd, pd, fd = x.to(dev), pos.to(dev), f.to(dev)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        y = xd.clone()
        launch.rope_out(y, pd, fd, y, False, False, 1.0)
    torch.cuda.current_stream(dev).wait_stream(side)
    _inside(y, want, bound)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        z = torch.ops.mi355.rope(xd, pd, fd, False, False, 1.0)
    for k in range(3):
        xd.copy_(x.to(dev) * (2.0 ** k))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(z, torch.ops.mi355.rope(xd, pd, fd, False, False, 1.0))


def test_lazily_negated_operands_and_gradients(dev):
    """Tensors that carry torch's negation as a flag (the imaginary part of a conjugate) are read with their sign, and so are
    the gradients that come back through one; a gradient of zeros that has no memory gives zeros."""
    announce("rope of lazily negated tensors")
    z = torch.randn(5, 2, 64, dtype=torch.complex64, device=dev)
    x = z.conj().imag
    assert x.is_neg()
    pos, f = torch.arange(5, dtype=torch.int32, device=dev), _freq(64, device=dev)[0].float()
    call = lambda t, g=f: torch.ops.mi355.rope(t, pos, g, False, False, 1.0)
    want = call(x.resolve_neg().clone())
    assert torch.equal(call(x), want)
    neg_f = torch.complex(f, -f).conj().imag  # f again, negated twice
    assert neg_f.is_neg() and torch.equal(call(x, neg_f), call(x.resolve_neg().clone(), neg_f.resolve_neg().clone()))
    leaf = torch.randn(5, 2, 64, device=dev, requires_grad=True)
    y = call(leaf)
    g = torch.randn(5, 2, 64, dtype=torch.complex64, device=dev).conj().imag
    assert torch.equal(torch.autograd.grad(y, leaf, g, retain_graph=True)[0], torch.autograd.grad(y, leaf, g.resolve_neg().clone(), retain_graph=True)[0])
    zero = torch._efficientzerotensor((5, 2, 64), device=dev)
    assert torch.equal(torch.autograd.grad(y, leaf, zero)[0], torch.zeros_like(leaf))
    # x itself required to have a gradient while lazily negated
    w = z.clone().requires_grad_()
    v = w.conj().imag
    torch.testing.assert_close(torch.autograd.grad(call(v), w, want)[0], torch.autograd.grad(call(-w.imag), w, want)[0], rtol=0, atol=0)


def test_rows_past_32_bit_offsets(dev):
    """Rows a mebi-element apart, read and written in place; a cache whose last slots lie more than 2^32 elements in."""
    from oracle import serving

    announce("rope far rows")
    T, pitch = 2300, 1 << 20
    far = torch.empty(T * pitch, dtype=torch.float16, device=dev).view(T, pitch)[:, 64:64 + 256].view(T, 2, 128)
    x = torch.randn(T, 2, 128).half()
    far.copy_(x)
    pos, f = torch.arange(T, dtype=torch.int32), _freq(128)[0]
    want, bound = serving.rope_ref(x, pos, f, False)
    _inside(torch.ops.mi355.rope(far, pos.to(dev), f.to(dev), False, False, 1.0), want, bound)
    from iree_turbine_amd import launch

    launch.rope_out(far, pos.to(dev), f.to(dev), far, False, False, 1.0)
    _inside(far, want, bound)
    del far
    P = (1 << 32) // (256 * 8 * 128) + 2
    kc, vc = (torch.empty(P, 256, 8, 128, dtype=torch.float16, device=dev) for _ in range(2))
    last = P * 256
    slots = torch.tensor([last - 1, 0, last, -(2**40), last - 300], device=dev)
    q, k, v = (torch.randn(5, h, 128).half() for h in (8, 8, 8))
    p5 = pos[:5] * 100
    torch.ops.mi355.rope_kv_append(q.to(dev), k.to(dev), v.to(dev), p5.to(dev), f.to(dev), kc, vc, slots, False, 1.0)
    want, bound = serving.rope_ref(k, p5, f, False)
    flat_k, flat_v = kc.view(-1, 8, 128), vc.view(-1, 8, 128)
    for row, slot in ((0, last - 1), (1, 0), (4, last - 300)):
        _inside(flat_k[slot], want[row], bound[row])
        assert torch.equal(flat_v[slot].cpu(), v[row])


def test_gradient_with_lazily_negated_frequencies(dev):
    """Frequencies that carry torch's negation as a flag turn the gradient the way that their values say."""
    announce("rope gradient, lazily negated frequencies")
    pos, f = torch.arange(5, dtype=torch.int32, device=dev) * 3, _freq(64, device=dev)[0]
    lazy = torch._neg_view(f)
    assert lazy.is_neg() and lazy.is_contiguous()
    x, g = (torch.randn(5, 2, 64, device=dev) for _ in range(2))
    leaf = x.clone().requires_grad_()
    y, plain = (torch.ops.mi355.rope(leaf, pos, freq, False, False, 1.0) for freq in (lazy, -f))
    assert torch.equal(y, plain)
    want, = torch.autograd.grad(plain, leaf, g)
    assert torch.equal(torch.autograd.grad(y, leaf, g)[0], want)
    assert not torch.equal(want, torch.ops.mi355.rope(g, pos, f, False, True, 1.0))


def test_backward_captured_beside_an_eager_graph_of_the_same_leaf(dev):
    """Refused while an eager graph of the leaf is alive: its accumulator works on the default stream, which cannot wait for a
    captured one.  Without it the captured pass replays what the eager one gives."""
    announce("rope backward captured, eager graph alive")
    pos, f = torch.arange(9, dtype=torch.int32, device=dev) * 31, _freq(64, device=dev)[0]
    leaf, g = torch.randn(9, 2, 64, device=dev, requires_grad=True), torch.randn(9, 2, 64, device=dev)
    call = lambda: torch.ops.mi355.rope(leaf, pos, f, False, False, 1.0)
    alive = call()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="under capture while a graph of the same leaf"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.autograd.grad(call(), leaf, g)
    torch.cuda.synchronize()
    want, = torch.autograd.grad(alive, leaf, g)
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, = torch.autograd.grad(call(), leaf, g)
    for k in range(3):
        g.copy_(torch.randn(9, 2, 64))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, torch.ops.mi355.rope(g, pos, f, False, True, 1.0))
        assert torch.equal(got, torch.autograd.grad(call(), leaf, g)[0])
    assert want.shape == got.shape
