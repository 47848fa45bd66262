"""CPU-side tests of the packed serving step's operators: Meta kernels, refusals at the op and at the C entry, rotary
frequencies, and the oracles against independent statements.  Nothing is launched."""

import ctypes
import math

import pytest
import torch

import iree_turbine_amd as ita
from iree_turbine_amd import _lib, op_reg
from oracle import serving

OPS = torch.ops.mi355
I32, I64, F32, F64 = torch.int32, torch.int64, torch.float32, torch.float64


def m(*size, dt=torch.float16):
    return torch.empty(*size, dtype=dt, device="meta")


def strides(*v):
    return (ctypes.c_int64 * len(v))(*v)


def varlen_args(**change):
    a = dict(q=m(9, 4, 128), k=m(11, 2, 128), v=m(11, 2, 128), cq=m(4, dt=I32), ck=m(4, dt=I32), causal=True, scale=0.0)
    a.update(change)
    return a


def tree_args(**change):
    a = dict(q=m(2, 5, 8, 128), kc=m(6, 16, 2, 128), vc=m(6, 16, 2, 128), bt=m(2, 3, dt=I32), sl=m(2, dt=I32), par=m(2, 5, dt=I32), scale=0.0, splits=0)
    a.update(change)
    return a


def verify_args(**change):
    a = dict(p=m(2, 5, 40, dt=F32), q=m(2, 5, 40, dt=F32), tok=m(2, 5, dt=I32), par=m(2, 5, dt=I32), u=m(2, 5, dt=F32))
    a.update(change)
    return a


def layout_args(**change):
    a = dict(bt=m(2, 3, dt=I32), ctx=m(2, dt=I32), new=m(2, dt=I32), free=m(7, dt=I32), page=16, rows=20)
    a.update(change)
    return a


def rope_args(**change):
    a = dict(x=m(5, 3, 96), pos=m(5, dt=I32), f=m(32, dt=F64), inter=False, inv=False, scale=1.0)
    a.update(change)
    return a


def append_args(**change):
    a = dict(q=m(5, 8, 128), k=m(5, 2, 128), v=m(5, 2, 128), pos=m(5, dt=I32), f=m(64, dt=F64), kc=m(6, 16, 2, 128), vc=m(6, 16, 2, 128),
             slots=m(5, dt=I64), inter=True, scale=1.0)
    a.update(change)
    return a


def test_meta_kernels_give_the_results_shapes():
    assert OPS.flash_attn_varlen_fwd(*varlen_args().values()).shape == (9, 4, 128)
    assert OPS.paged_tree_attn(*tree_args().values()).shape == (2, 5, 8, 128)
    assert [tuple(t.shape) for t in OPS.verify_draft(*verify_args().values())] == [(2, 5), (2,), (2,)]
    assert [tuple(t.shape) for t in OPS.verify_draft(*verify_args(q=None).values())] == [(2, 5), (2,), (2,)]
    got = OPS.paged_batch_layout(*layout_args().values())
    assert [(tuple(t.shape), t.dtype) for t in got] == [((2,), I32), ((3,), I32), ((20,), I32), ((20,), I32), ((20,), I64), ((1,), I32)]
    assert OPS.rope_kv_append(*append_args().values()).shape == (5, 8, 128)
    x = m(5, 3, 96, dt=torch.bfloat16).requires_grad_()
    y = OPS.rope(*rope_args(x=x).values())
    assert y.dtype == torch.bfloat16 and torch.autograd.grad(y.sum(), x)[0].shape == x.shape


@pytest.mark.parametrize("change,text", [
    (dict(q=m(9, 4, 64), k=m(11, 2, 64), v=m(11, 2, 64)), "head dim"),
    (dict(k=m(11, 3, 128), v=m(11, 3, 128)), "query heads"),
    (dict(v=m(10, 2, 128)), "shapes differ"),
    (dict(q=m(9, 4, 128, dt=torch.bfloat16)), "all be float16 or all be bfloat16"),
    (dict(cq=m(4, dt=I64)), "cu_seqlens_q"),
    (dict(ck=m(5, dt=I32)), "cu_seqlens_k"),
    (dict(cq=m(1, dt=I32), ck=m(1, dt=I32)), "cu_seqlens_q"),
    (dict(q=m(0, 4, 128)), "rows"),
])
def test_varlen_refusals(change, text):
    with pytest.raises(ValueError, match=text):
        OPS.flash_attn_varlen_fwd(*varlen_args(**change).values())


@pytest.mark.parametrize("change,text", [
    (dict(q=m(2, 65, 8, 128), par=m(2, 65, dt=I32)), "nodes per sequence"),
    (dict(q=m(2, 5, 7, 128)), "q heads over"),
    (dict(q=m(2, 5, 8, 64)), "head dim"),
    (dict(kc=m(6, 8, 2, 128), vc=m(6, 8, 2, 128)), "page size"),
    (dict(par=m(2, 4, dt=I32)), "parents"),
    (dict(par=m(2, 5, dt=I64)), "parents"),
    (dict(sl=m(3, dt=I32)), "rows must equal"),
    (dict(q=m(2, 5, 258, 128)), "up to 128"),
    (dict(vc=m(6, 16, 2, 128, dt=torch.bfloat16)), "all be float16 or all be bfloat16"),
])
def test_tree_refusals(change, text):
    with pytest.raises(ValueError, match=text):
        OPS.paged_tree_attn(*tree_args(**change).values())


@pytest.mark.parametrize("change,text", [
    (dict(p=m(2, 5, 40)), "target_probs"),
    (dict(q=m(2, 5, 41, dt=F32)), "draft_probs"),
    (dict(tok=m(2, 4, dt=I32)), "tokens"),
    (dict(tok=m(2, 5, dt=I64)), "tokens"),
    (dict(u=m(2, 5, dt=F64)), "uniforms"),
    (dict(p=m(2, 65, 40, dt=F32), q=None, tok=m(2, 65, dt=I32), par=m(2, 65, dt=I32), u=m(2, 65, dt=F32)), "65 nodes"),
])
def test_verify_refusals(change, text):
    with pytest.raises(ValueError, match=text):
        OPS.verify_draft(*verify_args(**change).values())


@pytest.mark.parametrize("change,text", [
    (dict(page=8), "page size"),
    (dict(rows=0), "num_tokens"),
    (dict(new=m(3, dt=I32)), "new_lens"),
    (dict(ctx=m(2, dt=I64)), "context_lens"),
    (dict(free=m(7, dt=I64)), "free_pages"),
    (dict(bt=m(2, 6, dt=I32)[:, ::2]), "contiguous"),
])
def test_layout_refusals(change, text):
    with pytest.raises(ValueError, match=text):
        OPS.paged_batch_layout(*layout_args(**change).values())


@pytest.mark.parametrize("change,text", [
    (dict(f=m(49, dt=F64)), "rotary elements"),
    (dict(f=m(0, dt=F64)), "rotary elements"),
    (dict(f=m(32)), "inv_freq"),
    (dict(pos=m(5, dt=I64)), "positions"),
    (dict(pos=m(4, dt=I32)), "positions"),
    (dict(x=m(5, 3, 96, dt=F64)), "x must be"),
    (dict(x=m(5, 96)), "x must be"),
])
def test_rope_refusals(change, text):
    with pytest.raises(ValueError, match=text):
        OPS.rope(*rope_args(**change).values())


@pytest.mark.parametrize("change,text", [
    (dict(k=m(5, 3, 128), v=m(5, 3, 128)), "number of kv heads"),
    (dict(k=m(4, 2, 128), v=m(4, 2, 128)), "unequal tokens"),
    (dict(slots=m(5, dt=I32)), "slots"),
    (dict(kc=m(6, 16, 4, 128)[:, :, ::2], vc=m(6, 16, 4, 128)[:, :, ::2]), "contiguous"),
    (dict(f=m(65, dt=F64)), "rotary elements"),
    (dict(v=m(5, 2, 128, dt=torch.bfloat16)), "all be float16 or all be bfloat16"),
])
def test_append_refusals(change, text):
    with pytest.raises(ValueError, match=text):
        OPS.rope_kv_append(*append_args(**change).values())


def test_cpu_tensors_are_refused():
    with pytest.raises(NotImplementedError):
        OPS.rope(torch.zeros(2, 2, 64), torch.zeros(2, dtype=I32), torch.zeros(32, dtype=F64), False, False, 1.0)


def test_c_entries_refuse_bad_arguments_without_a_gpu():
    lib = _lib.load()
    st = strides(512, 128)
    va = lambda **c: lib.mi355_flash_attn_varlen_fwd(*{**dict(q=16, k=16, v=16, o=16, cq=16, ck=16, S=2, tq=9, tk=9, H=4, Hkv=2, D=128, qs=st, ks=st, vs=st, os=st,
                                                              scale=1.0, causal=1, zero=0, dtype=1, ws=None, wb=0, stream=None), **c}.values())
    assert va(q=None) == -1 and va(D=64) == -2 and va(o=24) == -3 and va(dtype=0) == -4 and va(S=0) == -2 and va(Hkv=3) == -2
    assert va(qs=strides(513, 128)) == -3 and va(ks=strides(64, 128)) == -2 and va(os=strides(512, 0)) == -2 and va(scale=math.nan) == -2
    assert va(tk=1 << 25) == -2
    cut = lib.mi355_flash_attn_varlen_workspace_bytes
    assert cut(4, 80, 6000, 16, 1, 1) > 0 and cut(4, 80, 200, 16, 1, 1) == 0 and cut(4, 8000, 8000, 32, 8, 1) == 0 and cut(65, 80, 60000, 16, 1, 1) == 0
    assert cut(0, 80, 6000, 16, 1, 1) == 0 and cut(4, 80, 6000, 16, 3, 1) == 0
    assert va(S=4, tq=80, tk=6000, H=16, Hkv=1, ws=24, wb=cut(4, 80, 6000, 16, 1, 1), qs=strides(2048, 128)) == -3
    ta = lambda **c: lib.mi355_paged_tree_attn(*{**dict(q=16, k=16, v=16, bt=16, sl=16, par=16, out=16, pa=None, pm=None, S=2, N=5, hq=8, hkv=2, D=128, page=16, mp=4,
                                                        P=9, splits=1, scale=1.0, dtype=1, stream=None), **c}.values())
    assert ta(par=None) == -1 and ta(N=65) == -2 and ta(splits=2) == -5 and ta(page=48) == -2 and ta(hq=9) == -2 and ta(dtype=0) == -4
    assert ta(k=24) == -3 and ta(splits=1025) == -2 and ta(hq=258) == -2 and ta(scale=0.0) == -2
    need = lib.mi355_verify_draft_workspace_bytes
    assert need(3, 5, 32000) > 0 and need(0, 5, 100) == 0 and need(3, 65, 100) == 0
    ve = lambda **c: lib.mi355_verify_draft(*{**dict(p=16, q=None, tok=16, par=16, u=16, path=16, n=16, nxt=16, S=3, N=5, V=32000, ws=16, wb=need(3, 5, 32000), stream=None), **c}.values())
    assert ve(u=None) == -1 and ve(N=65) == -2 and ve(ws=None) == -5 and ve(wb=need(3, 5, 32000) - 1) == -5 and ve(ws=24) == -3
    la = lambda **c: lib.mi355_paged_batch_layout(*{**dict(bt=16, ctx=16, new=16, free=16, F=3, S=2, W=4, page=16, T=9, sl=16, cu=16, pos=16, ids=16, slots=16, need=16,
                                                           stream=None), **c}.values())
    assert la(cu=None) == -1 and la(page=48) == -2 and la(T=0) == -2 and la(S=1 << 17) == -2 and la(free=None) == -1
    ro = lambda **c: lib.mi355_rope(*{**dict(x=16, out=16, pos=16, f=16, f64=1, T=2, H=2, D=64, R=64, xs=st, os=st, inter=0, inv=0, scale=1.0, dtype=1, stream=None), **c}.values())
    assert ro(x=None) == -1 and ro(R=63) == -2 and ro(R=66) == -2 and ro(dtype=7) == -4 and ro(xs=strides(-8, 128)) == -2 and ro(scale=math.inf) == -2
    ap = lambda **c: lib.mi355_rope_kv_append(*{**dict(q=16, k=16, v=16, qo=16, kc=16, vc=16, pos=16, f=16, f64=1, slots=16, T=2, hq=4, hkv=2, D=128, R=128, n=64, qs=st, ks=st,
                                                       vs=st, inter=0, scale=1.0, dtype=1, stream=None), **c}.values())
    assert ap(slots=None) == -1 and ap(D=64) == -2 and ap(R=130) == -2 and ap(dtype=0) == -4 and ap(n=0) == -2


def test_rope_frequencies():
    f, scale = ita.rope_inv_freq(128)
    assert f.dtype == F64 and scale == 1.0
    torch.testing.assert_close(f, 10000.0 ** (-torch.arange(64, dtype=F64) / 64), rtol=1e-14, atol=0)
    lin, _ = ita.rope_inv_freq(128, scaling="linear", factor=4.0)
    torch.testing.assert_close(lin, f / 4, rtol=1e-15, atol=0)
    ntk, _ = ita.rope_inv_freq(128, scaling="ntk", factor=4.0)
    assert ntk[0] == 1.0 and math.isclose(float(ntk[-1]), float(f[-1]) / 4, rel_tol=1e-12)
    yarn, scale = ita.rope_inv_freq(128, scaling="yarn", factor=16.0, trained_len=4096)
    turns = f * 4096 / (2 * math.pi)
    assert torch.equal(yarn[turns >= 32], f[turns >= 32])
    torch.testing.assert_close(yarn[turns <= 1], f[turns <= 1] / 16, rtol=1e-15, atol=0)
    assert math.isclose(scale, 0.1 * math.log(16) + 1) and bool((yarn.diff() < 0).all())
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=64, scaling="none such"), dict(rotary_dim=64, factor=0.5)):
        with pytest.raises(ValueError):
            ita.rope_inv_freq(**bad)


def test_oracle_rope_is_a_rotation_and_its_gradient():
    x = torch.randn(4, 3, 20, dtype=F64, requires_grad=True)
    pos = torch.tensor([0, 1, 77, 100000], dtype=I32)
    f = ita.rope_inv_freq(12)[0]
    for inter in (False, True):
        y, _ = serving.rope_ref(x, pos, f, inter, scale=1.25)
        assert torch.equal(y[0, :, 12:], x[0, :, 12:])
        torch.testing.assert_close(y[..., :12].norm(dim=-1), 1.25 * x[..., :12].norm(dim=-1))
        g = torch.randn_like(y)
        want, _ = serving.rope_ref(g, pos, f, inter, inverse=True, scale=1.25)
        torch.testing.assert_close(torch.autograd.grad(y, x, g)[0], want)
        # pair 2 of head 1 at position 77, written out
        i, j = (4, 5) if inter else (2, 8)
        c, s = math.cos(77 * float(f[2])), math.sin(77 * float(f[2]))
        a, b = (x.detach()[2, 1, n].item() for n in (i, j))
        assert math.isclose(y.detach()[2, 1, i].item(), 1.25 * (a * c - b * s)) and math.isclose(y.detach()[2, 1, j].item(), 1.25 * (a * s + b * c))


def test_oracle_attention_against_torch():
    q, k, v = (torch.randn(n, h, 128).half() for n, h in ((7, 4), (9, 2), (9, 2)))
    vis = torch.ones(7, 9, dtype=torch.bool).tril(2)
    out, bound = serving.attention_ref(q, k, v, vis)
    want = torch.nn.functional.scaled_dot_product_attention(q.double().transpose(0, 1), k.double().repeat_interleave(2, 1).transpose(0, 1),
                                                            v.double().repeat_interleave(2, 1).transpose(0, 1), attn_mask=vis).transpose(0, 1)
    torch.testing.assert_close(out, want)
    assert float(bound.max()) < 0.02 and float(bound.min()) > 0


def test_oracle_verification_keeps_the_target_distribution():
    """Chains and trees of independent siblings leave the first token's distribution the target's, whatever the draft's is."""
    torch.manual_seed(3)
    S, V = 20000, 4
    p = torch.softmax(torch.randn(V), 0)
    q = torch.softmax(torch.randn(V), 0)
    for parents, draft in (([-1, 0], True), ([-1, 0, 0, 0], True), ([-1, 0, 0], False)):
        N = len(parents)
        target, dr = p.expand(S, N, V), q.expand(S, N, V) if draft else None
        tokens = torch.multinomial(q, S * N, replacement=True).view(S, N).int() if draft else torch.tensor([0, 2, 1][:N]).int().expand(S, N)
        path, count, last = serving.verify_ref(target[:4000], dr[:4000] if draft else None, tokens[:4000], torch.tensor(parents).int().expand(4000, N), torch.rand(4000, N))
        first = torch.where(count > 0, tokens[:4000].gather(1, path[:, :1].clamp(min=0).long())[:, 0], last)
        share = torch.bincount(first.long(), minlength=V).double() / 4000
        assert float((share - p).abs().max()) < 5 * math.sqrt(0.25 / 4000)


def test_rope_gradient_formula_is_traced_and_differentiable_twice():
    """On meta tensors and through make_fx the gradient is the op with `inverse` turned."""
    from torch.fx.experimental.proxy_tensor import make_fx

    x = m(5, 3, 96, dt=F32).requires_grad_()
    pos, f = m(5, dt=I32), m(32, dt=F64)
    y = OPS.rope(x, pos, f, False, False, 1.0)
    g = m(5, 3, 96, dt=F32).requires_grad_()
    first, = torch.autograd.grad(y, x, g, create_graph=True)
    second, = torch.autograd.grad(first, g, m(5, 3, 96, dt=F32))
    assert first.shape == second.shape == x.shape
    with torch.no_grad():
        assert not OPS.rope(x, pos, f, False, False, 1.0).requires_grad

    def step(x, pos, f, dy):
        x = x.detach().requires_grad_()
        y = OPS.rope(x, pos, f, True, False, 2.0)
        return torch.autograd.grad(y, x, dy)[0]

    calls = [n for n in make_fx(step)(m(5, 3, 96, dt=F32), pos, f, m(5, 3, 96, dt=F32)).graph.nodes if "rope" in str(n.target)]
    assert [n.args[4] for n in calls] == [False, True]


def test_native_host_side_leaves_other_calls_alone():
    host = _lib.host_ops()
    names = [n for n in dir(host) if not n.startswith("_") and n != "bind"]
    assert sorted(names) == sorted(["rope_grad"] + [op.host for op in op_reg.ALL_CUSTOM_OP_REGS.values() if op.host])
    cpu = (torch.zeros(2, 2, 64), torch.zeros(2, dtype=I32), torch.zeros(32, dtype=F64), False, False, 1.0)
    for name in names:
        f = getattr(host, name)
        assert f() is None and f(*cpu) is None and f(*([3] * 6)) is None and f(*([None] * 10)) is None
    with pytest.raises(TypeError):
        host.bind()
    with pytest.raises(ValueError):
        host.bind(*([0] * 10))
    assert _lib.host_ops() is host


def test_missing_native_host_side_is_an_error(monkeypatch, tmp_path):
    monkeypatch.setattr(_lib, "_host", None)
    monkeypatch.setattr(_lib, "HOST_PATH", tmp_path / "mi355_host_ops.so")
    with pytest.raises(_lib.KernelLibraryError, match="build it"):
        _lib.host_ops()


@pytest.mark.parametrize("m", [65, 130, 257, 515, 700, 900, 1033, 1500, 1900, 2300, 2600, 4000])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_oracle_attention_bound_sees_a_lost_tile(dtype, m):
    """At the lengths that the attention tests use, a result without one tile of 64 keys, one 32-key step or one of 16 chunks
    is outside the bound, wherever it lies."""
    q, k, v = (torch.randn(n, h, 128).to(dtype) for n, h in ((4, 4), (m, 2), (m, 2)))
    vis = torch.ones(4, m, dtype=torch.bool)
    out, bound = serving.attention_ref(q, k, v, vis)
    for width in {32, 64, -(-m // 1024) * 64}:
        for at in {0, (m - width) // 2, m - width}:
            lost = vis.clone()
            lost[:, at : at + width] = False
            assert float(((serving.attention_ref(q, k, v, lost)[0] - out).abs() / bound).max()) > 1, (width, at)
    assert float((out.abs() / bound).median()) > 1  # nor would zeros pass


def test_oracle_attention_bound_holds_for_16_bit_weights():
    """The bound's own model, step by step: weights against a maximum that lags by up to 2^8, rounded to 16 bits, summed either way,
    scaled down later.  Wide scores leave most fp16 weights below 2^-14."""
    for dtype in (torch.float16, torch.bfloat16):
        for spread in (1.0, 3.0, 12.0):
            q, k, v = (torch.randn(n, 1, 128) for n in (16, 500, 500))
            q, k, v = (q * spread).to(dtype), k.to(dtype), v.to(dtype)
            out, bound = serving.attention_ref(q, k, v, torch.ones(16, 500, dtype=torch.bool))
            s = (q[:, 0].float() @ k[:, 0].float().t()) * 128**-0.5
            for lag in (0.0, 5.5):  # in nats
                w = torch.exp(s - s.amax(-1, keepdim=True) + lag)
                r = w.to(dtype).double()
                for total in (w.double().sum(-1, keepdim=True), r.sum(-1, keepdim=True)):
                    got = ((r @ v[:, 0].double()) / total).to(dtype).double()
                    assert bool(((got - out[:, 0]).abs() <= bound[:, 0]).all())


@pytest.fixture
def rope_on_cpu():
    """The oracle's rotation as the op's CPU kernel, below the op's own derivative formulas."""
    with torch.library._scoped_library("mi355", "IMPL") as lib:
        lib.impl("rope", lambda x, *a: serving.rope_ref(x, *a)[0].to(x.dtype), "CPU")
        yield


def _rotation():
    pos, f = torch.tensor([0, 5, 1000], dtype=I32), ita.rope_inv_freq(12)[0]
    x, t = (torch.randn(3, 2, 16, dtype=F64) for _ in range(2))
    return (lambda v: OPS.rope(v, pos, f, True, False, 1.5)), (lambda v: OPS.rope(v, pos, f, True, True, 1.5)), x, t


def test_rope_forward_mode(rope_on_cpu):
    """The tangent is the rotation of the operand's: of tensors with and without requires_grad, without grad mode, and through
    the gradient."""
    import torch.autograd.forward_ad as fw

    call, back, x, t = _rotation()
    with fw.dual_level():
        for leaf in (x, x.clone().requires_grad_()):
            y = fw.unpack_dual(call(fw.make_dual(leaf, t)))
            assert torch.equal(y.tangent, call(t)) and torch.equal(y.primal, call(x))
        with torch.no_grad():
            assert torch.equal(fw.unpack_dual(call(fw.make_dual(x, t))).tangent, call(t))
        assert fw.unpack_dual(call(x)).tangent is None
        # the gradient's tangent, by one node and by the node of the node
        leaf = x.clone().requires_grad_()
        for graph in (False, True):
            dx, = torch.autograd.grad(call(leaf), leaf, fw.make_dual(x, t), create_graph=graph)
            assert torch.equal(fw.unpack_dual(dx).tangent, back(t)) and torch.equal(fw.unpack_dual(dx).primal, back(x))
    assert torch.autograd.gradcheck(call, (x.clone().requires_grad_(),), check_forward_ad=True, check_batched_grad=True)
    assert torch.autograd.gradgradcheck(call, (x.clone().requires_grad_(),))


@pytest.mark.filterwarnings("ignore:There is a performance drop")
def test_rope_under_torch_func(rope_on_cpu):
    call, back, x, t = _rotation()
    torch.testing.assert_close(torch.func.grad(lambda v: (call(v) * t).sum())(x), back(t))
    y, dy = torch.func.jvp(call, (x,), (t,))
    assert torch.equal(y, call(x)) and torch.equal(dy, call(t))
    y, pull = torch.func.vjp(call, x)
    assert torch.equal(y, call(x)) and torch.equal(pull(t)[0], back(t))
    many = torch.stack([x, t, x - t])
    want = torch.stack([call(v) for v in many])
    assert torch.equal(torch.func.vmap(call)(many), want)
    torch.testing.assert_close(torch.func.vmap(torch.func.grad(lambda v: (call(v) * t).sum()))(many), back(t).expand(3, 3, 2, 16))
    assert torch.equal(torch.func.vmap(torch.func.jvp, in_dims=(None, None, 0))(call, (x,), (many,))[1], want)
    fwd, rev = torch.func.jacfwd(call)(x), torch.func.jacrev(call)(x)
    torch.testing.assert_close(fwd, rev)
    torch.testing.assert_close(torch.einsum("abcdef,def->abc", rev, t), call(t))
    h = torch.func.hessian(lambda v: (call(v) ** 2).sum() / 2)(x)  # R^T R = 1.5^2 on the turned elements
    torch.testing.assert_close(torch.einsum("abcdef,def->abc", h, t), torch.cat([t[..., :12] * 2.25, t[..., 12:]], -1))
    leaf = x.clone().requires_grad_()
    got, = torch.autograd.grad(call(leaf), leaf, many, is_grads_batched=True)
    assert torch.equal(got, torch.stack([back(v) for v in many]))


def test_batch_layout_refuses_shared_memory():
    """Lengths are read by all workgroups while the first writes its results: none of those lies in an operand's memory.  Addresses
    only; every one of these calls is refused before a launch."""
    lib = _lib.load()
    S, W, T, F = 3, 4, 9, 5
    size = dict(bt=S * W * 4, sl=S * 4, cu=(S + 1) * 4, pos=T * 4, ids=T * 4, slots=T * 8, need=4, ctx=S * 4, new=S * 4, free=F * 4)
    base = {name: 4096 * (i + 1) for i, name in enumerate(size)}

    def call(**at):
        a = {**base, **at}
        return lib.mi355_paged_batch_layout(a["bt"], a["ctx"], a["new"], a["free"], F, S, W, 16, T, a["sl"], a["cu"], a["pos"], a["ids"], a["slots"], a["need"], None)

    written = ["bt", "sl", "cu", "pos", "ids", "slots", "need"]
    for one in written:
        for other in size:
            if one != other:
                for at in (base[other], base[other] + size[other] - 4, base[other] - size[one] + 4):
                    assert call(**{one: at}) == -6, (one, other)
    assert b"share memory" in lib.mi355_last_error()


def test_host_side_of_another_torch_is_an_error(monkeypatch, tmp_path):
    """A library that does not load (other symbols than this torch's, or no library at all) says what to do."""
    (tmp_path / "mi355_host_ops.so").write_bytes(b"not a library")
    monkeypatch.setattr(_lib, "_host", None)
    monkeypatch.setattr(_lib, "HOST_PATH", tmp_path / "mi355_host_ops.so")
    with pytest.raises(_lib.KernelLibraryError, match="build it again"):
        _lib.host_ops()
