"""GPU: the native host side of the serving operators gives what the way through Python gives, leaves every other call to it,
and its gradient node behaves as one."""

import pytest
import torch

import iree_turbine_amd as ita
from conftest import announce
from iree_turbine_amd import _lib, op_reg

pytestmark = pytest.mark.gpu
OPS = torch.ops.mi355


# operands that may have an entry less: frequencies, free pages, the columns of a block table
FEWER_IS_FINE = {("rope", 2), ("rope_kv_append", 4), ("paged_batch_layout", 0), ("paged_batch_layout", 3), ("paged_tree_attn", 3)}


def _calls(dev):
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g).half().to(dev)
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)
    f = ita.rope_inv_freq(128, device=dev)[0]
    kc, vc = r(9, 16, 2, 128), r(9, 16, 2, 128)
    table = torch.tensor([[3, 1, 7], [0, 2, 8]], dtype=torch.int32, device=dev)
    par = i(-1, 0, 0, -1, 0, 1).view(2, 3)
    p = torch.softmax(torch.randn(2, 3, 50, generator=g), -1).to(dev)
    return {
        "rope": (r(5, 4, 128), i(0, 3, 9, 1, 1), f, False, True, 1.5),
        "rope_kv_append": (r(3, 4, 128), r(3, 2, 128), r(3, 2, 128), i(5, 6, 7), f, kc, vc, torch.tensor([4, -1, 100], device=dev), True, 1.0),
        "paged_batch_layout": (table.clone(), i(20, 3), i(9, 1), i(5, 4, 6), 16, 12),
        "flash_attn_varlen_fwd": (r(12, 4, 128), r(12, 2, 128), r(12, 2, 128), i(0, 5, 12), i(0, 5, 12), True, 0.0),
        "paged_tree_attn": (r(2, 3, 4, 128), kc, vc, table, i(40, 33), par, 0.0, 0),
        "verify_draft": (p, p.flip(0).contiguous(), i(1, 2, 3, 4, 5, 6).view(2, 3), par, torch.rand(2, 3, generator=g).to(dev)),
    }


def _same(a, b):
    a, b = ([t] if isinstance(t, torch.Tensor) else list(t) for t in (a, b))
    assert len(a) == len(b) and all(x.dtype == y.dtype and x.stride() == y.stride() and torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("name", ["rope", "rope_kv_append", "paged_batch_layout", "flash_attn_varlen_fwd", "paged_tree_attn", "verify_draft"])
def test_same_as_the_way_through_python(dev, name):
    announce(f"host ops {name}")
    args = _calls(dev)[name]
    copies = lambda: tuple(a.clone() if isinstance(a, torch.Tensor) else a for a in args)
    mine, theirs = copies(), copies()
    native = getattr(_lib.host_ops(), name)(*mine)
    assert native is not None
    _same(native, op_reg.ALL_CUSTOM_OP_REGS[f"mi355.{name}"].eager_execute(*theirs))
    for a, b in zip(mine, theirs):  # what is written in place
        if isinstance(a, torch.Tensor):
            assert torch.equal(a, b)
    # operands that are not laid out as the kernels take them are left to Python, and the op gives the same
    for k, a in enumerate(args):
        if not isinstance(a, torch.Tensor) or (name, k) in (("rope_kv_append", 5), ("rope_kv_append", 6), ("paged_batch_layout", 0)):
            continue
        odd = list(copies())
        odd[k] = torch.stack([a, torch.zeros_like(a)], -1)[..., 0]
        assert not odd[k].is_contiguous() and getattr(_lib.host_ops(), name)(*odd) is None
        _same(getattr(OPS, name)(*odd), native)


@pytest.mark.parametrize("name", ["rope", "rope_kv_append", "paged_batch_layout", "flash_attn_varlen_fwd", "paged_tree_attn", "verify_draft"])
def test_what_breaks_the_contract_is_refused(dev, name):
    """One operand at a time: a row fewer, an axis more, another type, on the host.  Nothing is launched for any of them."""
    announce(f"host ops refusals {name}")
    args = _calls(dev)[name]
    op, native = getattr(OPS, name), getattr(_lib.host_ops(), name)
    for k, a in enumerate(args):
        if not isinstance(a, torch.Tensor):
            continue
        bad = [a[None], a.to(torch.int16), a.cpu()]
        if (name, k) not in FEWER_IS_FINE:
            bad.append(a[..., :-1].contiguous())
        for b in bad:
            changed = (*args[:k], b, *args[k + 1 :])
            assert native(*changed) is None, (k, b.shape, b.dtype, b.device)
            with pytest.raises((ValueError, RuntimeError, NotImplementedError)):
                op(*changed)
    assert native(*args[:-1]) is None and native(*args, 1) is None and native(*([None] * len(args))) is None


def test_gradient_node(dev):
    """Twice differentiable, careful about its saved tensors, through hooks, and with gradients of any strides."""
    announce("host ops gradient node")
    pos, f = torch.arange(6, dtype=torch.int32, device=dev), ita.rope_inv_freq(64, device=dev)[0]
    x = torch.randn(6, 3, 96, device=dev, requires_grad=True)
    call = lambda t: OPS.rope(t, pos, f, True, False, 2.0)
    y = call(x)
    assert "RopeGrad" in y.grad_fn.name() and y.grad_fn.name() != "_RopeGradBackward"
    g = torch.randn(6, 3, 96, device=dev)
    back = OPS.rope(g, pos, f, True, True, 2.0)
    assert torch.equal(torch.autograd.grad(y, x, g, retain_graph=True)[0], back)
    for odd in (g.transpose(0, 2).contiguous().transpose(0, 2), torch.stack([g, g], -1)[..., 1], g[:1].expand(6, 3, 96)):
        assert torch.equal(torch.autograd.grad(y, x, odd, retain_graph=True)[0], OPS.rope(odd.contiguous(), pos, f, True, True, 2.0))
    gr = g.clone().requires_grad_()
    dx = torch.autograd.grad(y, x, gr, create_graph=True)[0]
    again = torch.autograd.grad(dx, gr, x.detach(), create_graph=True)[0]
    assert again is not None and torch.equal(again, call(x.detach()))
    packed = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (packed.append(t.shape), t.cpu())[1], lambda t: t.to(dev)):
        z = call(x)
    assert len(packed) == 2 and torch.equal(torch.autograd.grad(z, x, g)[0], back)
    with torch.no_grad():
        assert not call(x).requires_grad
    z = call(x)
    pos.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(z, x, g)
    pos.sub_(1)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        z = call(x * 1.0)
    torch.cuda.current_stream(dev).wait_stream(side)
    dx = torch.autograd.grad(z, x, g)[0]
    torch.cuda.synchronize()
    assert torch.equal(dx, back)


def test_threads_and_streams(dev):
    """Calls from several threads, each on a stream of its own."""
    import threading

    announce("host ops threads")
    args = _calls(dev)
    want = OPS.flash_attn_varlen_fwd(*args["flash_attn_varlen_fwd"])
    turned = OPS.rope(*args["rope"])
    torch.cuda.synchronize()
    bad = []

    def work():
        s = torch.cuda.Stream(dev)
        with torch.cuda.stream(s):
            outs = [(OPS.flash_attn_varlen_fwd(*args["flash_attn_varlen_fwd"]), OPS.rope(*args["rope"])) for _ in range(50)]
        s.synchronize()
        bad.extend(1 for a, b in outs if not (torch.equal(a, want) and torch.equal(b, turned)))

    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


@pytest.mark.filterwarnings("ignore:There is a performance drop")
def test_forward_mode_and_transforms_on_the_device(dev):
    """Tangents, torch.func and batched gradients of the rotation give what calls on plain tensors give."""
    import torch.autograd.forward_ad as fw

    announce("rope forward mode and torch.func")
    pos, f = torch.arange(5, dtype=torch.int32, device=dev) * 77, ita.rope_inv_freq(64, device=dev)[0]
    call, back = (lambda v: OPS.rope(v, pos, f, False, False, 1.5)), (lambda v: OPS.rope(v, pos, f, False, True, 1.5))
    x, t = (torch.randn(5, 2, 96, device=dev) for _ in range(2))
    with fw.dual_level():
        for leaf in (x, x.clone().requires_grad_()):
            y = fw.unpack_dual(call(fw.make_dual(leaf, t)))
            assert torch.equal(y.tangent, call(t)) and torch.equal(y.primal, call(x))
        leaf = x.clone().requires_grad_()
        for graph in (False, True):
            dx, = torch.autograd.grad(call(leaf), leaf, fw.make_dual(x, t), create_graph=graph)
            assert torch.equal(fw.unpack_dual(dx).tangent, back(t)) and torch.equal(fw.unpack_dual(dx).primal, back(x))
    many = torch.stack([x, t, x - t])
    want = torch.stack([call(v) for v in many])
    assert torch.equal(torch.func.vmap(call)(many), want)
    assert torch.equal(torch.func.jvp(call, (x,), (t,))[1], call(t)) and torch.equal(torch.func.vjp(call, x)[1](t)[0], back(t))
    assert torch.equal(torch.func.grad(lambda v: (call(v) * t).sum())(x), back(t))
    assert torch.equal(torch.func.vmap(torch.func.grad(lambda v: (call(v) * t).sum()))(many), back(t).expand(3, 5, 2, 96))
    assert torch.equal(torch.func.vmap(torch.func.jvp, in_dims=(None, None, 0))(call, (x,), (many,))[1], want)
    assert torch.equal(torch.func.jvp(lambda v: torch.func.grad(lambda w: (call(w) ** 2).sum() / 2)(v), (x,), (t,))[1], back(call(t)))
    leaf = x.clone().requires_grad_()
    y = call(leaf)
    assert "RopeGrad" in y.grad_fn.name()
    assert torch.equal(torch.autograd.grad(y, leaf, many, is_grads_batched=True)[0], torch.stack([back(v) for v in many]))


def test_gradient_of_what_saved_tensor_hooks_give_back(dev):
    """Positions and frequencies that come back laid out otherwise are read as they are; on the host, of another type or
    length they are refused, nothing is launched for them."""
    announce("rope gradient, unpacked tensors")
    pos, f = torch.arange(6, dtype=torch.int32, device=dev) * 9, ita.rope_inv_freq(64, device=dev)[0]
    x, g = (torch.randn(6, 3, 96, device=dev) for _ in range(2))
    leaf = x.clone().requires_grad_()

    def grad(unpack):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            y = OPS.rope(leaf, pos, f, True, False, 2.0)
        assert y.grad_fn.name() != "_RopeGradBackward"
        return torch.autograd.grad(y, leaf, g)[0]

    want = OPS.rope(g, pos, f, True, True, 2.0)
    assert torch.equal(grad(lambda t: t), want)
    assert torch.equal(grad(lambda t: torch.stack([t, t], -1)[..., 0]), want)
    assert torch.equal(grad(lambda t: torch._neg_view(-t)), want)
    for bad in (lambda t: t.cpu(), lambda t: t.to(torch.int64), lambda t: t.repeat(2), lambda t: t[:0]):
        with pytest.raises((ValueError, RuntimeError, NotImplementedError)):
            grad(bad)


@pytest.mark.parametrize("name", ["rope", "rope_kv_append", "paged_batch_layout", "flash_attn_varlen_fwd", "paged_tree_attn", "verify_draft"])
def test_registered_as_torch_expects(dev, name):
    """Schemas say what is written, fake tensors describe the results, and compiled calls with their gradients give the eager ones'."""
    announce(f"opcheck {name}")
    args = _calls(dev)[name]
    torch.library.opcheck(getattr(OPS, name).default, args)
    if name == "rope":
        torch.library.opcheck(OPS.rope.default, (args[0].clone().requires_grad_(), *args[1:]))


def test_limits_are_those_of_the_contract(dev):
    """One past each limit of sizes: the native side leaves the call, and the op's own contract refuses it.  Broadcast operands stand
    for large ones; nothing is launched."""
    announce("host ops limits")
    h = lambda *s, dt=torch.float16: torch.zeros(1, dtype=dt, device=dev).expand(*s) if len(s) else None
    flat = lambda *s, dt=torch.int32: torch.zeros(*s, dtype=dt, device=dev)
    f64, i64 = torch.float64, torch.int64
    f = lambda n: flat(n, dt=f64)
    rows = lambda t, heads: torch.zeros(1, heads, 128, dtype=torch.float16, device=dev).expand(t, heads, 128)
    kc = flat(4, 16, 2, 128, dt=torch.float16)
    table, lens = flat(2, 4), flat(2)
    rope = lambda **k: ("rope", *{**dict(x=flat(4, 2, 64, dt=torch.float16), pos=flat(4), f=f(32), i=False, v=False, s=1.0), **k}.values())
    append = lambda **k: ("rope_kv_append", *{**dict(q=rows(4, 4), k=rows(4, 2), v=rows(4, 2), pos=flat(4), f=f(64), kc=kc, vc=kc.clone(), slots=flat(4, dt=i64), i=False, s=1.0), **k}.values())
    layout = lambda **k: ("paged_batch_layout", *{**dict(t=table, c=lens, n=lens, fr=flat(3), p=16, T=5), **k}.values())
    varlen = lambda **k: ("flash_attn_varlen_fwd", *{**dict(q=rows(4, 4), k=rows(4, 2), v=rows(4, 2), cq=flat(3), ck=flat(3), causal=True, s=0.0), **k}.values())
    tree = lambda **k: ("paged_tree_attn", *{**dict(q=flat(2, 3, 4, 128, dt=torch.float16), kc=kc, vc=kc, t=table, l=lens, p=flat(2, 3), s=0.0, n=0), **k}.values())
    verify = lambda **k: ("verify_draft", *{**dict(p=flat(2, 3, 9, dt=torch.float32), d=None, t=flat(2, 3), a=flat(2, 3), u=flat(2, 3, dt=torch.float32)), **k}.values())
    many = 1 << 24
    calls = [
        rope(x=h(many, 1, 2), pos=flat(many), f=f(1)), rope(x=h(1, 65536, 2), pos=flat(1), f=f(1)), rope(x=h(1, 1, 65537), pos=flat(1), f=f(1)),
        rope(x=h(1, 1, 1100), pos=flat(1), f=f(513)), rope(f=f(33)), rope(x=h(1, 20000, 60000), pos=flat(1), f=f(1)),
        append(q=rows(many, 1), k=rows(many, 2), v=rows(many, 2), pos=flat(many), slots=flat(many, dt=i64)), append(q=rows(4, 65536)), append(f=f(65)),
        append(kc=flat(4, 8, 2, 128, dt=torch.float16), vc=flat(4, 8, 2, 128, dt=torch.float16)),
        layout(t=flat(65536, 1), c=flat(65536), n=flat(65536)), layout(t=flat(1, (1 << 22) + 1), c=flat(1), n=flat(1)), layout(T=(1 << 30) + 1), layout(T=0), layout(p=512),
        varlen(q=rows(many + 1, 2)), varlen(k=rows(many + 1, 2), v=rows(many + 1, 2)), varlen(q=rows(4, 65536)), varlen(q=rows(many, 130)), varlen(cq=flat(65537), ck=flat(65537)),
        varlen(cq=flat(1), ck=flat(1)),
        tree(q=flat(2, 65, 4, 128, dt=torch.float16), p=flat(2, 65)), tree(q=flat(2, 3, 258, 128, dt=torch.float16)), tree(n=1025), tree(t=flat(2, 0)),
        verify(p=flat(65536, 1, 1, dt=torch.float32), t=flat(65536, 1), a=flat(65536, 1), u=flat(65536, 1, dt=torch.float32)),
        verify(p=flat(1, 65, 1, dt=torch.float32), t=flat(1, 65), a=flat(1, 65), u=flat(1, 65, dt=torch.float32)),
        verify(p=flat(1, 1, many + 1, dt=torch.float32), t=flat(1, 1), a=flat(1, 1), u=flat(1, 1, dt=torch.float32)),
    ]
    for name, *args in calls:
        sizes = [tuple(a.shape) if isinstance(a, torch.Tensor) else a for a in args]
        assert getattr(_lib.host_ops(), name)(*args) is None, (name, sizes)
        with pytest.raises(ValueError):
            getattr(OPS, name)(*args)


def test_dispatch_modes_see_the_gradient(dev):
    """A dispatch mode that is entered for the backward pass alone sees the gradient's call as it sees the forward's."""
    from torch.utils._python_dispatch import TorchDispatchMode

    announce("rope gradient under a dispatch mode")

    class Names(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.seen = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.seen.append(str(func))
            return func(*args, **(kwargs or {}))

    pos, f = torch.arange(4, dtype=torch.int32, device=dev), ita.rope_inv_freq(64, device=dev)[0]
    leaf, g = torch.randn(4, 2, 64, device=dev, requires_grad=True), torch.randn(4, 2, 64, device=dev)
    with Names() as forward:
        y = OPS.rope(leaf, pos, f, False, False, 1.0)
    assert "mi355.rope.default" in forward.seen
    y = OPS.rope(leaf, pos, f, False, False, 1.0)
    assert y.grad_fn.name() != "_RopeGradBackward"
    with Names() as backward:
        got, = torch.autograd.grad(y, leaf, g)
    assert "mi355.rope.default" in backward.seen
    assert torch.equal(got, OPS.rope(g, pos, f, False, True, 1.0))
