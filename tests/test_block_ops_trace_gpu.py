"""The block operators and the clip in traces, run: graphs recorded by make_fx, torch.jit.trace and
torch.compile give what the eager calls give, bit for bit (the same kernels on the same values)."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

pytestmark = pytest.mark.gpu
H = torch.bfloat16


def _randn(*s, seed=0, grad=False, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed + sum(s))
    return torch.randn(*s, device="cuda", generator=g).to(dtype).requires_grad_(grad)


def _ffn():
    return [_randn(*s, seed=k, grad=True, dtype=H) for k, s in enumerate([(70, 64), (72, 64), (72, 64)])]


def _norm():
    return [_randn(*s, seed=k, grad=True) for k, s in enumerate([(70, 64), (70, 64), (64,), (70, 1)])]


def _both(f, ins):
    o = f(*ins)
    return (o.detach(), *torch.autograd.grad(o, ins, torch.ones_like(o)))


def _block(kind):
    from sca2_b200 import ops
    if kind == "ffn":
        return (lambda x, g, u: ops.gated_ffn(x, g, u)), _ffn()
    return (lambda x, u, w, g: ops.residual_norm(x, u, w, gate=g, post_weight=w)[1]), _norm()


@pytest.mark.parametrize("mode", ["real", "fake"])
@pytest.mark.parametrize("kind", ["ffn", "norm"])
def test_make_fx(kind, mode):
    f, ins = _block(kind)
    ref = _both(f, ins)
    gm = make_fx(lambda *t: _both(f, t), tracing_mode=mode)(*ins)
    assert all(torch.equal(a, b) for a, b in zip(ref, gm(*ins)))
    new = [t.detach() * 0.5 for t in ins]  # other values than those of the trace
    ref = _both(f, [t.clone().requires_grad_(True) for t in new])
    assert all(torch.equal(a, b) for a, b in zip(ref, gm(*new)))


@pytest.mark.parametrize("kind", ["ffn", "norm"])
@pytest.mark.filterwarnings("ignore")
def test_jit_trace(kind):
    f, ins = _block(kind)
    t = torch.jit.trace(f, [i.detach() for i in ins], check_trace=False)
    new = [i.detach() * 0.5 for i in ins]
    assert torch.equal(t(*new), f(*new))


def test_clip_in_a_trace():
    from sca2_b200 import ops
    src = lambda: [_randn(40), _randn(3, 5, dtype=H)]
    a, b = src()
    n = ops.clip_grads([a, b], 0.1)
    norm = ops.grad_norm(src())
    gm = make_fx(lambda x, y: ops.clip_grads([x, y], 0.1))(*src())
    x, y = src()
    assert torch.equal(gm(x, y), n) and torch.equal(x, a) and torch.equal(y, b)
    assert torch.equal(make_fx(lambda x, y: ops.grad_norm([x, y]))(*src())(*src()), norm)
    into = lambda x, y, p, q: ops.clip_grads([x, y], 0.1, out=[p, q])
    for g in (make_fx(into)(*src(), torch.empty(40, device="cuda"), torch.empty(3, 5, device="cuda")),
              torch.compile(into, fullgraph=True, backend="aot_eager")):
        p, q = torch.zeros(40, device="cuda"), torch.zeros(3, 5, device="cuda", dtype=H)
        assert torch.equal(g(*src(), p, q), n) and torch.equal(p, a) and torch.equal(q, b)
    empty = torch.compile(lambda x: x + ops.clip_grads([], 1.0) + ops.grad_norm([]), fullgraph=True, backend="aot_eager")
    assert torch.equal(empty(norm), norm)
    torch.library.opcheck(torch.ops.sca2b200.clip_grads_out, (src(), [torch.zeros(40, device="cuda"), torch.zeros(3, 5, device="cuda")], 0.1))


@pytest.mark.parametrize("kind", ["ffn", "norm"])
def test_vmap_backward(kind):
    """Gradients of leaves outside of vmap: the calls one by one give the same."""
    f, ins = _block(kind)
    x = torch.stack([ins[0].detach() * k for k in (0.5, 1.0, 2.0)]).requires_grad_(True)
    rest = [t.detach().clone().requires_grad_(True) for t in ins[1:]]
    g = _randn(3, *f(*ins).shape, seed=9, dtype=ins[0].dtype)
    out = torch.func.vmap(lambda a: f(a, *rest))(x)
    got = torch.autograd.grad(out, (x, *rest), g)
    one = [torch.autograd.grad(f(a, *rest), (a, *rest), d) for a, d in
           zip([t.detach().requires_grad_(True) for t in x], g)]
    assert torch.equal(got[0], torch.stack([o[0] for o in one]))
    for k, t in enumerate(got[1:], 1):  # three gradients added, in an order that is autograd's: 2 roundings each way
        ref = sum(o[k].double() for o in one)
        size = sum(o[k].double().abs() for o in one)
        assert bool(((t.double() - ref).abs() <= 2.02 * torch.finfo(t.dtype).eps / 2 * size + 1e-30).all())


def test_vmap_over_parameters():
    """Slices that are not contiguous, of parameters too."""
    from sca2_b200 import ops
    x, u = _randn(70, 64), _randn(70, 64, seed=1)
    ws = [_randn(64, 3, seed=2 + k, grad=True) for k in range(3)]
    f = lambda w, s, p: ops.residual_norm(x, u, w, scale=s, post_weight=p)
    y, z = torch.func.vmap(f, in_dims=1)(*ws)
    got = torch.autograd.grad(z, ws, torch.ones_like(z))
    for k in range(3):
        one = [w.detach()[:, k].contiguous().requires_grad_(True) for w in ws]
        ry, rz = f(*one)
        assert torch.equal(y[k], ry) and torch.equal(z[k], rz)
        for g, r in zip(got, torch.autograd.grad(rz, one, torch.ones_like(rz))):
            assert torch.equal(g[:, k], r)


def test_clip_of_parameters_compiled():
    """Leaves that require gradients, as in the plain call: nothing becomes part of a graph."""
    from sca2_b200 import ops
    a, b = _randn(40, grad=True), _randn(3, 5, grad=True)
    x, y = a.detach().clone().requires_grad_(True), b.detach().clone().requires_grad_(True)
    n = ops.clip_grads([a, b], 0.1)
    m = torch.compile(lambda u, v: ops.clip_grads([u, v], 0.1), fullgraph=True, backend="aot_eager")(x, y)
    assert torch.equal(n, m) and not m.requires_grad and torch.equal(a, x) and torch.equal(b, y) and x.is_leaf
    r = torch.compile(lambda u, v: ops.grad_norm([u, v]), fullgraph=True, backend="aot_eager")(x, y)
    assert torch.equal(r, ops.grad_norm([a, b])) and not r.requires_grad
