"""The block operators and the clip as torch's transformations meet them, without a GPU: what a trace
records, what batching keeps for the backward, what is refused.  The launches are stubbed (they write
nothing), so only structure is compared, never values."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

from sca2_b200 import _lib, ops

H = torch.bfloat16


class Mode(TorchDispatchMode):
    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


@pytest.fixture
def stub(monkeypatch):
    """CPU tensors pass for CUDA ones and every launch is recorded instead of made."""
    calls = []
    monkeypatch.setattr(ops, "_need_cuda", lambda *ts: torch.device("cuda", 0))
    monkeypatch.setattr(ops, "_launch", lambda what, fn, dev, *args: calls.append((what, args)))
    return calls


def _ffn(grad=False):
    return [torch.zeros(s, dtype=H).requires_grad_(grad) for s in ((4, 16), (24, 16), (24, 16))]


def _norm(grad=False):
    return [torch.zeros(s).requires_grad_(grad) for s in ((4, 16), (4, 16), (16,))]


def _targets(gm):
    return [str(n.target) for n in gm.graph.nodes if n.op == "call_function"]


def _grads(f, outs):
    def g(*args):
        o = f(*args)
        return torch.autograd.grad(o, args, torch.ones_like(o))
    return g


# (function, its tensors, the operators that its trace has to hold)
CASES = {
    "ffn": (lambda x, g, u: ops.gated_ffn(x, g, u), _ffn, ["gated_ffn_fwd"]),
    "norm": (lambda x, u, w: ops.residual_norm(x, u, w)[1], _norm, ["residual_norm_fwd"]),
    "grad_norm": (lambda x, u, w: ops.grad_norm([x, u, w]), _norm, ["grad_norm"]),
    "clip": (lambda x, u, w: ops.clip_grads([x, u, w], 1.0), _norm, ["clip_grads_"]),
    "clip_out": (lambda x, u, w: ops.clip_grads([x], 1.0, out=[u]), _norm, ["clip_grads_out"]),
}


@pytest.mark.parametrize("kw", [dict(), dict(pre_dispatch=True), dict(tracing_mode="fake"), dict(tracing_mode="symbolic")],
                         ids=lambda k: "-".join(map(str, k.values())) or "real")
@pytest.mark.parametrize("case", CASES)
def test_make_fx_records_the_operators(stub, case, kw):
    f, ins, want = CASES[case]
    got = _targets(make_fx(f, **kw)(*ins()))
    assert all(any(f"sca2b200.{w}.default" in t for t in got) for w in want), got


@pytest.mark.parametrize("case", ["ffn", "norm"])
def test_make_fx_records_the_gradients(stub, case):
    f, ins, want = CASES[case]
    got = _targets(make_fx(_grads(f, 1))(*ins(True)))
    for w in (want[0], want[0].replace("fwd", "bwd")):
        assert any(f"sca2b200.{w}.default" in t for t in got), got
    leaves = ins(True)  # a graph made outside of the trace
    out = f(*leaves)
    got = _targets(make_fx(lambda d: torch.autograd.grad(out, leaves, d, retain_graph=True))(torch.ones_like(out)))
    assert any(f"sca2b200.{want[0].replace('fwd', 'bwd')}.default" in t for t in got), got


@pytest.mark.parametrize("case", CASES)
@pytest.mark.filterwarnings("ignore")
def test_jit_trace_records_the_operators(stub, case):
    f, ins, want = CASES[case]
    assert f"sca2b200::{want[0]}" in str(torch.jit.trace(f, ins(), check_trace=False).graph)


def test_dispatch_modes_see_the_operators(stub):
    class Seen(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.ops = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.ops.append(str(func))
            return func(*args, **(kwargs or {}))
    for f, ins, want in CASES.values():
        with Seen() as seen:
            f(*ins())
        assert all(f"sca2b200.{w}.default" in seen.ops for w in want), seen.ops


def test_plain_calls_go_straight_to_the_library(stub):
    for f, ins, _ in CASES.values():
        f(*ins())
    assert [w for w, _ in stub] == ["gated_ffn", "residual_norm", "grad_norm", "clip_grads", "clip_grads"]


class Seen(torch.Tensor):
    """A tensor that notes the operators it meets."""
    ops = []

    @staticmethod
    def __new__(cls, t):
        r = torch.Tensor._make_wrapper_subclass(cls, t.shape, dtype=t.dtype, device=t.device, requires_grad=t.requires_grad)
        r.inner = t.detach()
        return r

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        cls.ops.append(str(func))
        un = lambda t: t.inner if isinstance(t, cls) else [un(i) for i in t] if isinstance(t, (list, tuple)) else t
        return func(*[un(a) for a in args], **{k: un(v) for k, v in (kwargs or {}).items()})


@pytest.mark.parametrize("case", CASES)
def test_any_tensor_of_a_subclass_brings_the_operators(stub, case):
    f, ins, want = CASES[case]
    for k in range({"clip_out": 2}.get(case, 3)):
        Seen.ops = []
        f(*[Seen(t) if j == k else t for j, t in enumerate(ins())])
        assert f"sca2b200.{want[0]}.default" in Seen.ops, k
    if case in ("ffn", "norm"):  # a gradient of a subclass that reaches a plain graph
        leaves = ins(True)
        out = f(*leaves)
        Seen.ops = []
        torch.autograd.grad(out, leaves, Seen(torch.ones_like(out)))
        assert f"sca2b200.{want[0].replace('fwd', 'bwd')}.default" in Seen.ops


def test_fake_weights_beside_plain_inputs(stub):
    from torch._subclasses.fake_tensor import FakeTensor, FakeTensorMode
    mode = FakeTensorMode(allow_non_fake_inputs=True)
    x, w, _ = _ffn()
    assert isinstance(ops.gated_ffn(x, mode.from_tensor(w), w), FakeTensor)
    x, u, w = _norm()
    y, z = ops.residual_norm(x, u, mode.from_tensor(w))
    assert isinstance(y, FakeTensor) and isinstance(z, FakeTensor)
    assert isinstance(ops.clip_grads([x, mode.from_tensor(u)], 1.0), FakeTensor)
    assert not stub


@pytest.mark.parametrize("case", ["ffn", "norm"])
def test_forward_mode_is_refused(stub, case):
    """A tangent would be lost without a word, in either pass."""
    import torch.autograd.forward_ad as fw
    f, ins, _ = CASES[case]
    refused = lambda: pytest.raises(ops._lib.Sca2Error, match="forward")
    for k in range(3):
        with fw.dual_level(), refused():
            f(*[fw.make_dual(t, torch.ones_like(t)) if j == k else t for j, t in enumerate(ins())])
        plain = ins()
        one = lambda t, k=k: f(*[t if j == k else o for j, o in enumerate(plain)])
        x = plain[k]
        for call in (lambda: torch.func.jvp(one, (x,), (x,)), lambda: torch.func.jacfwd(one)(x),
                     lambda: torch.func.jvp(lambda t: torch.func.vmap(lambda s: one(t))(torch.zeros(2)), (x,), (x,))):
            with refused():
                call()
        with pytest.raises(RuntimeError):  # torch.func.grad itself does not take registered operators
            torch.func.jvp(torch.func.grad(lambda t: one(t).float().sum()), (x,), (x,))
    leaves = ins(True)
    out = f(*leaves)
    with fw.dual_level(), refused():
        torch.autograd.grad(out, leaves, fw.make_dual(torch.ones_like(out), torch.ones_like(out)))
    with fw.dual_level():  # without a tangent a level costs nothing
        f(*ins())


def test_a_batched_join_keeps_its_statistics(stub):
    """A leaf outside of vmap: the batched tensor does not say that it requires gradients, its output does."""
    x, u, w = (torch.zeros(s) for s in ((3, 4, 16), (3, 4, 16), (16,)))
    for leaf in (x, w):
        leaf.requires_grad_(True)
        stub.clear()
        y, z = torch.func.vmap(lambda a, b: ops.residual_norm(a, b, w))(x, u)
        assert z.requires_grad
        forward = [args for what, args in stub if what == "residual_norm"]
        assert len(forward) == 3 and all(args[3] for args in forward)  # the statistics' address
        torch.autograd.grad(z.sum() + y.sum(), leaf)
        assert [args[1] for what, args in stub if what == "residual_norm_bwd"] == [args[3] for args in forward][::-1]
        leaf.requires_grad_(False)
    stub.clear()
    with torch.no_grad():
        torch.func.vmap(lambda a, b: ops.residual_norm(a, b, w))(x, u)
    assert not any(args[3] for what, args in stub)


def test_a_tensor_that_overlaps_itself_is_not_clipped_in_place(stub):
    x = torch.zeros(8, 16)
    for bad in (x[:1, :1].expand(8, 16), x.view(-1).unfold(0, 8, 4), x[:, :3].as_strided((4, 3), (2, 1))):
        with pytest.raises(ops._lib.Sca2Error, match="overlap"):
            ops.clip_grads([torch.zeros(5), bad], 1.0)
        assert not stub
        ops.grad_norm([bad])
        ops.clip_grads([bad], 1.0, out=[torch.zeros(bad.shape)])
        stub.clear()
    for good in (x.t(), x[::2, 3:9], x.view(2, 4, 16).permute(2, 0, 1), x[:1, 2:3].expand(1, 1, 1), x[:0].expand(3, 0, 16)):
        ops.clip_grads([good], 1.0)
    assert len(stub) == 5


def _op_calls():
    """Calls of the registered operators with one argument that does not fit the others."""
    o = torch.ops.sca2b200
    z = lambda *s, t=H: torch.zeros(*s, dtype=t)
    x, w, dh = z(4, 16), z(24, 16), z(4, 24)
    for a in ((x, w, z(16, 16)), (x, z(24, 8), z(24, 8)), (x.float(), w, w), (x, w.half(), w), (z(4, 12), z(24, 12), z(24, 12)),
              (x, z(16), z(16))):
        yield lambda a=a: o.gated_ffn_fwd(*a, 0)
        yield lambda a=a: o.gated_ffn_bwd(*a, 0, dh, True, True)
    for bad in (z(3, 24), z(4, 16), z(24)):
        yield lambda bad=bad: o.gated_ffn_bwd(x, w, w, 0, bad, True, True)
    f = torch.float32
    x, v, st = z(4, 16, t=f), z(16, t=f), z(4, 4, t=f)
    ins = dict(x=x, u=x, w=v, b=v, gate=x, scale=v, pw=v, pb=v)
    for k, bad in (("u", z(4, 8, t=f)), ("u", z(3, 16, t=f)), ("w", z(8, t=f)), ("b", z(16)), ("gate", z(4, 2, t=f)), ("gate", z(4, 16)),
                   ("gate", z(4, t=f)), ("scale", z(1, t=f)), ("pw", z(16, t=torch.double)), ("pb", z(16, 1, t=f)), ("x", z(4, 16, t=torch.half)),
                   ("w", None), ("pw", None)):
        a = [*{**ins, k: bad}.values(), 0, 1e-5, f]
        yield lambda a=a: o.residual_norm_fwd(*a, True)
        yield lambda a=a: o.residual_norm_bwd(*a, st, x, x)
    a = [*ins.values(), 0, 1e-5, f]
    yield lambda: o.residual_norm_fwd(*ins.values(), 0, 1e-5, torch.half, True)
    for st2, dy, dz in ((z(0, 4, t=f), x, x), (z(3, 4, t=f), x, x), (z(4, 4), x, x), (z(4, 8, t=f)[:, ::2], x, x), (st, z(3, 16, t=f), x),
                        (st, x, z(4, 8, t=f))):
        yield lambda s=st2, p=dy, q=dz: o.residual_norm_bwd(*a, s, p, q)


def test_registered_operators_check_their_arguments(stub):
    for k, call in enumerate(_op_calls()):
        with pytest.raises(ops._lib.Sca2Error):
            call()
        assert not stub, k


def test_registered_operators_refuse_cpu_tensors(monkeypatch):
    """Without the stub of the device check: no host address reaches a launch."""
    made = []
    monkeypatch.setattr(ops, "_launch", lambda *a: made.append(a))
    o, (x, w, _), n = torch.ops.sca2b200, _ffn(), torch.zeros(4, 16)
    v, dh = torch.zeros(16), torch.zeros(4, 24, dtype=H)
    for call in (lambda: o.gated_ffn_fwd(x, w, w, 0), lambda: o.gated_ffn_bwd(x, w, w, 0, dh, True, True),
                 lambda: o.residual_norm_fwd(n, n, v, v, None, None, None, None, 0, 1e-5, torch.float32, True),
                 lambda: o.residual_norm_bwd(n, n, v, v, None, None, None, None, 0, 1e-5, torch.float32, torch.zeros(4, 4), n, n),
                 lambda: o.grad_norm([n]), lambda: o.clip_grads_([n], 1.0), lambda: o.clip_grads_out([n], [n], 1.0)):
        with pytest.raises(ops._lib.Sca2Error, match="CUDA"):
            call()
    assert not made


def test_a_gate_of_another_type_keeps_its_bits(stub):
    x, u = torch.zeros(4, 16), torch.zeros(4, 16, dtype=H)
    for gate in (torch.zeros(4, 1), torch.zeros(4, 16), torch.zeros(4, 16, dtype=torch.half)):
        ops.residual_norm(x, u, gate=gate)
    assert [args[0].u_dtype for _, args in stub] == [_lib.SCA2_F32] * 3
    ops.residual_norm(x, u, gate=u)
    assert stub[-1][1][0].u_dtype == _lib.SCA2_BF16


@pytest.mark.parametrize("case", ["grad_norm", "clip", "clip_out"])
def test_not_differentiable_in_a_trace_either(stub, case):
    """Tensors that require gradients: the norm and what is written do not become part of a graph."""
    f, ins, _ = CASES[case]
    for leaf in (True, False):
        ts = [t if leaf else t * 1 for t in ins(True)]
        nodes = [t.grad_fn for t in ts]
        with Mode():
            n = f(*ts)
        assert not n.requires_grad and [t.grad_fn for t in ts] == nodes
