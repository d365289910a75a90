"""Gradient norm and clipping (ops.grad_norm, ops.clip_grads) against their definition in 64 bits.

Tolerances: the norm is summed in 64 bits and rounded to fp32 once after its square root, so it is
off by half a step, 2^-24, plus the 64-bit sums' 1e-12; the factor (a sum, a division) and the
product add three half steps, so a clipped value is within 2^-22 of the formula's, plus its own
rounding where it is stored in bf16 (2^-8)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F, H = torch.float32, torch.bfloat16


def _tensors(sizes, dts=(F,), seed=0, size=0.1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(size * torch.randn(s, device="cuda", generator=g)).to(dts[k % len(dts)]) for k, s in enumerate(sizes)]


def _norm64(ts):
    return math.sqrt(sum(float(t.double().square().sum()) for t in ts))


def _check(src, dst, norm, max_norm):
    n = _norm64(src)
    assert norm.dtype == F and norm.shape == ()
    assert abs(float(norm) - n) <= (2.0 ** -24 + 1e-11) * n
    c = min(1.0, max_norm / (n + 1e-6))
    for s, d in zip(src, dst):
        ref = s.double() * c
        tol = (2.0 ** -22 + (2.0 ** -8 if d.dtype == H else 0)) * ref.abs() + 1e-44
        assert bool(((d.double() - ref).abs() <= tol).all())


SIZES = [[(5,)], [(1,)], [(4096,)], [(4095,)], [(4097,)], [(3, 7, 11), (), (0,), (129,), (64, 64)],
         [(k % 37 + 1,) for k in range(99)], [(k % 37 + 1,) for k in range(101)], [(k % 5 + 1,) for k in range(2300)],
         [(1000, 1001), (7,), (333, 513)]]


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{s[0]}")
@pytest.mark.parametrize("dts", [(F,), (H,), (F, H)], ids=["f32", "bf16", "mixed"])
@pytest.mark.parametrize("max_norm", [0.01, 1e9])
def test_against_definition(sizes, dts, max_norm):
    from sca2_b200 import ops
    src = _tensors(sizes, dts)
    assert abs(float(ops.grad_norm(src)) - _norm64(src)) <= (2.0 ** -24 + 1e-11) * _norm64(src)
    keep = [t.clone() for t in src]
    out = [torch.full_like(t, 7.0, dtype=F) for t in src]
    n = ops.clip_grads(src, max_norm, out=out)
    _check(keep, out, n, max_norm)
    assert all(torch.equal(a, b) for a, b in zip(src, keep))
    n2 = ops.clip_grads(src, max_norm)  # in place
    assert torch.equal(n, n2)
    _check(keep, src, n, max_norm)
    if max_norm > 1:
        assert all(torch.equal(a, b) for a, b in zip(src, keep))


def test_destinations_of_any_alignment():
    from sca2_b200 import ops
    src = _tensors([(4097,), (8192,), (3,), (5000,)], (F, H))
    flat = torch.full((sum(t.numel() for t in src) + 2,), 7.0, device="cuda")
    outs, at = [], 1
    for t in src:
        outs.append(flat[at:at + t.numel()])
        at += t.numel()
    n = ops.clip_grads(src, 0.5, out=outs)
    _check(src, outs, n, 0.5)
    assert float(flat[0]) == 7.0 and float(flat[-1]) == 7.0  # what lies around them is left alone
    low = torch.zeros(20000, device="cuda", dtype=H)
    outs = [low[1:4098], low[4099:12291], low[12291:12294], low[12295:17295]]
    n = ops.clip_grads(src, 0.5, out=outs)
    _check(src, outs, n, 0.5)
    views = [low[k:k + 4097] for k in (0, 5000)]
    views[0].copy_(src[0]), views[1].copy_(src[0])
    keep = [v.clone() for v in views]
    _check(keep, views, ops.clip_grads(views, 0.5), 0.5)


def test_not_contiguous():
    from sca2_b200 import ops
    t = _tensors([(300, 200)])[0]
    for v in (t.t(), t[:, ::2], t[::3, 5:77]):
        keep, whole = v.clone(), t.clone()
        _check([keep], [v], ops.clip_grads([v], 0.5), 0.5)
        v.copy_(keep)
        assert torch.equal(t, whole)
        assert abs(float(ops.grad_norm(v)) - _norm64([v])) <= (2.0 ** -24 + 1e-11) * _norm64([v])


@pytest.mark.parametrize("size", [1e25, 1e-25, 3e37])
def test_extreme_sizes(size):
    """Squares that 32 bits cannot hold."""
    from sca2_b200 import ops
    src = _tensors([(5000,), (77,)], size=size)
    n = _norm64(src)
    assert abs(float(ops.grad_norm(src)) - n) <= (2.0 ** -24 + 1e-11) * n or n > 3.4e38
    keep = [t.clone() for t in src]
    norm = ops.clip_grads(src, 1.0)
    if n < 3.4e38:
        _check(keep, src, norm, 1.0)


def test_not_finite():
    """As torch.nn.utils.clip_grad_norm_: an infinite norm makes finite values 0 and infinite ones
    NaN, a NaN norm makes all NaN."""
    from sca2_b200 import ops
    a, b = _tensors([(5000,), (100,)])
    b[5] = math.inf
    assert math.isinf(float(ops.clip_grads([a, b], 1.0)))
    assert torch.equal(a, torch.zeros_like(a)) and torch.isnan(b[5]) and int(torch.isnan(b).sum()) == 1
    a, b = _tensors([(5000,), (100,)])
    b[5] = math.nan
    assert math.isnan(float(ops.clip_grads([a, b], 1.0)))
    assert torch.isnan(a).all() and torch.isnan(b).all()


def test_nothing():
    from sca2_b200 import ops
    assert float(ops.grad_norm([])) == 0 and float(ops.clip_grads([], 1.0)) == 0
    z = torch.zeros(0, device="cuda")
    assert float(ops.clip_grads([z, z], 1.0)) == 0 and float(ops.grad_norm([z])) == 0
    t = _tensors([(50,)])[0]
    ops.clip_grads([t], 0.0)
    assert torch.equal(t, torch.zeros_like(t))


def test_shared_memory_is_refused():
    from sca2_b200 import _lib, ops
    t, o = _tensors([(100,), (100,)])
    keep = t.clone()
    for src, dst in (([t, t], None), ([t[:60], t[50:]], None), ([t, o], [o, t]), ([t, o], [o[:100], o]),
                     ([t[:90]], [t[10:]]), ([t.view(H)[:100]], [t])):
        with pytest.raises(_lib.Sca2Error, match="overlap"):
            ops.clip_grads(src, 1.0, out=dst)
    assert torch.equal(t, keep)
    assert abs(float(ops.grad_norm([t, t])) - _norm64([t, t])) < 1e-6  # reading twice is fine
    ops.clip_grads([t[:50], t[50:]], 0.5)
    _check([keep], [t], torch.tensor(_norm64([keep])), 0.5)


def test_not_contiguous_tensors_apart():
    from sca2_b200 import _lib, ops
    t = _tensors([(64, 64)])[0]
    keep = t.clone()
    for ts in ([t[:, ::2], t[:, ::2]], [t[:, :40], t[:, 30:]], [t[::2], t], [t.t(), t]):
        with pytest.raises(_lib.Sca2Error, match="overlap"):
            ops.clip_grads(ts, 0.5)
    assert torch.equal(t, keep)
    parts = [t[:20, ::2], t[20:40].t(), t[40:]]
    ref = [p.clone() for p in parts]
    _check(ref, parts, ops.clip_grads(parts, 0.5), 0.5)
    with torch.inference_mode():
        i = keep.clone()
        _check([keep], [i], ops.clip_grads([i], 0.5), 0.5)


def test_sparse_is_refused():
    from sca2_b200 import _lib, ops
    t = torch.eye(4, device="cuda").to_sparse()
    for call in (lambda: ops.grad_norm([t]), lambda: ops.clip_grads([t], 1.0)):
        with pytest.raises(_lib.Sca2Error, match="dense"):
            call()


def test_compiled():
    from sca2_b200 import ops
    a, b = _tensors([(40,), (3, 5)])
    x, y = a.clone(), b.clone()
    n = ops.clip_grads([a, b], 0.1)
    f = torch.compile(lambda u, v: ops.clip_grads([u, v], 0.1), fullgraph=True, backend="aot_eager")
    assert torch.equal(f(x, y), n) and torch.equal(x, a) and torch.equal(y, b)
    g = torch.compile(lambda u, v: ops.grad_norm([u, v]), fullgraph=True, backend="aot_eager")
    assert torch.equal(g(a, b), ops.grad_norm([a, b]))


def test_versions():
    """An in-place clip counts as one for autograd's check of saved tensors."""
    from sca2_b200 import ops
    t = _tensors([(50,)])[0]
    v = t._version
    ops.clip_grads([t], 0.5)
    assert t._version > v


def test_streams_and_graphs():
    from sca2_b200 import ops
    src = _tensors([(100, 300), (7,), (4097,)], (F, H))
    out = [[torch.zeros_like(t, dtype=F) for t in src] for _ in range(2)]
    ref = [torch.zeros_like(t, dtype=F) for t in src]
    n = ops.clip_grads(src, 0.5, out=ref)
    graphs, norms = [], []
    for o in out:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            norms.append(ops.clip_grads(src, 0.5, out=o))
        graphs.append(g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
    torch.cuda.synchronize()
    for o, m in zip(out, norms):
        assert torch.equal(m, n) and all(torch.equal(a, b) for a, b in zip(o, ref))
    for t in src:  # new values, same addresses
        t.mul_(3)
    graphs[0].replay()
    torch.cuda.synchronize()
    _check(src, out[0], norms[0], 0.5)


def test_custom_ops():
    src = _tensors([(40,), (3, 5)])
    torch.library.opcheck(torch.ops.sca2b200.grad_norm, (src,))
    torch.library.opcheck(torch.ops.sca2b200.clip_grads_, (src, 0.5))


def test_train_step_clips():
    """lm.train_step(max_norm=): the update of the clipped gradients (plain SGD shows them)."""
    from sca2_b200 import lm as L
    torch.manual_seed(0)
    model = L.LaplaceLM(64, d=32, n_layers=2, M=12, dv=8, L=8, ff=48, chunk=16, theta_scale=0.3).cuda()
    tok = torch.randint(0, 64, (2, 33), device="cuda")
    L.lm_loss(model, tok).backward()
    grads = {n: p.grad.clone() for n, p in model.named_parameters() if p.grad is not None}
    before = {n: p.detach().clone() for n, p in model.named_parameters()}
    n = _norm64(grads.values())
    model.zero_grad(set_to_none=True)
    L.train_step(model, torch.optim.SGD(model.parameters(), lr=1.0), tok, dtype=None, max_norm=0.25 * n)
    for name, p in model.named_parameters():
        if name in grads:
            ref = before[name].double() - 0.25 * grads[name].double()
            # the backward's atomics may move a gradient by a few fp32 steps of its largest value
            assert float((p.detach().double() - ref).abs().max()) <= 1e-5 * (float(grads[name].abs().max()) + float(before[name].abs().max()))
