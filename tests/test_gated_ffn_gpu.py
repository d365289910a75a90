"""The gated feed-forward projections (ops.gated_ffn) against their definition in 64 bits: h and the
three gradients over row counts on both sides of each kernel's bounds (decode fragments, tiles of
256 rows), widths inside and across tiles, splits of the rows, strides, streams, graphs.

Tolerances, element by element.  Products of bf16 values are exact in fp32; a contraction over n
values adds them in fp32, whose error is below (n / 8 + 16) 2^-23 of the sum of the products' sizes
(blocks of 16 are summed at once, a chain of at most n / 16 additions follows, each of which may
truncate).  The activations are good to 2^-20 of their terms.  Roundings to bf16 are 2^-8 of the
value each: h once; dg and du once and the gradients once more.  Whole outputs of over 1000 values
are also compared in the 2-norm: two roundings of 0.45 x 2^-8 root mean square each give 0.64 x 2^-8;
the bar is 2^-8."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
H = torch.bfloat16
U = 2.0 ** -8


def _inputs(rows, d, f, seed=0, x_pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed + rows + 31 * d + 17 * f)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)
    x = r(rows, d + x_pad).to(H)[:, :d]
    return x, (r(f, d) * d ** -0.5).to(H), (r(f, d) * d ** -0.5).to(H), r(rows, f).to(H)


def _act(g, act):
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    p = 0.5 * torch.erfc(-g / math.sqrt(2))
    return g * p, p + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)


def _exact(x, wg, wu, dh, act):
    """{name: (value, tolerance)} in 64 bits."""
    x, wg, wu, dh = (t.detach().double() for t in (x, wg, wu, dh))
    add = lambda n: (n / 8 + 16) * 2.0 ** -23
    g, u = x @ wg.t(), x @ wu.t()
    eg, eu = add(x.shape[1]) * (x.abs() @ wg.abs().t()), add(x.shape[1]) * (x.abs() @ wu.abs().t())
    a, da = _act(g, act)
    fn = 2.0 ** -20 * (1 + g.abs())       # the functions' own error
    ea = 1.2 * eg + fn                    # |act'| <= 1.13 for both
    ed = 0.9 * eg + fn                    # |act''| <= 0.8 for both
    h = a * u
    dg, du = dh * u * da, dh * a
    edg = dh.abs() * (ed * u.abs() + 1.2 * eu + ed * eu) + U * dg.abs()
    edu = dh.abs() * ea + U * du.abs()
    out = {"h": (h, ea * u.abs() + a.abs() * eu + ea * eu + U * h.abs())}
    dx = dg @ wg + du @ wu
    out["dx"] = (dx, edg @ wg.abs() + edu @ wu.abs() + U * dx.abs()
                 + add(2 * wg.shape[0]) * (dg.abs() @ wg.abs() + du.abs() @ wu.abs()))
    for k, v, e in (("dwg", dg, edg), ("dwu", du, edu)):
        w = v.t() @ x
        out[k] = (w, e.t() @ x.abs() + U * w.abs() + add(x.shape[0]) * (v.abs().t() @ x.abs()))
    return out


def _near(name, got, ref, tol):
    err = (got.double() - ref).abs()
    worst = float((err / (tol + 1e-30)).max()) if err.numel() else 0.0
    assert got.dtype == H and got.shape == ref.shape and worst <= 1.0, (name, worst)
    if got.numel() > 1000:
        rel = float(err.norm() / ref.norm())
        assert rel <= U, (name, rel)


def _run(x, wg, wu, dh, act):
    from sca2_b200 import ops
    leaves = [t.detach().requires_grad_(True) for t in (x, wg, wu)]
    h = ops.gated_ffn(*leaves, act=act)
    return dict(zip(("h", "dx", "dwg", "dwu"), (h.detach(), *torch.autograd.grad(h, leaves, dh))))


def _check(x, wg, wu, dh, act="silu"):
    from sca2_b200 import _lib, ops
    got, ref = _run(x, wg, wu, dh, act), _exact(x, wg, wu, dh, act)
    assert _lib.device_faults() == 0
    for k in got:
        _near(k, got[k], *ref[k])
    with torch.no_grad():
        assert torch.equal(ops.gated_ffn(x, wg, wu, act=act), got["h"])


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("rows", [1, 7, 8, 9, 16, 17, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300, 513])
def test_rows(rows, act):
    _check(*_inputs(rows, 136, 200), act)


@pytest.mark.parametrize("d,f", [(8, 8), (8, 16), (64, 128), (64, 8), (72, 136), (128, 64), (256, 256), (264, 248), (520, 1096),
                                 (768, 2048), (1024, 512), (2056, 72), (40, 4104)])
@pytest.mark.parametrize("rows", [3, 50, 700])
def test_widths(rows, d, f):
    _check(*_inputs(rows, d, f))


@pytest.mark.parametrize("rows,d,f", [(20000, 256, 256), (9000, 64, 72), (33000, 128, 640), (5000, 768, 2048)])
def test_many_rows(rows, d, f):
    """Weight gradients split over the rows, several tiles for each pair of CTAs."""
    _check(*_inputs(rows, d, f), "gelu")


def test_values():
    """Against small whole numbers, where every sum is exact: each value in its place."""
    from sca2_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(1)
    i = lambda *s: torch.randint(-2, 3, s, device="cuda", generator=g).to(H)
    for rows in (5, 40, 600):
        x, wg, wu = i(rows, 136), i(264, 136), i(264, 136)
        pre, up = x.double() @ wg.double().t(), x.double() @ wu.double().t()
        ref = pre * torch.sigmoid(pre) * up
        got = ops.gated_ffn(x, wg, wu).double()
        assert bool(((got - ref).abs() <= (U + 2.0 ** -20) * ref.abs() + 1e-12).all())


def test_strides_and_views():
    from sca2_b200 import ops
    for rows in (20, 400):
        x, wg, wu, dh = _inputs(rows, 72, 136, x_pad=8)
        ref = _run(x.contiguous(), wg, wu, dh, "silu")
        both = torch.cat([wg, wu])
        for xs, a, b, g in ((x, wg, wu, dh), (x, both[:136], both[136:], dh),
                            (x, torch.cat([wg, wu], 1)[:, :72], torch.cat([wu, wg], 1)[:, :72], dh),
                            (x.t().contiguous().t(), wg.t().contiguous().t(), wu, dh.t().contiguous().t()),
                            (torch.cat([x.new_zeros(3), x.reshape(-1)])[3:].view(rows, 72), wg, wu, dh)):
            for k, v in _run(xs, a, b, g, "silu").items():
                assert torch.equal(v, ref[k]), k
        h = ops.gated_ffn(x.contiguous().view(4, rows // 4, 72), wg, wu)
        assert torch.equal(h.view(rows, 136), ref["h"])
        assert torch.equal(ops.gated_ffn(x[0], wg, wu), ops.gated_ffn(x[:1], wg, wu)[0])
        leaves = [t.detach().requires_grad_(True) for t in (x, wg, wu)]
        ops.gated_ffn(*leaves).sum().backward()  # a broadcast gradient
        one = _run(x, wg, wu, torch.ones_like(dh), "silu")
        assert torch.equal(leaves[0].grad, one["dx"]) and torch.equal(leaves[1].grad, one["dwg"])
        e = x[:1].expand(rows, 72)
        assert torch.equal(ops.gated_ffn(e, wg, wu), ops.gated_ffn(e.contiguous(), wg, wu))


def test_no_rows_and_partial_gradients():
    from sca2_b200 import ops
    x, wg, wu, dh = _inputs(300, 64, 72)
    leaves = [t.detach().requires_grad_(True) for t in (x[:0], wg, wu)]
    h = ops.gated_ffn(*leaves)
    assert h.shape == (0, 72)
    h.sum().backward()
    assert leaves[0].grad.shape == (0, 64) and torch.equal(leaves[1].grad, torch.zeros_like(wg))
    ref = _run(x, wg, wu, dh, "gelu")
    for need in ((1, 0, 0), (0, 1, 1), (0, 1, 0), (0, 0, 1)):
        t = [v.detach().requires_grad_(bool(n)) for v, n in zip((x, wg, wu), need)]
        ops.gated_ffn(*t, act="gelu").backward(dh)
        for v, n, k in zip(t, need, ("dx", "dwg", "dwu")):
            assert (v.grad is not None and torch.equal(v.grad, ref[k])) if n else v.grad is None
    w = wg.detach().requires_grad_(True)  # one weight in both places: the gradients add
    ops.gated_ffn(x, w, w).backward(dh)
    a = _run(x, wg, wg, dh, "silu")
    assert torch.equal(w.grad, a["dwg"] + a["dwu"])


def test_rows_are_independent():
    """NaN and infinities of one row of x, and of dh, stay in its row of h and dx."""
    for rows in (30, 600):
        x, wg, wu, dh = _inputs(rows, 72, 136)
        clean = _run(x, wg, wu, dh, "silu")
        x2, dh2 = x.clone(), dh.clone()
        x2[5, 3], dh2[11, 7] = math.nan, math.inf
        got = _run(x2, wg, wu, dh2, "silu")
        keep = [r for r in range(rows) if r not in (5, 11)]
        assert torch.equal(got["h"][keep], clean["h"][keep]) and torch.equal(got["dx"][keep], clean["dx"][keep])
        assert torch.equal(got["h"][11], clean["h"][11])
        assert torch.isnan(got["h"][5]).all() and not torch.isfinite(got["dx"][11]).any()


def test_large_preactivations():
    """Pre-activations far outside the exponential's range."""
    from sca2_b200 import ops
    for rows in (4, 300):
        x = torch.full((rows, 8), 64.0, device="cuda", dtype=H)
        w = torch.zeros(16, 8, device="cuda", dtype=H)
        w[:8], w[8:] = 2.0, -2.0
        one = torch.full((16, 8), 1 / 512, device="cuda", dtype=H)
        for act in ("silu", "gelu"):
            h = ops.gated_ffn(x, w, one, act=act)
            assert bool((h[:, :8] == 1024).all()) and bool((h[:, 8:] == 0).all())
            got = _run(x, w, one, torch.ones(rows, 16, device="cuda", dtype=H), act)
            assert all(bool(torch.isfinite(v).all()) for v in got.values())


def test_gradient_against_differences():
    """Central differences of sum(h dh) in 64 bits of the values that the kernel returns.  h is
    rounded to bf16, so the difference is taken over a large step along the gradient itself: the
    change of the sum, |grad|^2 2 t, is then far above its rounding (2^-8 |h||dh| root mean square)."""
    from sca2_b200 import ops
    x, wg, wu, dh = _inputs(257, 64, 136)
    dh = torch.ones_like(dh)
    got = _run(x, wg, wu, dh, "gelu")
    val = lambda *t: float(ops.gated_ffn(*t, act="gelu").double().sum())
    ins = {"dx": x, "dwg": wg, "dwu": wu}
    for k in ins:
        e = got[k].float() / got[k].float().norm()
        t = 0.05 * float(ins[k].float().norm())
        up, dn = ({n: (v.float() + s * t * e).to(H) if n == k else v for n, v in ins.items()} for s in (1, -1))
        step = up[k].double() - dn[k].double()  # what the rounding of the inputs left of it
        num, ana = val(*up.values()) - val(*dn.values()), float((got[k].double() * step).sum())
        assert abs(num - ana) <= 0.03 * abs(ana), (k, num, ana)


def test_streams_and_graphs():
    x, wg, wu, dh = _inputs(900, 256, 384)
    ref = _run(x, wg, wu, dh, "silu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(x, wg, wu, dh, "silu")
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(got[k], ref[k]) for k in ref)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_run(x, wg, wu, dh, "silu"))
        graphs.append(g)
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):  # at the same time
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(o[k], ref[k]) for k in ref)


def test_repeats_bit_for_bit():
    args = _inputs(20000, 256, 256)
    a = _run(*args, "silu")
    for _ in range(3):
        b = _run(*args, "silu")
        assert all(torch.equal(a[k], b[k]) for k in a)


def test_custom_op():
    from sca2_b200 import ops
    x, wg, wu, dh = _inputs(70, 64, 72)
    leaves = [t.detach().requires_grad_(True) for t in (x, wg, wu)]
    torch.library.opcheck(torch.ops.sca2b200.gated_ffn_fwd, (*leaves, 0))
    a = ops.gated_ffn(*leaves)
    b = torch.compile(ops.gated_ffn, fullgraph=True, backend="aot_eager")(*leaves)
    assert torch.equal(a, b)
    for p, q in zip(torch.autograd.grad(a, leaves, dh), torch.autograd.grad(b, leaves, dh)):
        assert torch.equal(p, q)


def test_not_twice_differentiable():
    from sca2_b200 import ops
    x, wg, wu, dh = _inputs(70, 64, 72)
    leaves = [t.detach().requires_grad_(True) for t in (x, wg, wu)]
    ref = _run(x, wg, wu, dh, "silu")
    (g,) = torch.autograd.grad(ops.gated_ffn(*leaves), leaves[:1], dh, create_graph=True)
    assert torch.equal(g, ref["dx"])
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()
