"""The residual join with norms (ops.residual_norm) against its definition in 64 bits: outputs and
every gradient over widths on both sides of each kernel variant, types, gates, strides, absent
parts; gradients against differences; empty and single rows; NaN stays in its row; streams, graphs.

Tolerances.  Each fp32 result is a handful of roundings (loads, sigmoid, sums by tree, products) of
2^-24 relative to the terms that make it, so |error| <= K 2^-24 (sum of the terms' sizes) with
K = 64; terms that cancel are counted by size, not by their sum.  A bf16 result adds its own rounding, 2^-8
of the value.  Sums over the rows: the same K over the sum of the terms' sizes, the longest chain
of additions in one thread being rows / 296 <= 40 here."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F, H = torch.float32, torch.bfloat16
K = 64 * 2.0 ** -24


def _inputs(rows, d, xt=F, ut=F, post=True, gate="channel", scale=True, bias=True, z=True, seed=0, pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed + 7 * d + rows)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)
    wide = lambda t, ty: (torch.cat([t, r(rows, pad)], 1) if pad else t).to(ty)[:, :d]  # row stride d + pad
    i = dict(x=wide(2 * r(rows, d) + 0.3, xt), u=wide(r(rows, d) - 0.2, ut))
    i["weight"] = 1 + 0.2 * r(d) if z else None
    i["bias"] = 0.3 * r(d) if z and bias else None
    i["gate"] = {"none": None, "token": r(rows, 1).to(ut), "channel": wide(r(rows, d), ut)}[gate]
    i["scale"] = 0.6 + 0.2 * r(d) if scale else None
    i["post_weight"] = 1 + 0.2 * r(d) if post else None
    i["post_bias"] = 0.3 * r(d) if post and bias else None
    return i, r(rows, d).to(xt), r(rows, d)


def _exact(i, dy, dz, kind, eps=1e-5):
    """Outputs and gradients in 64 bits, and the size of the terms behind each."""
    v = {k: None if t is None else t.detach().double() for k, t in i.items()}
    sizes, out = {}, {}

    def stats(t):
        m = t.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(t[:, :1])
        r = 1 / torch.sqrt((t - m).square().mean(-1, keepdim=True) + eps)
        return m, r

    def back(dn, n, r):
        m = dn.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(dn[:, :1])
        return r * (dn - m - n * (dn * n).mean(-1, keepdim=True))

    def back_size(ds, n, ns, r):  # ds, ns: sizes of dn and n
        return r * (ds + ds.mean(-1, keepdim=True) + ns * (ds * ns).mean(-1, keepdim=True))

    one = torch.ones((), device="cuda", dtype=torch.float64)
    post, has_z = v["post_weight"] is not None, v["weight"] is not None
    um, ur = stats(v["u"])
    un = (v["u"] - um) * ur if post else v["u"]
    uns = (v["u"].abs() + um.abs()) * ur if post else v["u"].abs()
    pw = v["post_weight"] if post else one
    pb = v["post_bias"] if v["post_bias"] is not None else 0 * one
    p, ps = un * pw + pb, uns * pw.abs() + pb.abs()
    s = torch.sigmoid(v["gate"]) if v["gate"] is not None else one
    sc = v["scale"] if v["scale"] is not None else one
    y = v["x"] + sc * s * p
    ys = v["x"].abs() + sc.abs() * s * ps
    out["y"], sizes["y"] = y, ys
    dyy = dy.double() if dy is not None else torch.zeros_like(y)
    dys = dyy.abs()
    if has_z:
        ym, yr = stats(y)
        yn, yns = (y - ym) * yr, (ys + ys.mean(-1, keepdim=True)) * yr
        b = v["bias"] if v["bias"] is not None else 0 * one
        out["z"], sizes["z"] = yn * v["weight"] + b, yns * v["weight"].abs() + b.abs()
        d = dz.double() if dz is not None else torch.zeros_like(y)
        dn = d * v["weight"]
        dyy = dyy + back(dn, yn, yr)
        # an error of the normalised row is one of its size; it enters the product sums as such
        dys = dys + back_size(dn.abs(), yn, yns, yr)
        out["weight"], sizes["weight"] = (d * yn).sum(0), (d.abs() * yns).sum(0)
        out["bias"], sizes["bias"] = d.sum(0), d.abs().sum(0)
    out["x"], sizes["x"] = dyy, dys
    dp, dps = dyy * sc * s, dys * sc.abs() * s
    if post:
        out["u"], sizes["u"] = back(dp * pw, un, ur), back_size(dps * pw.abs(), un, uns, ur)
    else:
        out["u"], sizes["u"] = dp, dps
    out["post_weight"], sizes["post_weight"] = (dp * un).sum(0), (dps * uns).sum(0)
    out["post_bias"], sizes["post_bias"] = dp.sum(0), dps.sum(0)
    out["scale"], sizes["scale"] = (dyy * s * p).sum(0), (dys * s * ps).sum(0)
    if v["gate"] is not None:
        dg, dgs = dyy * sc * p * s * (1 - s), dys * sc.abs() * ps * s
        if v["gate"].shape[-1] == 1 and y.shape[-1] != 1:
            dg, dgs = dg.sum(-1, keepdim=True), dgs.sum(-1, keepdim=True)
        out["gate"], sizes["gate"] = dg, dgs
    return out, sizes


def _near(name, got, ref, size):
    tol = K * size + (2.0 ** -8 * ref.abs() if got.dtype == H else 0)
    bad = (got.double() - ref).abs() > tol
    assert not bool(bad.any()) and bool(torch.isfinite(got).all()), \
        f"{name}: {int(bad.sum())} values off, largest {float(((got.double() - ref).abs() / (tol + 1e-300)).max())} of the tolerance"


def _check(i, dy, dz, kind="layer", zt=None, use=("y", "z")):
    from sca2_b200 import ops
    for t in i.values():
        if t is not None:
            t.requires_grad_(True)
    y, z = ops.residual_norm(i["x"], i["u"], i["weight"], i["bias"], gate=i["gate"], scale=i["scale"],
                             post_weight=i["post_weight"], post_bias=i["post_bias"], kind=kind, out_dtype=zt)
    assert y.dtype == i["x"].dtype and y.shape == i["x"].shape and (z is None) == (i["weight"] is None)
    dy = dy if "y" in use else None
    dz = dz.to(z.dtype) if z is not None and "z" in use else None
    outs = [(o, g) for o, g in ((y, dy), (z, dz)) if g is not None]
    keys = [k for k, t in i.items() if t is not None]
    grads = torch.autograd.grad([o for o, _ in outs], [i[k] for k in keys], [g for _, g in outs], allow_unused=True)
    ref, size = _exact(i, dy, dz, kind)
    _near("y", y.detach(), ref["y"], size["y"])
    if z is not None:
        assert z.dtype == (zt or i["x"].dtype)
        _near("z", z.detach(), ref["z"], size["z"])
    for k, g in zip(keys, grads):
        assert g.dtype == i[k].dtype and g.shape == i[k].shape
        _near("d" + k, g, ref[k], size[k])
    with torch.no_grad():  # without gradients: the same values
        y2, z2 = ops.residual_norm(i["x"], i["u"], i["weight"], i["bias"], gate=i["gate"], scale=i["scale"],
                                   post_weight=i["post_weight"], post_bias=i["post_bias"], kind=kind, out_dtype=zt)
    assert torch.equal(y, y2) and (z is None or torch.equal(z, z2))


@pytest.mark.parametrize("rows,d", [(1, 1), (3, 2), (5, 7), (9, 8), (2, 128), (37, 256), (33, 264), (7, 768), (5, 1001),
                                    (6, 1024), (11, 1028), (4, 1032), (5, 2048), (3, 2049), (3, 2052), (2, 4095), (3, 4096)])
@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_widths(rows, d, kind):
    _check(*_inputs(rows, d, bias=kind == "layer"), kind=kind)


@pytest.mark.parametrize("rows", [383, 384, 1184, 1185, 1331, 1332, 3071, 3073, 5000])
@pytest.mark.parametrize("d", [96, 333, 768, 1536])
def test_many_rows(rows, d):
    _check(*_inputs(rows, d, F, H), zt=H)


@pytest.mark.parametrize("rows,d", [(2047, 1028), (2048, 1028), (2100, 2048), (2101, 2052), (2050, 4096), (2049, 2501)])
@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_many_wide_rows(rows, d, kind):
    _check(*_inputs(rows, d, F, H, bias=kind == "layer"), kind=kind, zt=H)
    _check(*_inputs(rows, d, bias=kind == "layer"), kind=kind)


@pytest.mark.parametrize("d", [1, 2, 3, 5, 33, 130, 515, 770, 1023, 1025, 2049, 3001, 4093])
@pytest.mark.parametrize("xt,ut", [(F, H), (H, F), (H, H)])
def test_many_rows_of_any_alignment(d, xt, ut):
    """Rows that begin anywhere: odd widths, and (tensors shifted by a value, odd row strides) odd places."""
    rows = 1300 if d <= 515 else max(2050, min(4 * d, 4100))
    i, dy, dz = _inputs(rows, d, xt, ut)
    _check(i, dy, dz, zt=ut)
    if d in (5, 130, 770, 1025):
        off = lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)
        _check({n: off(t.detach()) for n, t in i.items()}, dy, dz, kind="layer", zt=xt)
        i, dy, dz = _inputs(rows, d, xt, ut, pad=3)
        _check(i, dy, dz)


@pytest.mark.parametrize("rows,d", [(1300, 136), (1300, 135), (2050, 1100), (2050, 1101)])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("gate", ["none", "token", "channel"])
@pytest.mark.parametrize("scale", [False, True])
@pytest.mark.parametrize("z", [False, True])
def test_options_of_many_rows(rows, d, post, gate, scale, z):
    i, dy, dz = _inputs(rows, d, H if scale else F, H, post, gate, scale, True, z)
    _check(i, dy, dz, use=("z",) if z and not post else ("y", "z"))


@pytest.mark.parametrize("xt", [F, H])
@pytest.mark.parametrize("ut", [F, H])
@pytest.mark.parametrize("zt", [F, H])
@pytest.mark.parametrize("rows,d", [(50, 64), (50, 75), (1250, 64), (1250, 300), (2060, 1056)])
def test_types(xt, ut, zt, rows, d):
    _check(*_inputs(rows, d, xt, ut), zt=zt)


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("gate", ["none", "token", "channel"])
@pytest.mark.parametrize("scale", [False, True])
@pytest.mark.parametrize("z", [False, True])
@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_options(post, gate, scale, z, kind):
    i, dy, dz = _inputs(21, 136, F, H, post, gate, scale, kind == "layer", z)
    _check(i, dy, dz, kind=kind)


@pytest.mark.parametrize("use", [("y",), ("z",)])
def test_one_output_used(use):
    _check(*_inputs(13, 264), use=use)


@pytest.mark.parametrize("pad", [1, 4, 8])
@pytest.mark.parametrize("d", [136, 75])
def test_strided_rows(pad, d):
    _check(*_inputs(40, d, H, H, pad=pad))


def test_shapes_and_views():
    from sca2_b200 import ops
    i, _, _ = _inputs(24, 64)
    ref = ops.residual_norm(i["x"], i["u"], i["weight"], i["bias"], gate=i["gate"])
    v = lambda t: t.view(2, 3, 4, 64)
    y, z = ops.residual_norm(v(i["x"]), v(i["u"]), i["weight"], i["bias"], gate=v(i["gate"]))
    assert torch.equal(y.view(24, 64), ref[0]) and torch.equal(z.view(24, 64), ref[1])
    # rows that one stride does not describe, a transposed tensor, a broadcast one, halves of one
    # projection, one row without a leading dimension
    t = lambda x: x.view(4, 6, 64).transpose(0, 1)
    y, z = ops.residual_norm(t(i["x"]), t(i["u"]), i["weight"], i["bias"], gate=t(i["gate"]))
    assert torch.equal(y, t(ref[0])) and torch.equal(z, t(ref[1]))
    c = lambda x: x.t().contiguous().t()
    y, z = ops.residual_norm(c(i["x"]), c(i["u"]), i["weight"], i["bias"], gate=c(i["gate"]))
    assert torch.equal(y, ref[0]) and torch.equal(z, ref[1])
    both = torch.cat([i["u"], i["gate"]], 1)
    u, g = both.chunk(2, 1)
    y, z = ops.residual_norm(i["x"], u, i["weight"], i["bias"], gate=g)
    assert torch.equal(y, ref[0]) and torch.equal(z, ref[1])
    y, z = ops.residual_norm(i["x"][:1].expand(24, 64), i["u"], i["weight"])
    y1, z1 = ops.residual_norm(i["x"][:1].repeat(24, 1), i["u"], i["weight"])
    assert torch.equal(y, y1) and torch.equal(z, z1)
    y, z = ops.residual_norm(i["x"][0], i["u"][0], i["weight"], i["bias"], gate=i["gate"][0])
    assert torch.equal(y, ref[0][0]) and torch.equal(z, ref[1][0])


def test_weights_off_alignment():
    """Parameters and rows that begin between 16-byte boundaries take the scalar kernels."""
    from sca2_b200 import ops
    i, dy, dz = _inputs(20, 128)
    off = lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)
    for k in i:
        _check({n: (off(t.detach()) if n == k else t.detach().clone()) for n, t in i.items()}, dy, dz)


def test_no_rows():
    from sca2_b200 import ops
    w = torch.ones(64, device="cuda", requires_grad=True)
    x = torch.zeros(2, 0, 64, device="cuda", requires_grad=True)
    y, z = ops.residual_norm(x, x, w, post_weight=w, gate=torch.zeros(2, 0, 1, device="cuda"), scale=w)
    assert y.shape == z.shape == (2, 0, 64)
    (y.sum() + z.sum()).backward()
    assert torch.equal(w.grad, torch.zeros_like(w)) and x.grad.shape == x.shape


def test_nan_and_inf_stay_in_their_row():
    from sca2_b200 import ops
    i, dy, dz = _inputs(40, 264)
    clean = ops.residual_norm(i["x"], i["u"], i["weight"], i["bias"], gate=i["gate"], post_weight=i["post_weight"])
    i["u"][7, 3], i["x"][11, 200] = float("nan"), float("inf")
    keep = [r for r in range(40) if r not in (7, 11)]
    x = i["x"].clone().requires_grad_(True)
    y, z = ops.residual_norm(x, i["u"], i["weight"], i["bias"], gate=i["gate"], post_weight=i["post_weight"])
    assert torch.equal(y[keep], clean[0][keep]) and torch.equal(z[keep], clean[1][keep])
    assert not torch.isfinite(z[7]).any() and not torch.isfinite(z[11]).all()
    (dx,) = torch.autograd.grad((y, z), x, (dy, dz))
    assert torch.isfinite(dx[keep]).all()


def test_gate_extremes():
    """Logits of the type's lowest value, infinities: the gate is 0 or 1 and its gradient 0."""
    from sca2_b200 import ops
    i, dy, dz = _inputs(4, 64, gate="token", post=False)
    i["gate"] = torch.tensor([[-math.inf], [torch.finfo(F).min], [math.inf], [torch.finfo(F).max]], device="cuda",
                             requires_grad=True)
    y, _ = ops.residual_norm(i["x"], i["u"], gate=i["gate"])
    assert torch.equal(y[:2], i["x"][:2]) and torch.equal(y[2:], (i["x"] + i["u"])[2:])
    (g,) = torch.autograd.grad(y, i["gate"], dy)
    assert torch.equal(g, torch.zeros_like(g))


def test_gradient_against_differences():
    """Central differences of sum(y dy + z dz) along random directions, step h = 2^-7: the formula's
    error is O(h^2) third derivatives, so the ratio is good to a percent; the sums' fp32 rounding
    (about 1e-6 of sums of size 100) divided by 2h stays below that too."""
    from sca2_b200 import ops
    i, dy, dz = _inputs(6, 96)
    keys = [k for k in i]
    run = lambda v: ops.residual_norm(v["x"], v["u"], v["weight"], v["bias"], gate=v["gate"], scale=v["scale"],
                                      post_weight=v["post_weight"], post_bias=v["post_bias"])
    val = lambda v: sum(float((o.double() * g.double()).sum()) for o, g in zip(run(v), (dy, dz)))
    leaves = {k: t.clone().requires_grad_(True) for k, t in i.items()}
    grads = torch.autograd.grad(run(leaves), [leaves[k] for k in keys], (dy, dz))
    g = torch.Generator(device="cuda").manual_seed(3)
    h = 2.0 ** -7
    for k, gr in zip(keys, grads):
        e = torch.randn(i[k].shape, device="cuda", generator=g)
        e = e + 2 * torch.sign((e * gr).sum()) * gr / gr.norm() * e.norm()  # a direction along which it moves
        e = e / e.norm() * i[k].norm() * 0.1
        up, dn = ({**i, k: i[k] + s * h * e} for s in (1, -1))
        num, ana = (val(up) - val(dn)) / (2 * h), float((gr.double() * e.double()).sum())
        assert abs(num - ana) <= 0.01 * abs(ana) + 1e-3, (k, num, ana)


def test_streams_and_graph():
    from sca2_b200 import ops
    i, dy, dz = _inputs(300, 768, F, H)
    names = [k for k, t in i.items() if t is not None]

    def step(v):
        y, z = ops.residual_norm(v["x"], v["u"], v["weight"], v["bias"], gate=v["gate"], scale=v["scale"],
                                 post_weight=v["post_weight"], post_bias=v["post_bias"])
        return (y.detach(), z.detach(), *torch.autograd.grad((y, z), [v[k] for k in names], (dy, dz)))

    ref = step({k: t.clone().requires_grad_(True) for k, t in i.items()})
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step({k: t.clone().requires_grad_(True) for k, t in i.items()})
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(ref, got):
        assert torch.equal(a, b)
    # two graphs of one call on the same leaves, replayed together: no workspace is shared
    leaves = {k: torch.zeros_like(t).copy_(t).requires_grad_(True) for k, t in i.items()}
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(leaves))
        graphs.append(g)
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
    torch.cuda.synchronize()
    for out in outs:
        for a, b in zip(ref, out):
            assert torch.equal(a, b)


def test_repeats_bit_for_bit():
    from sca2_b200 import ops
    i, dy, dz = _inputs(5000, 768, F, H)
    for t in i.values():
        t.requires_grad_(True)
    runs = []
    for _ in range(3):
        o = ops.residual_norm(i["x"], i["u"], i["weight"], i["bias"], gate=i["gate"], scale=i["scale"],
                              post_weight=i["post_weight"], post_bias=i["post_bias"])
        runs.append(torch.autograd.grad(o, list(i.values()), (dy, dz)))
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], r))


def test_custom_op():
    i, dy, dz = _inputs(6, 40)
    ins = [None if t is None else t.requires_grad_(True) for t in
           (i["x"], i["u"], i["weight"], i["bias"], i["gate"], i["scale"], i["post_weight"], i["post_bias"])]
    torch.library.opcheck(torch.ops.sca2b200.residual_norm_fwd, (*ins, 0, 1e-5, F, True))
    from sca2_b200 import ops
    f = lambda x, u: ops.residual_norm(x, u, i["weight"], i["bias"], gate=i["gate"])[1]
    x, u = i["x"].detach().requires_grad_(True), i["u"].detach().requires_grad_(True)
    a, b = f(x, u), torch.compile(f, fullgraph=True, backend="aot_eager")(x, u)
    assert torch.equal(a, b)
    for p, q in zip(torch.autograd.grad(a, (x, u), dz), torch.autograd.grad(b, (x, u), dz)):
        assert torch.equal(p, q)


def test_not_twice_differentiable():
    from sca2_b200 import ops
    i, dy, dz = _inputs(6, 40)
    x = i["x"].requires_grad_(True)
    y, z = ops.residual_norm(x, i["u"], i["weight"])
    (g,) = torch.autograd.grad((y, z), x, (dy, dz), create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()
