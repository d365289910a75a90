"""The residual join, the gated feed-forward and the clip on tensors whose offsets pass 32 bits: the
far rows equal those of a small call, which the other tests hold against 64 bits.  And a capture
beside a living eager graph of the same memory."""
import pytest
import torch

pytestmark = pytest.mark.gpu
H = torch.bfloat16


def _room(gb):
    if torch.cuda.mem_get_info()[0] < gb << 30:
        pytest.skip(f"needs {gb} GB of device memory")


def _far(rows):
    """Rows around the 2^31st and 2^32nd byte and value of rows of `rows[1]` values, and the last."""
    n, d = rows
    at = [2 ** 31 // d, 2 ** 30 // d, 2 ** 31 // (2 * d), n - 2]
    return sorted({r for a in at for r in range(max(0, a - 2), min(n, a + 2))})


def test_residual_norm():
    from sca2_b200 import ops
    _room(60)
    n, d = 2 ** 31 // 1000 + 5000, 1000
    x = torch.empty(n, d, device="cuda", dtype=H).normal_()
    u = torch.empty(n, d, device="cuda", dtype=H).normal_()
    w, b, s, dz = (torch.randn(d, device="cuda") for _ in range(4))
    rows = _far((n, d))
    xs, us = x.requires_grad_(True), u.requires_grad_(True)
    y, z = ops.residual_norm(xs, us, w, b, scale=s, post_weight=w)
    xr, ur = x.detach()[rows].requires_grad_(True), u.detach()[rows].requires_grad_(True)
    yr, zr = ops.residual_norm(xr, ur, w, b, scale=s, post_weight=w)
    # The small call takes the few-row kernel: the same formulas, sums in another order.  Each result
    # is within 64 x 2^-24 of the size of its terms (below 32 here: normalised values times weights)
    # of the exact value and is then rounded to bf16 by at most 2^-8 of it, so two of them differ by
    # at most twice that.
    near = lambda a, b: bool(((a.float() - b.float()).abs() <= 2 ** -7 * b.float().abs() + 2 * 64 * 2 ** -24 * 32).all())
    assert near(y[rows], yr) and near(z[rows], zr)
    g = dz.to(H).expand(n, d)
    dx, du = torch.autograd.grad(z, (xs, us), g)
    rx, ru = torch.autograd.grad(zr, (xr, ur), g[:len(rows)])
    for got, ref in ((dx[rows], rx), (du[rows], ru)):
        assert float((got.float() - ref.float()).abs().max()) <= 2 ** -7 * float(ref.float().abs().max())


def test_residual_norm_of_any_alignment():
    """As above with odd rows of a wider tensor: the copies of words around each group."""
    from sca2_b200 import ops
    _room(60)
    n, d = 2 ** 31 // 1001 + 5000, 1001
    x = torch.empty(n, d + 6, device="cuda", dtype=H).normal_()[:, 3:3 + d]
    u = torch.empty(n, d, device="cuda", dtype=H).normal_()
    w, s, dz = (torch.randn(d, device="cuda") for _ in range(3))
    rows = _far((n, d))
    xs, us = x.detach().requires_grad_(True), u.requires_grad_(True)
    y, z = ops.residual_norm(xs, us, w, scale=s, kind="rms")
    xr, ur = x[rows].requires_grad_(True), u.detach()[rows].requires_grad_(True)
    yr, zr = ops.residual_norm(xr, ur, w, scale=s, kind="rms")
    # two roundings to bf16 apart, and the sums' order: as above
    near = lambda a, b: bool(((a.float() - b.float()).abs() <= 2 ** -7 * b.float().abs() + 2 * 64 * 2 ** -24 * 32).all())
    assert near(y[rows], yr) and near(z[rows], zr)
    g = dz.to(H).expand(n, d)
    dx, du = torch.autograd.grad(z, (xs, us), g)
    rx, ru = torch.autograd.grad(zr, (xr, ur), g[:len(rows)])
    for got, ref in ((dx[rows], rx), (du[rows], ru)):
        assert float((got.float() - ref.float()).abs().max()) <= 2 ** -7 * float(ref.float().abs().max())


def test_gated_ffn():
    from sca2_b200 import ops
    _room(60)
    n, d, f = 2 ** 31 // 1024 + 3000, 64, 1024
    x = torch.empty(n, d, device="cuda", dtype=H).normal_()
    wg, wu = ((torch.randn(f, d, device="cuda") * d ** -0.5).to(H) for _ in range(2))
    rows = [r for r in _far((n, f))]
    rows = rows + list(range(300 - len(rows)))  # enough for the same kernel
    xs = x.requires_grad_(True)
    h = ops.gated_ffn(xs, wg, wu)
    xr = x.detach()[rows].requires_grad_(True)
    hr = ops.gated_ffn(xr, wg, wu)
    assert torch.equal(h[rows], hr)
    dh = torch.randn(f, device="cuda").to(H)
    (dx,) = torch.autograd.grad(h, xs, dh.expand(n, f))
    (rx,) = torch.autograd.grad(hr, xr, dh.expand(len(rows), f))
    assert torch.equal(dx[rows], rx)


def test_clip():
    from sca2_b200 import ops
    _room(40)
    n = 2 ** 31 + 12345
    g = torch.full((n,), 0.5, device="cuda", dtype=H)
    small = torch.full((100,), 0.25, device="cuda")
    g[-1] = 64.0
    norm = ops.clip_grads([small, g], 1.0)
    ref = (0.25 * (n - 1) + 64.0 ** 2 + 100 * 0.0625) ** 0.5
    assert abs(float(norm) - ref) <= 2 ** -24 * ref
    c = 1.0 / (ref + 1e-6)
    for i, v in ((0, 0.5), (2 ** 31 - 1, 0.5), (2 ** 31 + 1, 0.5), (n - 2, 0.5), (n - 1, 64.0)):
        assert abs(float(g[i]) - v * c) <= 2 ** -8 * v * c + 1e-12
    assert abs(float(small[99]) - 0.25 * c) <= 2 ** -22 * 0.25 * c


def test_capture_beside_an_eager_graph():
    """Forward, backward and clip captured while an eager graph of the same tensors is kept and run
    later.  The captured leaves are detached aliases: autograd ties a leaf's gradient to the stream of
    its first living graph, and a capture that met the eager graph's leaves would be invalid, for any
    operator."""
    from sca2_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)
    leaves = [t.requires_grad_(True) for t in (r(300, 64).to(H), r(72, 64).to(H), r(72, 64).to(H), r(300, 72).to(H), r(72))]
    dz = r(300, 72).to(H)

    def forward(x, wg, wu, u, w):
        return ops.residual_norm(u, ops.gated_ffn(x, wg, wu), w, gate=u)[1]

    eager = forward(*leaves)
    own = [t.detach().requires_grad_(True) for t in leaves]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = torch.autograd.grad(forward(*own), own, dz)
        norm = ops.clip_grads(out, 0.5)
    graph.replay()
    ref = torch.autograd.grad(eager, leaves, dz)
    n = ops.clip_grads(ref, 0.5)
    torch.cuda.synchronize()
    assert torch.equal(norm, n) and all(torch.equal(a, b) for a, b in zip(ref, out))
