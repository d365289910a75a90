"""The residual join of a block's tail (layers.ResidualJoin) where its kernel does not reach: types
beside fp32 and bf16, rows wider than 4096 values, tensors on the CPU.  Against the definition in 64
bits; the fp32 arithmetic is a handful of roundings of 2^-24 of terms below 32 in size, and a result
of 16 bits adds its own rounding."""
import pytest
import torch
import torch.nn.functional as F

from sca2_b200 import layers

TAILS = [dict(post_norm=True), dict(gate="token"), dict(gate="channel", res_scale=0.3),
         dict(post_norm=True, gate="channel", res_scale=0.5)]


def make(d, tail, dtype, device="cpu"):
    torch.manual_seed(d)
    join, norm = layers.ResidualJoin(d, layers.TailCfg(**tail), 1e-5), layers.LayerNorm(d)
    with torch.no_grad():
        for p in (*join.parameters(), *norm.parameters()):
            p.add_(0.05 * torch.randn_like(p))
        if join.gate is not None:
            join.gate.weight.mul_(d ** -0.5)
    return join.to(device, dtype), norm.to(device, dtype)


def exact(join, norm, x, u, g, with_norm=True):
    """y and z in 64 bits; g: the gate's logits or None."""
    w = lambda t: None if t is None else t.detach().double()
    x, u, g = w(x), w(u), w(g)
    if join.norm is not None:
        u = F.layer_norm(u, u.shape[-1:], w(join.norm.weight), w(join.norm.bias), 1e-5)
    if join.scale is not None:
        u = u * w(join.scale)
    if g is not None:
        u = u * torch.sigmoid(g)
    y = x + u
    return y, F.layer_norm(y, y.shape[-1:], w(norm.weight), w(norm.bias), 1e-5) if with_norm else None


def check(join, norm, x, u, zin, out_dtype):
    got = {}
    if join.gate is not None:
        join.gate.register_forward_hook(lambda m, i, o: got.__setitem__("g", o))
    y, z = join(x, u, zin, norm)
    ry, rz = exact(join, norm, x, u, got.get("g"))
    assert y.dtype == x.dtype and z.dtype == out_dtype
    for o, r in ((y, ry), (z, rz)):
        own = torch.finfo(o.dtype).eps / 2 if o.dtype != torch.float64 else 0
        work = 64 * 2.0 ** -24 * 32 if o.dtype != torch.float64 else 1e-12
        assert bool(((o.double() - r).abs() <= own * r.abs() + work).all())
    assert join(x, u, zin)[1] is None
    return y, z


@pytest.mark.parametrize("tail", TAILS, ids=lambda t: "-".join(t))
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.float16, torch.bfloat16])
def test_join_on_the_cpu(tail, dtype):
    join, norm = make(24, tail, dtype)
    r = lambda: torch.randn(2, 5, 24).to(dtype)
    x = r().requires_grad_(True)
    y, z = check(join, norm, x, r(), r(), dtype)
    z.float().sum().backward()
    assert bool(torch.isfinite(x.grad).all()) and all(p.grad is not None for p in join.parameters())


def test_gradients_against_differences():
    join, norm = make(12, TAILS[-1], torch.float64)
    x, u, z = (torch.randn(3, 12, dtype=torch.float64, requires_grad=True) for _ in range(3))
    assert torch.autograd.gradcheck(lambda *a: join(*a, norm), (x, u, z))
