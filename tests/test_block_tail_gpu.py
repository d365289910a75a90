"""The block's tail with its options (layers.TailCfg: gated FFN, norms after the branches, gates,
residual scales) as the layers and the language model run it: one layer's output and the gradients
of every tail parameter against 64 bits, decode steps against the prefill, the whole-stack graph
decoder, and training steps with clipping.

Tolerances.  fp32: TOL_F32 of the largest value, as for the layers (the products are cuBLAS's).  Under
bf16 autocast the reference runs in 64 bits on the kernel's own branch output; each of its chained
products (gate logits, the three FFN products) rounds operands and result by 2^-8 at most and the sums over d or ff
average them: the bar is the repository's 2e-2 of the largest value."""
import pytest
import torch
import torch.nn.functional as F

from tests._util import TOL_BF16_ABS, TOL_F32, relerr

pytestmark = pytest.mark.gpu
TAILS = [dict(ffn_act="silu"), dict(post_norm=True), dict(gate="token"), dict(gate="channel", res_scale=0.3),
         dict(ffn_act="gelu", post_norm=True, gate="token", res_scale=0.5),
         dict(ffn_act="silu", post_norm=True, gate="channel", res_scale=0.5)]


def _cfg(tail, d=64, ff=128):
    from sca2_b200 import layers
    return layers.LayerCfg(d=d, Mc=32, Md=4, G=8, ff=ff, freq="rope", theta_scale=0.02, max_len=256, dv=64,
                           c_heads=1, c_decay=True, tail=layers.TailCfg(**tail))


def _layer(tail):
    from sca2_b200 import layers
    torch.manual_seed(5)
    layer = layers.GatedLayer(_cfg(tail)).cuda()
    with torch.no_grad():
        for p in layer.parameters():
            p.add_(0.05 * torch.randn_like(p))
    return layer


def _tail64(layer, x, z, m, p):
    """The tail in 64 bits from the residual stream, its norm and the mixed branch; p: parameters."""
    ln = lambda t, n: F.layer_norm(t, t.shape[-1:], p[n + ".weight"], p[n + ".bias"], 1e-5)

    def join(x, u, z, n):
        if n + ".norm.weight" in p:
            u = ln(u, n + ".norm")
        if n + ".gate.weight" in p:
            u = u * torch.sigmoid(F.linear(z, p[n + ".gate.weight"], p[n + ".gate.bias"]))
        return x + u * p[n + ".scale"] if n + ".scale" in p else x + u

    y = join(x, m, z, "join1")
    f = ln(y, "fn")
    if "ff.up.weight" in p:
        act = F.silu if layer.ff.act == "silu" else F.gelu
        w = F.linear(act(F.linear(f, p["ff.gate.weight"])) * F.linear(f, p["ff.up.weight"]), p["ff.down.weight"])
    else:
        w = F.linear(F.gelu(F.linear(f, p["ff.0.weight"], p["ff.0.bias"])), p["ff.2.weight"], p["ff.2.bias"])
    return join(y, w, f, "join2")


@pytest.mark.parametrize("tail", TAILS, ids=lambda t: "-".join(f"{k}={v}" for k, v in t.items()))
@pytest.mark.parametrize("autocast", [False, True])
def test_layer_tail(tail, autocast):
    layer = _layer(tail)
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(2, 150, 64, device="cuda", generator=g)
    dy = torch.randn(2, 150, 64, device="cuda", generator=g)
    kept = {}
    layer.mix.register_forward_hook(lambda m, i, o: kept.__setitem__("m", o.detach()))
    layer.n.register_forward_hook(lambda m, i, o: kept.__setitem__("z", o.detach()))
    with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
        y = layer(x)
    y.backward(dy)
    names = [n for n, _ in layer.named_parameters() if n.split(".")[0] in ("fn", "ff", "join1", "join2")]
    p = {n: q.detach().double().requires_grad_(True) for n, q in layer.named_parameters()}
    ref = _tail64(layer, x.double(), kept["z"].double(), kept["m"].double(), p)
    grads = torch.autograd.grad(ref, [p[n] for n in names], dy.double())
    tol = TOL_BF16_ABS if autocast else TOL_F32
    assert relerr(y, ref) < tol
    for n, r in zip(names, grads):
        assert relerr(dict(layer.named_parameters())[n].grad, r) < tol, n


def test_without_options_nothing_changes():
    from sca2_b200 import layers
    torch.manual_seed(1)
    a = layers.GatedLayer(_cfg({})).cuda()
    torch.manual_seed(1)
    cfg = _cfg({})
    cfg.tail = None
    b = layers.GatedLayer(cfg).cuda()
    assert a.state_dict().keys() == b.state_dict().keys()
    x = torch.randn(1, 40, 64, device="cuda")
    assert torch.equal(a(x), b(x))


def _lm(kind, tail):
    from sca2_b200 import layers, lm as L
    torch.manual_seed(3)
    if kind == "gated":
        m = L.GatedLM(128, _cfg(tail), n_layers=2).cuda()
    else:
        m = L.LaplaceLM(128, d=64, n_layers=2, tail=layers.TailCfg(**tail), M=12, dv=8, L=8, ff=128, chunk=16,
                        theta_scale=0.3).cuda()
    L.init_weights(m, 0.1)
    return m


@pytest.mark.parametrize("kind", ["gated", "lapa"])
def test_decode(kind):
    """Steps after a prompt give the prefill's logits, and the graph decoder the steps' tokens."""
    from sca2_b200 import lm as L
    m = _lm(kind, TAILS[-1]).eval()
    tok = torch.randint(0, 128, (3, 24), device="cuda", generator=torch.Generator(device="cuda").manual_seed(4))
    with torch.no_grad():
        full = m(tok)
        logits, st = m.prefill(tok[:, :16])
        assert relerr(logits, full[:, :16]) < TOL_F32
        for t in range(16, 24):
            step, st = m.step(tok[:, t], st)
            assert relerr(step, full[:, t]) < 2 * TOL_F32
        first = full[:, -1].argmax(-1)
        got = L.GraphDecoder(m, st).generate(first, 6)
        want, t = [], first
        for _ in range(6):
            lg, st = m.step(t, st)
            t = lg.argmax(-1)
            want.append(t)
    assert torch.equal(got, torch.stack(want, 1))
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16, cache_enabled=False):
        lg, st = m.prefill(tok)
        out = L.GraphDecoder(m, st).generate(first, 3)  # the decode kernels inside a graph
        assert out.shape == (3, 3) and int(out.min()) >= 0 and int(out.max()) < 128


@pytest.mark.parametrize("kind", ["gated", "lapa"])
def test_training_steps(kind):
    """Steps run with clipping: every gradient is there, finite, and of the asked norm; and a step's
    weights are those of the same step made by hand."""
    from sca2_b200 import lm as L, ops
    m = _lm(kind, TAILS[-1])
    tok = L.zipf_tokens(2, 65, 128, seed=6, device="cuda")
    opt = torch.optim.SGD(m.parameters(), lr=0.5)
    for _ in range(3):
        before = [p.detach().clone() for p in m.parameters()]
        loss = L.train_step(m, opt, tok, max_norm=0.1)
        assert bool(torch.isfinite(loss))
        # plain SGD: the step is lr x the clipped gradient
        delta = torch.stack([(a.double() - p.detach().double()).square().sum() for a, p in zip(before, m.parameters())])
        assert abs(float(delta.sum().sqrt()) / 0.5 - 0.1) < 1e-4
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = L.lm_loss(m, tok)
    loss.backward()
    missing = [n for n, p in m.named_parameters() if p.grad is None]
    assert not [n for n in missing if n.split(".")[2:3] and n.split(".")[2] in ("fn", "ff", "join1", "join2")], missing
    grads = [p.grad for p in m.parameters() if p.grad is not None]
    assert all(bool(torch.isfinite(g).all()) for g in grads)
    ops.clip_grads(grads, 1e-3)
    assert abs(float(ops.grad_norm(grads)) - 1e-3) < 1e-6


def test_training_step_in_a_graph():
    """The tail, its backward and the clip captured together, while an eager step's graph of the
    same leaves exists; replays give the eager gradients."""
    from sca2_b200 import layers, ops
    torch.manual_seed(7)
    ffn, join = layers.GatedFFN(64, 128).cuda().bfloat16(), layers.ResidualJoin(64, layers.TailCfg(post_norm=True, gate="channel", res_scale=0.5), 1e-5).cuda().bfloat16()
    ps = [*ffn.parameters(), *join.parameters()]
    x = torch.randn(300, 64, device="cuda").bfloat16()

    def step():
        y, _ = join(x, ffn(x), x)
        grads = torch.autograd.grad(y, ps, torch.ones_like(y))
        return (*grads, ops.clip_grads(grads, 0.5))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ref = step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for _ in range(2):
        g.replay()
    torch.cuda.synchronize()
    for a, b in zip(ref, out):
        assert torch.equal(a, b)


def test_vmap():
    """Batched by torch.func.vmap: the registered operators, one call for each."""
    from sca2_b200 import ops
    torch.manual_seed(8)
    x, u, w = torch.randn(3, 5, 64, device="cuda"), torch.randn(3, 5, 64, device="cuda"), torch.randn(64, device="cuda")
    y, z = torch.func.vmap(lambda x, u: ops.residual_norm(x, u, w))(x, u)
    ry, rz = ops.residual_norm(x, u, w)
    assert torch.equal(y, ry) and torch.equal(z, rz)
    xh, wh = x.bfloat16(), torch.randn(2, 32, 64, device="cuda").bfloat16()
    assert torch.equal(torch.func.vmap(lambda x: ops.gated_ffn(x, wh[0], wh[1]))(xh), ops.gated_ffn(xh, wh[0], wh[1]))
