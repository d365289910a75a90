"""The operators of a residual block's tail and of a training step, as they are measured.

Three operators of `sca2_b200.ops`, each with its plain form in elementary torch operations:

  gated_ffn       h = act(x Wg^T) * (x Wu^T), the two projections of a gated feed-forward block
                  with the activation and the product, and its gradients
  residual_norm   y = x + scale * sigmoid(gate) * norm_post(u), z = norm(y): the residual join
                  after a block with the norms on both of its sides, and its gradients
  clip_grads      the global 2-norm of a list of gradients, and the gradients scaled so that it
                  is at most max_norm

A case is one call with its sizes; `train` cases return the outputs and every gradient.
"""
import math

import torch

own = False

DEV = "cuda"
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------------
#  cases
# ------------------------------------------------------------------------------------------
def listed():
    return [
        # one new token through one block of the 12-layer, d = 768 language model
        dict(name="ffn_token", op="ffn", rows=1, d=768, f=2048, act="silu", train=False),
        # a decode batch of 64 sequences, d = 1024, width 8/3 d rounded to 16
        dict(name="ffn_decode", op="ffn", rows=64, d=1024, f=2736, act="gelu", train=False),
        # a small ragged batch: no size is a multiple of a tile
        dict(name="ffn_ragged", op="ffn", rows=1003, d=520, f=1096, act="gelu", train=True),
        # a prompt batch of 8 x 4096 tokens through the d = 1024 layer, no gradients
        dict(name="ffn_prompt", op="ffn", rows=32768, d=1024, f=4096, act="silu", train=False),
        # one block of the language model's training step, 32 x 2048 tokens
        dict(name="ffn_train", op="ffn", rows=65536, d=768, f=2048, act="silu", train=True),
        # the joins of one decode step, 64 sequences, bf16 block output on an fp32 residual stream
        dict(name="norm_step", op="norm", rows=64, d=768, kind="layer", x="f32", u="bf16", z="bf16", post=True,
             gate="channel", scale=True, train=False),
        # the language model's training step under bf16 autocast: everything on
        dict(name="norm_train", op="norm", rows=65536, d=768, kind="layer", x="f32", u="bf16", z="bf16", post=True,
             gate="channel", scale=True, train=True),
        # an odd width and row count, bf16 throughout, RMS norms, one gate for each token
        dict(name="norm_odd", op="norm", rows=4099, d=1001, kind="rms", x="bf16", u="bf16", z="bf16", post=True,
             gate="token", scale=False, train=True),
        # a prompt batch in fp32, the plain pre-norm join with a residual scale
        dict(name="norm_prompt", op="norm", rows=32768, d=1024, kind="layer", x="f32", u="f32", z="f32", post=False,
             gate="none", scale=True, train=False),
        # a 4-layer, d = 128 model: latency
        dict(name="clip_small", op="clip", layers=4, d=128, f=256, vocab=256, low=0, pad=8, max_norm=1.0),
        # the 12-layer, d = 768 language model, fp32 gradients of fp32 master weights
        dict(name="clip_lm", op="clip", layers=12, d=768, f=2048, vocab=16384, low=0, pad=8, max_norm=1.0),
        # bf16 and fp32 gradients mixed, odd sizes, destinations packed without padding
        dict(name="clip_ragged", op="clip", layers=7, d=333, f=901, vocab=5003, low=2, pad=1, max_norm=0.5),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["ffn", "ffn", "norm", "norm", "clip"])
    if op == "ffn":
        d, f = 8 * _log_int(rng, 8, 192), 8 * _log_int(rng, 8, 512)
        train = rng.random() < 0.5
        # at most the work of the largest listed case (12 x 65536 x 768 x 2048 operations)
        most = int(65536 * 768 * 2048 * (1 if train else 3) / (d * f))
        return dict(op="ffn", rows=_log_int(rng, 1, max(1, min(65536, most))), d=d, f=f,
                    act=rng.choice(["silu", "gelu"]), train=train)
    if op == "norm":
        d = _log_int(rng, 32, 4096)
        d = d if rng.random() < 0.3 else (d + 7) // 8 * 8
        train = rng.random() < 0.5
        most = int(65536 * 768 / d)
        return dict(op="norm", rows=_log_int(rng, 1, max(1, most)), d=d, kind=rng.choice(["layer", "rms"]),
                    x=rng.choice(["f32", "bf16"]), u=rng.choice(["f32", "bf16"]), z=rng.choice(["f32", "bf16"]),
                    post=rng.random() < 0.5, gate=rng.choice(["none", "token", "channel"]),
                    scale=rng.random() < 0.5, train=train)
    return dict(op="clip", layers=rng.randint(1, 12), d=_log_int(rng, 33, 768), f=_log_int(rng, 65, 2048),
                vocab=_log_int(rng, 100, 16384), low=rng.choice([0, 1, 2, 3]), pad=rng.choice([1, 8]),
                max_norm=rng.choice([0.5, 1.0, 1e9]))


def _clip_shapes(c):
    """(shape, type) of the gradients: an embedding, then for each layer two norms, four square
    projections and a gated feed-forward block.  Every `low`-th tensor is bf16 (0: none)."""
    d, f = c["d"], c["f"]
    block = [(d,), (d,), (d, d), (d, d), (d, d), (d, d), (d,), (d,), (f, d), (f, d), (d, f)]
    shapes = [(c["vocab"], d)] + block * c["layers"]
    return [(s, "bf16" if c["low"] and i % c["low"] == c["low"] - 1 else "f32") for i, s in enumerate(shapes)]


def work(c):
    if c["op"] == "ffn":
        n, d, f = c["rows"], c["d"], c["f"]
        by, fl = 2 * (n * d + 2 * f * d + n * f), 4 * n * d * f
        if c["train"]:  # dh in; dx and both weight gradients out; two products of each kind
            by, fl = by + 2 * (n * f + n * d + 2 * f * d), 3 * fl
        return {"bytes": by, "flops": fl}
    if c["op"] == "norm":
        n, d = c["rows"], c["d"]
        sz = {"f32": 4, "bf16": 2}
        gate = {"none": 0, "token": n, "channel": n * d}[c["gate"]] * sz[c["u"]]
        params = 4 * d * ((2 if c["kind"] == "layer" else 1) * (2 if c["post"] else 1) + (1 if c["scale"] else 0))
        by = n * d * (2 * sz[c["x"]] + sz[c["u"]] + sz[c["z"]]) + gate + params
        fl = 16 * n * d
        if c["train"]:  # dy, dz in; dx, du, dgate and the parameters' gradients out
            by, fl = by + n * d * (2 * sz[c["x"]] + sz[c["u"]] + sz[c["z"]]) + gate + params, 3 * fl
        return {"bytes": by, "flops": fl}
    by = fl = 0
    for shape, t in _clip_shapes(c):
        n = math.prod(shape)
        by, fl = by + n * ((4 if t == "f32" else 2) + 4), fl + 3 * n
    return {"bytes": by, "flops": fl}


# ------------------------------------------------------------------------------------------
#  inputs
# ------------------------------------------------------------------------------------------
def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    randn = lambda *s: torch.randn(*s, device=DEV, generator=g)  # noqa: E731
    s = {"c": c}
    if c["op"] == "ffn":
        n, d, f = c["rows"], c["d"], c["f"]
        # x: a normed residual stream; weights: the language model's N(0, 0.02^2) widened so that
        # the pre-activations have unit size whatever the width
        s["x"] = randn(n, d).bfloat16()
        s["wg"] = (randn(f, d) * d ** -0.5).bfloat16()
        s["wu"] = (randn(f, d) * d ** -0.5).bfloat16()
        if c["train"]:
            s["dh"] = randn(n, f).bfloat16()
            for k in ("x", "wg", "wu"):
                s[k].requires_grad_(True)
        return s
    if c["op"] == "norm":
        n, d = c["rows"], c["d"]
        # a residual stream with a mean and some louder channels, a block output, its gate's logits
        loud = 1 + 4 * (torch.rand(d, device=DEV, generator=g) < 0.02).float()
        s["x"] = (randn(n, d) * loud + 0.3).to(DT[c["x"]])
        s["u"] = (0.7 * randn(n, d) + 0.1).to(DT[c["u"]])
        s["w"] = 1 + 0.1 * randn(d)
        s["b"] = 0.1 * randn(d) if c["kind"] == "layer" else None
        s["pw"] = 1 + 0.1 * randn(d) if c["post"] else None
        s["pb"] = 0.1 * randn(d) if c["post"] and c["kind"] == "layer" else None
        s["scale"] = 0.5 + 0.1 * randn(d) if c["scale"] else None
        s["gate"] = {"none": lambda: None, "token": lambda: randn(n, 1).to(DT[c["u"]]),
                     "channel": lambda: randn(n, d).to(DT[c["u"]])}[c["gate"]]()
        if c["train"]:
            s["dy"], s["dz"] = randn(n, d).to(DT[c["x"]]), randn(n, d).to(DT[c["z"]])
            s["wrt"] = [k for k in ("x", "u", "w", "b", "pw", "pb", "scale", "gate") if s[k] is not None]
            for k in s["wrt"]:
                s[k].requires_grad_(True)
        return s
    shapes = _clip_shapes(c)
    s["grads"] = [(0.01 * randn(*shape)).to(DT[t]) for shape, t in shapes]
    # fp32 destinations in one flat buffer, each starting at a multiple of `pad` values
    sizes = [x.numel() for x in s["grads"]]
    s["pads"] = [torch.zeros(-n % c["pad"], device=DEV) for n in sizes]
    s["flat"] = torch.zeros(sum(n + p.numel() for n, p in zip(sizes, s["pads"])), device=DEV)
    pieces = s["flat"].split([k for n, p in zip(sizes, s["pads"]) for k in (n, p.numel())])[::2]
    s["out"] = [p.view(x.shape) for p, x in zip(pieces, s["grads"])]
    return s


# ------------------------------------------------------------------------------------------
#  one pass
# ------------------------------------------------------------------------------------------
def run(s):
    c = s["c"]
    if own:
        return _own(s, c)
    return {"ffn": _ffn, "norm": _norm, "clip": _clip}[c["op"]](s, c)


def _own(s, c):
    from sca2_b200 import ops
    if c["op"] == "ffn":
        if not c["train"]:
            with torch.no_grad():
                return {"h": ops.gated_ffn(s["x"], s["wg"], s["wu"], act=c["act"])}
        h = ops.gated_ffn(s["x"], s["wg"], s["wu"], act=c["act"])
        dx, dwg, dwu = torch.autograd.grad(h, (s["x"], s["wg"], s["wu"]), s["dh"])
        return {"h": h.detach(), "dx": dx, "dwg": dwg, "dwu": dwu}
    if c["op"] == "norm":
        args = dict(gate=s["gate"], scale=s["scale"], post_weight=s["pw"], post_bias=s["pb"], kind=c["kind"],
                    out_dtype=DT[c["z"]])
        if not c["train"]:
            with torch.no_grad():
                y, z = ops.residual_norm(s["x"], s["u"], s["w"], s["b"], **args)
            return {"y": y, "z": z}
        y, z = ops.residual_norm(s["x"], s["u"], s["w"], s["b"], **args)
        grads = torch.autograd.grad((y, z), [s[k] for k in s["wrt"]], (s["dy"], s["dz"]))
        return {"y": y.detach(), "z": z.detach(), **{"d" + k: v for k, v in zip(s["wrt"], grads)}}
    norm = ops.clip_grads(s["grads"], c["max_norm"], out=s["out"])
    return {"norm": norm, "grads": s["flat"]}


def _act(g, act):
    """act(g) and its derivative."""
    if act == "silu":
        p = 1 / (1 + torch.exp(-g))
        return g * p, p * (1 + g * (1 - p))
    p = 0.5 * (1 + torch.erf(g * 0.5 ** 0.5))
    return g * p, p + g * torch.exp(-0.5 * g * g) * (2 * math.pi) ** -0.5


@torch.no_grad()
def _ffn(s, c):
    x, wg, wu = s["x"].float(), s["wg"].float(), s["wu"].float()
    g, u = x @ wg.t(), x @ wu.t()
    a, da = _act(g, c["act"])
    h = (a * u).bfloat16()
    if not c["train"]:
        return {"h": h}
    dh = s["dh"].float()
    dg, du = dh * u * da, dh * a
    return {"h": h, "dx": (dg @ wg + du @ wu).bfloat16(), "dwg": (dg.t() @ x).bfloat16(),
            "dwu": (du.t() @ x).bfloat16()}


def _stats(v, kind, eps=1e-5):
    """The normalised rows and 1 / their deviation."""
    m = v.mean(-1, keepdim=True) if kind == "layer" else 0.0
    r = 1 / torch.sqrt((v - m).square().mean(-1, keepdim=True) + eps)
    return (v - m) * r, r


def _norm_grad(dn, n, r, kind):
    """The gradient of the rows from that of the normalised rows."""
    m = dn.mean(-1, keepdim=True) if kind == "layer" else 0.0
    return r * (dn - m - n * (dn * n).mean(-1, keepdim=True))


@torch.no_grad()
def _norm(s, c):
    f = {k: v.float() if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    kind, xt, ut, zt = c["kind"], DT[c["x"]], DT[c["u"]], DT[c["z"]]
    zero = torch.zeros((), device=DEV)
    un, ur = _stats(f["u"], kind) if c["post"] else (f["u"], None)
    p = un * f["pw"] + (f["pb"] if f["pb"] is not None else zero) if c["post"] else un
    sg = 1 / (1 + torch.exp(-f["gate"])) if f["gate"] is not None else 1.0
    sc = f["scale"] if f["scale"] is not None else 1.0
    y = f["x"] + sc * sg * p
    yn, yr = _stats(y, kind)
    z = yn * f["w"] + (f["b"] if f["b"] is not None else zero)
    out = {"y": y.to(xt), "z": z.to(zt)}
    if not c["train"]:
        return out
    dy = f["dy"] + _norm_grad(f["dz"] * f["w"], yn, yr, kind)
    dp = dy * sc * sg
    out["dx"] = dy.to(xt)
    out["du"] = (_norm_grad(dp * f["pw"], un, ur, kind) if c["post"] else dp).to(ut)
    out["dw"] = (f["dz"] * yn).sum(0)
    if f["b"] is not None:
        out["db"] = f["dz"].sum(0)
    if f["pw"] is not None:
        out["dpw"] = (dp * un).sum(0)
    if f["pb"] is not None:
        out["dpb"] = dp.sum(0)
    if f["scale"] is not None:
        out["dscale"] = (dy * sg * p).sum(0)
    if f["gate"] is not None:
        dg = dy * sc * p * sg * (1 - sg)
        out["dgate"] = (dg.sum(-1, keepdim=True) if c["gate"] == "token" else dg).to(ut)
    return out


@torch.no_grad()
def _clip(s, c):
    # long sums of squares: 64 bits
    norm = torch.stack([g.double().square().sum() for g in s["grads"]]).sum().sqrt().float()
    coef = torch.clamp(c["max_norm"] / (norm + 1e-6), max=1.0)
    return {"norm": norm, "grads": torch.cat([t for g, p in zip(s["grads"], s["pads"])
                                              for t in ((g.float() * coef).reshape(-1), p)])}


# ------------------------------------------------------------------------------------------
#  in 64 bits, by differentiation of the definitions
# ------------------------------------------------------------------------------------------
def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "clip":
        every = torch.cat([g.double().reshape(-1) for g in s["grads"]])
        norm = torch.linalg.vector_norm(every)
        factor = min(1.0, c["max_norm"] / (float(norm) + 1e-6))
        flat = torch.zeros(s["flat"].numel(), dtype=torch.float64, device=DEV)
        at = 0
        for g, p in zip(s["grads"], s["pads"]):
            flat[at:at + g.numel()] = g.double().reshape(-1) * factor
            at += g.numel() + p.numel()
        return {"norm": norm, "grads": flat}
    v = {k: t.detach().double().requires_grad_(t.requires_grad) for k, t in s.items() if isinstance(t, torch.Tensor)}
    if c["op"] == "ffn":
        pre = torch.nn.functional.linear(v["x"], v["wg"])
        h = (torch.nn.functional.silu(pre) if c["act"] == "silu" else torch.nn.functional.gelu(pre)) \
            * torch.nn.functional.linear(v["x"], v["wu"])
        if not c["train"]:
            return {"h": h}
        dx, dwg, dwu = torch.autograd.grad(h, (v["x"], v["wg"], v["wu"]), v["dh"])
        return {"h": h.detach(), "dx": dx, "dwg": dwg, "dwu": dwu}

    def normed(t, weight, bias):
        if c["kind"] == "layer":
            return torch.nn.functional.layer_norm(t, (c["d"],), weight, bias, 1e-5)
        return t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + 1e-5) * weight

    t = normed(v["u"], v["pw"], v.get("pb")) if c["post"] else v["u"]
    if "scale" in v:
        t = t * v["scale"]
    if "gate" in v:
        t = t * torch.sigmoid(v["gate"])
    y = v["x"] + t
    z = normed(y, v["w"], v.get("b"))
    if not c["train"]:
        return {"y": y, "z": z}
    grads = torch.autograd.grad((y, z), [v[k] for k in s["wrt"]], (v["dy"], v["dz"]))
    return {"y": y.detach(), "z": z.detach(), **{"d" + k: g for k, g in zip(s["wrt"], grads)}}
