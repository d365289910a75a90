"""The residual join, gradient clipping and gated feed-forward without a GPU: refusals of the
Python functions and of the C entry points (host checks, before any launch), struct layouts, fake
implementations."""
import ctypes
import os
import shutil
import subprocess
import tempfile

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from sca2_b200 import _lib, ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20  # an address that is never read: every call below is refused first


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
def test_struct_layouts():
    fields = {"sca2_ffn_args": (_lib.FfnArgs, ["w_up", "ldx", "ldu", "rows", "d", "f", "act"]),
              "sca2_rnorm_args": (_lib.RNormArgs, ["gate", "sx", "w", "scale", "rows", "d", "z_dtype", "gate_mode", "eps"]),
              "sca2_rnorm_grads": (_lib.RNormGrads, ["du", "dw", "dpb"]),
              "sca2_grad_tensor": (_lib.GradTensor, ["dst", "n", "src_dtype", "dst_dtype"])}
    body = "".join(f'printf("%zu\\n", sizeof({t}));' + "".join(f'printf("%zu\\n", offsetof({t}, {f}));' for f in fs)
                   for t, (_, fs) in fields.items())
    with tempfile.TemporaryDirectory() as d:
        c = os.path.join(d, "p.c")
        open(c, "w").write('#include <stddef.h>\n#include <stdio.h>\n#include "sca2b200.h"\nint main(void){' + body + "return 0;}")
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), c, "-o", c + ".x"], check=True)
        got = [int(x) for x in subprocess.run([c + ".x"], capture_output=True, text=True, check=True).stdout.split()]
    want = [v for cls, fs in fields.values() for v in [ctypes.sizeof(cls)] + [getattr(cls, f).offset for f in fs]]
    assert got == want
    t = [torch.zeros(3)] * 2
    assert len(ops._grad_table(t, t, [[torch.float32] * 2])) == 2 * ctypes.sizeof(_lib.GradTensor)


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 8)
    for call in (lambda: ops.residual_norm(x, x, torch.ones(8)), lambda: ops.grad_norm([x]),
                 lambda: ops.clip_grads([x], 1.0), lambda: ops.gated_ffn(x.bfloat16(), x.bfloat16(), x.bfloat16())):
        with pytest.raises(_lib.Sca2Error, match="CUDA"):
            call()


def test_residual_norm_refusals():
    with FakeTensorMode():
        x, w = torch.empty(4, 8, device="cuda"), torch.empty(8, device="cuda")
        half, long = torch.empty(4, 8, device="cuda", dtype=torch.float16), torch.empty(4, 9, device="cuda")
        bad = [dict(u=long), dict(u=x[:3]), dict(weight=torch.empty(9, device="cuda")), dict(bias=w), dict(post_bias=w),
               dict(weight=w, kind="batch"), dict(weight=w, out_dtype=torch.float16), dict(u=half),
               dict(gate=torch.empty(4, 2, device="cuda")), dict(gate=torch.empty(4, device="cuda")),
               dict(gate=torch.empty(3, 8, device="cuda")), dict(scale=torch.empty(1, device="cuda"))]
        for kw in bad:
            kw = dict(kw)
            u = kw.pop("u", x)
            with pytest.raises(_lib.Sca2Error):
                ops.residual_norm(x, u, kw.pop("weight", None), kw.pop("bias", None), **kw)
        with pytest.raises(_lib.Sca2Error):
            ops.residual_norm(torch.empty((), device="cuda"), torch.empty((), device="cuda"))


def test_residual_norm_entry_refusals():
    lib = _lib.load()

    def args(**kw):
        a = _lib.RNormArgs()
        a.x = a.u = a.w = P
        a.sx = a.su = a.rows = a.d = 8
        for k, v in kw.items():
            setattr(a, k, v)
        return a
    bad = [dict(d=0), dict(rows=-1), dict(x=None), dict(u=None), dict(sx=7), dict(su=0), dict(x_dtype=2), dict(u_dtype=-1),
           dict(z_dtype=5), dict(kind=2), dict(gate_mode=3), dict(gate_mode=1), dict(gate_mode=2, gate=P, sg=7),
           dict(eps=-1.0), dict(eps=float("nan")), dict(pb=P), dict(b=P, w=None), dict(b=P, kind=1), dict(pb=P, pw=P, kind=1)]
    g = _lib.RNormGrads(P, P, P, P, P, P, P, P)
    for kw in bad:
        assert lib.sca2_residual_norm_fwd(args(**kw), P, P, None, None) == _lib.SCA2_ERR_ARG, kw
        assert lib.sca2_residual_norm_bwd(args(**kw), P, P, P, g, P, 1 << 40, None) == _lib.SCA2_ERR_ARG, kw
        assert lib.sca2_last_error().startswith(b"residual_norm")
    assert lib.sca2_residual_norm_fwd(args(d=4097, sx=4097, su=4097), P, P, None, None) == _lib.SCA2_ERR_UNSUPPORTED
    assert lib.sca2_residual_norm_fwd(None, P, P, None, None) == _lib.SCA2_ERR_ARG
    assert lib.sca2_residual_norm_fwd(args(), None, P, None, None) == _lib.SCA2_ERR_ARG
    assert lib.sca2_residual_norm_fwd(args(w=None), P, P, None, None) == _lib.SCA2_ERR_ARG
    assert lib.sca2_residual_norm_fwd(args(), P, P, P + 4, None) == _lib.SCA2_ERR_ARG
    n = lib.sca2_residual_norm_work_bytes(8, 8)
    assert n > 0 and lib.sca2_residual_norm_work_bytes(0, 8) == 0 and lib.sca2_residual_norm_work_bytes(8, 5000) == 0
    bwd = lambda a=None, st=P, dz=P, gr=g, wk=P, nb=n: lib.sca2_residual_norm_bwd(a or args(), st, P, dz, gr, wk, nb, None)
    for kw in (dict(st=None), dict(st=P + 4), dict(gr=None), dict(wk=None), dict(wk=P + 8), dict(nb=n - 1),
               dict(a=args(w=None)), dict(gr=_lib.RNormGrads(None, P)), dict(gr=_lib.RNormGrads(P, None)),
               dict(a=args(gate_mode=1, gate=P, sg=1), gr=_lib.RNormGrads(P, P, None))):
        assert bwd(**kw) == _lib.SCA2_ERR_ARG, kw


def test_clip_refusals():
    with FakeTensorMode():
        t, h = torch.empty(8, device="cuda"), torch.empty(8, device="cuda", dtype=torch.float16)
        for call in (lambda: ops.clip_grads([t], -1.0), lambda: ops.clip_grads([t], float("nan")),
                     lambda: ops.clip_grads([h], 1.0), lambda: ops.grad_norm([h]), lambda: ops.grad_norm([None]),
                     lambda: ops.clip_grads([t], 1.0, out=[]), lambda: ops.clip_grads([t], 1.0, out=[h]),
                     lambda: ops.clip_grads([t], 1.0, out=[t[:4]]),
                     lambda: ops.clip_grads([t.view(2, 4)], 1.0, out=[torch.empty(4, 2, device="cuda").t()])):
            with pytest.raises(_lib.Sca2Error):
                call()


def test_clip_entry_refusals():
    import struct
    lib = _lib.load()
    one = lambda s=P, d=P, n=8, a=0, b=0: struct.pack("=QQqii", s, d, n, a, b)
    big = 1 << 40
    for t in (one(s=0), one(d=0), one(n=-1), one(n=(1 << 41) + 1), one(a=2), one(b=3), one(s=P + 2), one(d=P + 2),
              one(a=1), one(d=P + 4), one() + one(), one(d=P + 4096) + one(s=P + 4096, d=P + 8192)):
        assert lib.sca2_clip_grads(t, len(t) // 32, 1.0, P, P, big, None) == _lib.SCA2_ERR_ARG, t
    t = one()
    assert lib.sca2_clip_grads(t, -1, 1.0, P, P, big, None) == _lib.SCA2_ERR_ARG
    assert lib.sca2_clip_grads(None, 1, 1.0, P, P, big, None) == _lib.SCA2_ERR_ARG
    assert lib.sca2_clip_grads(t, 1, -1.0, P, P, big, None) == _lib.SCA2_ERR_ARG
    assert lib.sca2_clip_grads(t, 1, 1.0, None, P, big, None) == _lib.SCA2_ERR_ARG
    assert lib.sca2_clip_grads(t, 1, 1.0, P, None, big, None) == _lib.SCA2_ERR_ARG
    assert lib.sca2_clip_grads(t, 1, 1.0, P, P + 4, big, None) == _lib.SCA2_ERR_ARG
    n = lib.sca2_clip_grads_work_bytes(1)
    assert n >= 8 and lib.sca2_clip_grads(t, 1, 1.0, P, P, n - 1, None) == _lib.SCA2_ERR_ARG
    assert lib.sca2_grad_norm(t, 1, P, P, n - 1, None) == _lib.SCA2_ERR_ARG
    assert lib.sca2_clip_grads_work_bytes(-1) == 0 and lib.sca2_clip_grads_work_bytes(2001) == 3 * n


def test_gated_ffn_refusals():
    assert ops.gated_ffn_supported(8, 16) and not ops.gated_ffn_supported(12, 16) and not ops.gated_ffn_supported(8, 4)
    with FakeTensorMode():
        e = lambda *s, t=torch.bfloat16: torch.empty(*s, device="cuda", dtype=t)
        x, w = e(4, 16), e(24, 16)
        for args in ((x, w, e(24, 8)), (x, w, e(32, 16)), (e(4, 8), w, w), (x, e(16), e(16)), (x, e(20, 16), e(20, 16)),
                     (e(4, 12), e(24, 12), e(24, 12)), (e(1).squeeze(0), w, w), (x, w, w, "relu"), (e(4, 16, t=torch.float32), w, w),
                     (x, w, e(24, 16, t=torch.float32)), (x, w, e(24, 16, t=torch.float16))):
            with pytest.raises(_lib.Sca2Error):
                ops.gated_ffn(*args)


def test_gated_ffn_entry_refusals():
    lib = _lib.load()

    def args(**kw):
        a = _lib.FfnArgs(P, P, P, 16, 16, 16, 300, 16, 24, 0)
        for k, v in kw.items():
            setattr(a, k, v)
        return a
    bad = [dict(x=None), dict(w_gate=None), dict(w_up=None), dict(rows=-1), dict(d=0), dict(f=0), dict(act=2), dict(ldx=8),
           dict(ldx=20), dict(ldg=8), dict(ldu=12), dict(x=P + 8), dict(w_gate=P + 2), dict(w_up=P + 4)]
    wide = [dict(d=12), dict(f=20), dict(rows=(1 << 30) + 1), dict(f=1 << 21), dict(rows=1 << 30, f=1 << 20)]
    n = lib.sca2_gated_ffn_work_bytes(300, 16, 24)
    assert n > 0 and lib.sca2_gated_ffn_work_bytes(0, 16, 24) == 0
    for kw, code in [(b, _lib.SCA2_ERR_ARG) for b in bad] + [(b, _lib.SCA2_ERR_UNSUPPORTED) for b in wide]:
        assert lib.sca2_gated_ffn_fwd(args(**kw), P, None) == code, kw
        assert lib.sca2_gated_ffn_bwd(args(**kw), P, P, P, P, P, n, None) == code, kw
    assert lib.sca2_gated_ffn_fwd(None, P, None) == _lib.SCA2_ERR_ARG
    assert lib.sca2_gated_ffn_fwd(args(), None, None) == _lib.SCA2_ERR_ARG
    assert lib.sca2_gated_ffn_fwd(args(), P + 2, None) == _lib.SCA2_ERR_ARG
    bwd = lambda dh=P, dx=P, g=P, u=P, w=P, nb=n: lib.sca2_gated_ffn_bwd(args(), dh, dx, g, u, w, nb, None)
    for kw in (dict(dh=None), dict(dh=P + 8), dict(dx=P + 8), dict(g=None), dict(u=None), dict(g=P + 2), dict(w=None),
               dict(w=P + 128), dict(nb=n - 1)):
        assert bwd(**kw) == _lib.SCA2_ERR_ARG, kw


def test_fake_shapes():
    with FakeTensorMode():
        b, w2 = torch.empty(2, 3, 16, device="cuda", dtype=torch.bfloat16), torch.empty(24, 16, device="cuda", dtype=torch.bfloat16)
        w = torch.empty(16, device="cuda", requires_grad=True)
        y, z = ops.residual_norm(b, b, w, post_weight=w)  # the public calls trace too
        assert y.shape == z.shape == b.shape and z.requires_grad
        assert ops.gated_ffn(b, w2, w2).shape == (2, 3, 24)
        h = torch.ops.sca2b200.gated_ffn_fwd(b, w2, w2, 0)
        assert h.shape == (2, 3, 24) and h.dtype == torch.bfloat16
        out = torch.ops.sca2b200.gated_ffn_bwd(b, w2, w2, 0, h, True, False)
        assert [tuple(t.shape) for t in out] == [(2, 3, 16), (0,), (0,)]
        x, u = torch.empty(2, 3, 40, device="cuda"), torch.empty(2, 3, 40, device="cuda", dtype=torch.bfloat16)
        w, g = torch.empty(40, device="cuda"), torch.empty(2, 3, 1, device="cuda", dtype=torch.bfloat16)
        y, z, st = torch.ops.sca2b200.residual_norm_fwd(x, u, w, None, g, w, None, None, 0, 1e-5, torch.bfloat16, True)
        assert y.shape == z.shape == x.shape and y.dtype == x.dtype and z.dtype == u.dtype and st.shape == (6, 4)
        out = torch.ops.sca2b200.residual_norm_bwd(x, u, w, None, g, w, None, None, 0, 1e-5, torch.bfloat16, st, y, z)
        assert [tuple(t.shape) for t in out] == [(2, 3, 40), (2, 3, 40), (40,), (0,), (2, 3, 1), (40,), (0,), (0,)]
        assert torch.ops.sca2b200.grad_norm([x, w]).shape == ()
        assert torch.ops.sca2b200.clip_grads_([x, w], 1.0).shape == ()


def test_tail_options():
    """The tail's parameters by option, the reference's names without any; bad options refused."""
    from sca2_b200 import layers
    cfg = lambda **t: layers.LayerCfg(d=32, Mc=16, Md=4, G=4, ff=48, freq="rope", dv=32, tail=layers.TailCfg(**t) if t else None)
    plain = set(layers.SCA2Layer(cfg()).state_dict())
    assert set(layers.SCA2Layer(cfg(res_scale=0.0, gate="")).state_dict()) == plain
    full = set(layers.SCA2Layer(cfg(ffn_act="silu", post_norm=True, gate="token", res_scale=0.1)).state_dict())
    assert {"ff.gate.weight", "ff.up.weight", "ff.down.weight", "join1.norm.weight", "join2.gate.bias", "join1.scale"} <= full
    assert {k for k in plain if not k.startswith("ff.")} <= full
    for bad in (dict(ffn_act="relu"), dict(gate="row"), dict(res_scale=-1.0)):
        with pytest.raises(ValueError):
            layers.TailCfg(**bad)
