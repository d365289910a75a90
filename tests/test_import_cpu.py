"""The package imports where torch was built without CUDA (layers are built and configured there)."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_import_without_cuda_bindings():
    code = ("import torch\n"
            "for n in [n for n in dir(torch._C) if n.startswith('_cuda')]: delattr(torch._C, n)\n"
            "from sca2_b200 import heads, layers, lm, ops, registry\n"
            "layers.GatedLayer(layers.LayerCfg(d=32, Mc=16, Md=4, G=4, ff=48, freq='rope', dv=32))\n"
            "try:\n"
            "    ops.residual_norm(torch.zeros(2, 8), torch.zeros(2, 8))\n"
            "except ops._lib.Sca2Error:\n"
            "    print('refused')\n")
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0 and "refused" in r.stdout, r.stderr
