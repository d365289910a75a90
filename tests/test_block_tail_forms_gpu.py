"""Forms of a block's tail beside those of test_block_tail_gpu.py: the types and widths that the join's
kernel does not take, the bf16 decode graph held against eager steps, a capture beside a living graph."""
import pytest
import torch

from tests._util import relerr
from tests.test_block_tail_forms_cpu import TAILS, check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tail", TAILS, ids=lambda t: "-".join(t))
@pytest.mark.parametrize("d,dtype", [(64, torch.float16), (64, torch.float64), (64, torch.float32), (64, torch.bfloat16),
                                     (4104, torch.float32), (4104, torch.bfloat16)])
def test_join(tail, d, dtype):
    join, norm = make(d, tail, dtype, "cuda")
    r = lambda: torch.randn(2, 5, d, device="cuda").to(dtype)
    check(join, norm, r(), r(), r(), dtype)


@pytest.mark.parametrize("tail", TAILS, ids=lambda t: "-".join(t))
@pytest.mark.parametrize("d", [64, 4104])
def test_join_under_autocast(tail, d):
    """fp16: an fp16 branch on an fp32 stream, whose next norm stays fp32; bf16 beyond 4096 values."""
    for dtype in (torch.float16, torch.bfloat16):
        join, norm = make(d, tail, torch.float32, "cuda")
        x, u, z = torch.randn(2, 5, d, device="cuda"), torch.randn(2, 5, d, device="cuda").to(dtype), torch.randn(2, 5, d, device="cuda")
        with torch.autocast("cuda", dtype=dtype):
            check(join, norm, x, u, z, torch.float32 if dtype == torch.float16 else dtype)


def test_layer_under_fp16_autocast():
    """A whole layer with its tail, forward and backward, near its fp32 result: the bar is the
    repository's 2e-2 for bf16, which has eight times fp16's step."""
    from sca2_b200 import layers
    torch.manual_seed(5)
    cfg = layers.LayerCfg(d=64, Mc=32, Md=4, G=8, ff=128, freq="rope", theta_scale=0.02, max_len=256, dv=64, c_heads=1,
                          c_decay=True, tail=layers.TailCfg(ffn_act="silu", post_norm=True, gate="channel", res_scale=0.5))
    layer = layers.GatedLayer(cfg).cuda()
    x = torch.randn(2, 50, 64, device="cuda")
    ref = layer(x)
    with torch.autocast("cuda", dtype=torch.float16):
        y = layer(x)
    assert relerr(y, ref) < 2e-2
    y.sum().backward()
    assert all(bool(torch.isfinite(p.grad).all()) for n, p in layer.named_parameters() if n.split(".")[0] in ("ff", "join1", "join2"))
