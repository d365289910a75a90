"""Forms of the residual join beside those of test_residual_norm_gpu.py, held against 64 bits with its
tolerances: a gate of another type than u, and every option on the forward that holds a whole row of
769 to 1024 values in a warp."""
import pytest
import torch

from tests.test_residual_norm_gpu import F, H, _check, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ut,gt", [(H, F), (F, H), (H, torch.float64)])
@pytest.mark.parametrize("gate", ["token", "channel"])
@pytest.mark.parametrize("rows,d", [(40, 136), (1300, 75)])
def test_gate_of_another_type(ut, gt, gate, rows, d):
    """The logits count with all their bits up to 32."""
    i, dy, dz = _inputs(rows, d, F, ut, gate=gate)
    i["gate"] = (6 * torch.randn(i["gate"].shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(4))).float().to(gt)
    _check(i, dy, dz)
