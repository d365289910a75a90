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


@pytest.mark.parametrize("rows,d", [(7105, 1024), (7109, 1020), (7112, 772), (7104, 1024)])
@pytest.mark.parametrize("gate", ["none", "token", "channel"])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("xt,ut", [(F, F), (F, H), (H, H)])
def test_a_warp_holds_a_row_of_1024_values(rows, d, gate, post, xt, ut):
    """More than 48 rows an SM: the forward with eight groups of columns a lane (7104 rows: the last that take the
    other kernel), ragged last steps, parts absent."""
    kind = "rms" if post and gate == "token" else "layer"
    i, dy, dz = _inputs(rows, d, xt, ut, post, gate, scale=gate != "none", bias=kind == "layer")
    _check(i, dy, dz, kind=kind, zt=ut)


@pytest.mark.parametrize("rows,d", [(1185, 768), (1189, 516)])
@pytest.mark.parametrize("post,gate,scale,z,kind", [(False, "none", False, True, "layer"), (False, "token", True, True, "rms"),
                                                    (True, "none", False, True, "rms"), (True, "token", False, True, "layer"),
                                                    (False, "channel", False, False, "layer"), (True, "channel", True, False, "rms")])
@pytest.mark.parametrize("xt,ut", [(F, F), (H, H)])
def test_a_warp_holds_a_row_of_768_values(rows, d, post, gate, scale, z, kind, xt, ut):
    i, dy, dz = _inputs(rows, d, xt, ut, post, gate, scale, kind == "layer", z)
    _check(i, dy, dz, kind=kind, zt=ut)
