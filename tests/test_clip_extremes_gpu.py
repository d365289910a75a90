"""Norms at fp32's limits: the largest that it holds, and those beyond."""
import math

import pytest
import torch

from tests.test_clip_grads_gpu import F, H, _check, _norm64, _tensors

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("size", [3e36, 4.7e36])
@pytest.mark.parametrize("dts", [(F,), (F, H)])
def test_just_below_the_limit(size, dts):
    from sca2_b200 import ops
    src = _tensors([(5000,), (77,)], dts, size=size)
    assert 2e38 < _norm64(src) < 3.4e38
    n = _norm64(src)
    assert abs(float(ops.grad_norm(src)) - n) <= (2.0 ** -24 + 1e-11) * n
    for max_norm in (1.0, 1e38):
        dst = [torch.zeros_like(t, dtype=F) for t in src]
        _check(src, dst, ops.clip_grads(src, max_norm, out=dst), max_norm)


@pytest.mark.parametrize("size", [3e37, 1e37])
@pytest.mark.parametrize("dts", [(F,), (F, H)])
def test_beyond_the_limit(size, dts):
    """Finite values whose norm is not an fp32 number: infinite, and the values become 0."""
    from sca2_b200 import ops
    src = _tensors([(5000,), (77,)], dts, size=size)
    assert all(bool(torch.isfinite(t).all()) for t in src) and _norm64(src) > 3.5e38
    assert math.isinf(float(ops.grad_norm(src)))
    out = [torch.ones_like(t) for t in src]
    assert math.isinf(float(ops.clip_grads(src, 1.0, out=out))) and math.isinf(float(ops.clip_grads(src, 1.0)))
    for t in (*src, *out):
        assert torch.equal(t, torch.zeros_like(t))
