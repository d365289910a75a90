"""Tensors that hold their values in another way than their memory says."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _negated(t):
    """-t as torch keeps it lazily: the imaginary part of a conjugate, values 2 apart, sign by a flag."""
    v = torch.complex(torch.zeros_like(t), t).conj().imag
    assert v.is_neg() and torch.equal(v, -t)
    return v


def test_lazily_negated_tensors():
    """One value a row, where such a view needs no copy for its strides, and one value in all."""
    from sca2_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(3)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)
    x, u, gate, w, s = r(5, 1), r(5, 1), r(5, 1), r(1), r(1)
    ref = ops.residual_norm(-x, -u, -w, gate=-gate, scale=-s)
    got = ops.residual_norm(_negated(x), _negated(u), _negated(w), gate=_negated(gate), scale=_negated(s))
    assert torch.equal(ref[0], got[0]) and torch.equal(ref[1], got[1])
    n = _negated(r(1).abs() + 1)
    out = torch.zeros(1, device="cuda")
    want = n / n.abs() * 0.5
    ops.clip_grads([n], 0.5, out=[out])
    assert float((out - want).abs()) < 1e-6
    ops.clip_grads([n], 0.5)
    assert float((n - want).abs()) < 1e-6


def test_a_negated_destination_is_refused():
    from sca2_b200 import _lib, ops
    with pytest.raises(_lib.Sca2Error, match="contiguous"):
        ops.clip_grads([torch.ones(1, device="cuda")], 0.5, out=[_negated(torch.ones(1, device="cuda"))])


def test_a_tensor_that_overlaps_itself_is_not_clipped_in_place():
    """Refused before anything is written: the gradient of a sum is one value, expanded."""
    from sca2_b200 import _lib, ops
    plain = torch.randn(100, device="cuda")
    x = torch.zeros(8, 16, device="cuda", requires_grad=True)
    (expanded,) = torch.autograd.grad(x.sum(), x)
    assert expanded.stride() == (0, 0)
    windows = torch.randn(40, device="cuda").unfold(0, 8, 4)
    for bad in (expanded, windows, windows.t(), torch.zeros(6, device="cuda").as_strided((3, 2), (2, 1))[:, :1].expand(3, 5)):
        keep, was, version = plain.clone(), bad.clone(), plain._version
        with pytest.raises(_lib.Sca2Error, match="overlap"):
            ops.clip_grads([plain, bad], 0.5)
        assert torch.equal(plain, keep) and torch.equal(bad, was) and plain._version == version
        # read, it counts with the values that it shows
        n = ops.grad_norm([plain, bad])
        ref = float((plain.double().square().sum() + bad.double().square().sum()).sqrt())
        assert abs(float(n) - ref) <= (2.0 ** -24 + 1e-11) * ref
        out = [torch.zeros(100, device="cuda"), torch.zeros(bad.shape, device="cuda")]
        assert torch.equal(ops.clip_grads([plain, bad], 0.5, out=out), n)
    one = torch.randn(5, 1, device="cuda").expand(5, 1)[:, :, None]  # strides of single values do not matter
    ops.clip_grads([plain, one.as_strided((5, 1, 1), (1, 0, 7))], 0.5)
