"""residual_norm on the CPU path: the formulas against torch's own norms, and the refusals."""
import pytest
import torch
import torch.nn.functional as F

from gpubridge_b200.ops.residual_norm import residual_norm

D = 24


def _inputs(seed=0, dtype=torch.float64):
    g = torch.Generator().manual_seed(seed)
    return ([torch.randn(2, 5, D, generator=g, dtype=dtype) for _ in range(2)]
            + [torch.randn(D, generator=g, dtype=dtype) for _ in range(4)])


def test_equals_the_separate_operations():
    r, u, w, b, pw, pb = _inputs()
    gate = torch.randn(2, 1, D, dtype=torch.float64)
    got = residual_norm(r, u, w, b, post_weight=pw, post_bias=pb, gate=gate, scale=0.5, kind="layer")
    stream = r + 0.5 * gate * F.layer_norm(u, (D,), pw, pb, 1e-5)
    assert torch.allclose(got.stream, stream, atol=1e-12)
    assert torch.allclose(got.normed, F.layer_norm(stream, (D,), w, b, 1e-5), atol=1e-12)
    got = residual_norm(r, u, w, post_weight=pw, eps=1e-3)
    stream = r + F.rms_norm(u, (D,), pw, 1e-3)
    assert torch.allclose(got.stream, stream, atol=1e-12)
    assert torch.allclose(got.normed, F.rms_norm(stream, (D,), w, 1e-3), atol=1e-12)
    assert residual_norm(r, u).normed is None
    assert torch.equal(residual_norm(r, u).stream, r + u)


def test_the_norm_is_that_of_the_rounded_stream():
    r, u, w = (t.to(torch.bfloat16) for t in _inputs(dtype=torch.float32)[:3])
    got = residual_norm(r, u, w)
    assert got.stream.dtype == got.normed.dtype == torch.bfloat16
    again = residual_norm(got.stream, torch.zeros_like(u), w)
    assert torch.equal(got.normed, again.normed)


def test_refusals():
    r, u, w, b, pw, pb = _inputs()
    with pytest.raises(ValueError, match="kind"):
        residual_norm(r, u, w, kind="batch")
    with pytest.raises(ValueError, match="update has shape"):
        residual_norm(r, u[:1], w)
    with pytest.raises(ValueError, match="weight has shape"):
        residual_norm(r, u, w[:-1])
    with pytest.raises(ValueError, match="bias needs"):
        residual_norm(r, u, None, b)
    with pytest.raises(ValueError, match="bias needs"):
        residual_norm(r, u, w, post_bias=pb)
    for shape in ((2, D), (5, D), (2, 5, D), (1, 1, D), (D - 1,)):
        with pytest.raises(ValueError, match="gate is"):
            residual_norm(r, u, w, gate=torch.ones(shape))
    with pytest.raises(ValueError, match="floating"):
        residual_norm(r, u, w, out_dtype=torch.int32)
    with pytest.raises(ValueError, match="last dimension"):
        residual_norm(torch.zeros(3, 0), torch.zeros(3, 0))
