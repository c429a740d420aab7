"""An eps that the norm's root cannot be taken of is refused: rows of zeros would become NaN."""
import pytest
import torch

import sonicmoe


@pytest.mark.parametrize("eps", [1e-91, 1e-110, 1e-300, 5e-324, float("inf"), float("nan"), -1e-6])
def test_refused(eps):
    x, w = torch.zeros(2, 64, dtype=torch.bfloat16), torch.ones(64)
    with pytest.raises(ValueError, match="eps"):
        sonicmoe.rms_norm(x, w, eps=eps)
    with pytest.raises(ValueError, match="eps"):
        sonicmoe.rms_norm_quantized(x, w, eps=eps)
    if not eps > 1:
        from sonicmoe._lib import lib
        assert lib.smoe_rms_norm(16, 0, 64, None, 0, 64, 16, 0, 2, 64, eps, 16, None, None, 0, None, None, None) == 6


@pytest.mark.parametrize("eps", [0.0, 1e-90, 1e-40, 1e30])
def test_taken(eps):
    with pytest.raises(RuntimeError, match="CUDA"):
        sonicmoe.rms_norm(torch.zeros(2, 64), torch.ones(64), eps=eps)


@pytest.mark.gpu
@pytest.mark.parametrize("eps", [1e-90, 1e-60, 1e-20])
def test_rows_of_zeros(eps):
    """Their norm is zero; a gradient of 1 goes on times 1 / sqrt(eps), which f32 may not hold, and the weight's is zero."""
    for dtype in (torch.bfloat16, torch.float32):
        x = torch.zeros(3, 64, dtype=dtype, device="cuda", requires_grad=True)
        w = torch.ones(64, device="cuda", requires_grad=True)
        y = sonicmoe.rms_norm(x, w, eps=eps)
        dx, dw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
        assert not y.any() and not dw.any()
        want = torch.full((3, 64), eps ** -0.5, dtype=torch.float64)
        half = torch.finfo(dtype).eps / 2 + 2.0 ** -22
        got = dx.double().cpu()
        assert ((got - want).abs() <= half * want).all() if eps > 1e-70 else torch.isinf(got).all()
