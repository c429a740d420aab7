"""Forward-mode derivatives are refused by the calls that take the kernels without an autograd node."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

import sonicmoe


def dual(*shape, dtype):
    return fwAD.make_dual(torch.zeros(*shape, dtype=dtype), torch.ones(*shape, dtype=dtype))


@pytest.mark.parametrize("grad", [True, False])
def test_routing(grad):
    with fwAD.dual_level(), torch.set_grad_enabled(grad):
        with pytest.raises(NotImplementedError, match="forward-mode"):
            sonicmoe.group_limited_routing(dual(4, 16, dtype=torch.float32), 2)
        with pytest.raises(RuntimeError, match="CUDA"):
            sonicmoe.group_limited_routing(torch.zeros(4, 16), 2)


@pytest.mark.gpu
@pytest.mark.parametrize("grad", [True, False])
def test_block128_linear(grad):
    x, w = (torch.ones(128, 128, device="cuda").bfloat16() for _ in range(2))
    with fwAD.dual_level(), torch.set_grad_enabled(grad):
        for a, b in ((fwAD.make_dual(x, x), w), (x, fwAD.make_dual(w, w))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                sonicmoe.block128_linear(a, b)
        y = sonicmoe.block128_linear(x, w)
    assert torch.equal(y, torch.full_like(y, 128.0))
    with fwAD.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        sonicmoe.group_limited_routing(fwAD.make_dual(x.float(), x.float()), 2)
