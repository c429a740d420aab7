"""Forward-mode derivatives are refused, not dropped."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

import sonicmoe

BF = torch.bfloat16


def dual(*shape, dtype=BF):
    return fwAD.make_dual(torch.zeros(*shape, dtype=dtype), torch.ones(*shape, dtype=dtype))


def t(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


CALLS = {
    "norm x": lambda: sonicmoe.rms_norm(dual(2, 64), t(64)),
    "norm weight": lambda: sonicmoe.rms_norm(t(2, 64), dual(64)),
    "norm residual": lambda: sonicmoe.rms_norm(t(2, 64), t(64), dual(2, 64)),
    "payload": lambda: sonicmoe.rms_norm_quantized(dual(2, 64), t(64)),
    "payload and rows": lambda: sonicmoe.rms_norm_quantized(t(2, 64), dual(64, dtype=torch.float32), with_output=True),
    "products x": lambda: sonicmoe.grouped_linear(dual(4, 16), t(8, 16)),
    "products weight": lambda: sonicmoe.grouped_linear(t(4, 16), dual(8, 16)),
    "gradient norm": lambda: sonicmoe.gradient_norm([t(8, dtype=torch.float32), dual(8, dtype=torch.float32)]),
    "clipping": lambda: sonicmoe.clip_gradients([dual(8, dtype=torch.float32)], 1.0),
    "clipping out": lambda: sonicmoe.clip_gradients([t(8)], 1.0, out=[dual(8)]),
    "clipping norm": lambda: sonicmoe.clip_gradients([t(8)], 1.0, norm=dual(1, dtype=torch.float32)),
}


@pytest.mark.parametrize("call", CALLS.values(), ids=CALLS)
@pytest.mark.parametrize("grad", [True, False])
def test_refused(call, grad):
    with fwAD.dual_level(), torch.set_grad_enabled(grad):
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call()


def test_the_primal_alone_is_taken():
    """Without a tangent, inside a level and where tangents are switched off, the call goes on (and wants a GPU)."""
    with fwAD.dual_level():
        with pytest.raises(RuntimeError, match="CUDA"):
            sonicmoe.rms_norm(t(2, 64), t(64))
        x = dual(2, 64)
        with fwAD._set_fwd_grad_enabled(False), pytest.raises(RuntimeError, match="CUDA"):
            sonicmoe.rms_norm(x, t(64))
        with pytest.raises(RuntimeError, match="CUDA"):
            sonicmoe.grouped_linear(fwAD.unpack_dual(dual(4, 16)).primal, t(8, 16))
