"""What clip_gradients takes and refuses, on the host."""
import pytest
import torch

import sonicmoe


def test_a_single_output_for_a_single_gradient():
    """As the gradients may be one tensor, of several rows too; these pass the checks and want a GPU."""
    for shape in ((8,), (4, 6), ()):
        g, o = torch.zeros(shape), torch.zeros(shape, dtype=torch.bfloat16)
        for grads in (g, [g]):
            for out in (o, [o], (o,)):
                with pytest.raises(RuntimeError, match="CUDA"):
                    sonicmoe.clip_gradients(grads, 1.0, out=out)
    with pytest.raises(ValueError, match="1 outputs for 2 gradients"):
        sonicmoe.clip_gradients([torch.zeros(2), torch.zeros(2)], 1.0, out=torch.zeros(2, 2))
    with pytest.raises(ValueError, match="shapes"):
        sonicmoe.clip_gradients(torch.zeros(2), 1.0, out=torch.zeros(3))


@pytest.mark.gpu
def test_a_single_output_receives_the_result():
    g = torch.randn(5, 7, device="cuda")
    o = torch.empty(5, 7, device="cuda", dtype=torch.bfloat16)
    n = sonicmoe.clip_gradients(g, 0.5, out=o)
    want = g.double() * (0.5 / (float(n) + 1e-6))
    assert ((o.double() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -20)).all()
