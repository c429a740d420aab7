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


def test_expanded_gradients_are_not_changed_in_place():
    """What torch.autograd.grad returns for a sum: one value in every place.  Refused before the others are touched."""
    wide = torch.ones(1).expand(6)
    for bad in (wide, torch.ones(3, 1).expand(3, 4), torch.ones(4).expand(2, 4)):
        with pytest.raises(ValueError, match="several places"):
            sonicmoe.clip_gradients([torch.zeros(8), bad], 1.0)
    # into other tensors, and one that only looks expanded
    for grads, kw in (([wide], dict(out=[torch.zeros(6)])), ([torch.zeros(1).expand(1)], {}), ([torch.zeros(0, 1).expand(0, 5)], {}),
                      ([torch.zeros(4, 4).T], {}), ([torch.zeros(8)[::2]], {})):
        with pytest.raises(RuntimeError, match="CUDA"):
            sonicmoe.clip_gradients(grads, 1.0, **kw)


def test_the_norm_does_not_lie_in_a_strided_gradient():
    """Which is written from a copy at the end: the norm that is returned would be a clipped value."""
    base = torch.zeros(100)
    for grads, at in (([base[:64].view(8, 8).T], 13), ([base[10:50].view(5, 8)[:, :4]], 45), ([base[60:90:3]], 87), ([base[60:90:3]], 60)):
        with pytest.raises(ValueError, match="norm lies"):
            sonicmoe.clip_gradients(grads, 1.0, norm=base[at])
    for grads, at in (([base[:64].view(8, 8).T], 64), ([base[10:50].view(5, 8)[:, :4]], 46), ([base[60:90:3]], 88), ([base[60:90:3]], 59)):
        with pytest.raises(RuntimeError, match="CUDA"):
            sonicmoe.clip_gradients(grads, 1.0, norm=base[at])


@pytest.mark.gpu
def test_a_single_output_receives_the_result():
    g = torch.randn(5, 7, device="cuda")
    o = torch.empty(5, 7, device="cuda", dtype=torch.bfloat16)
    n = sonicmoe.clip_gradients(g, 0.5, out=o)
    want = g.double() * (0.5 / (float(n) + 1e-6))
    assert ((o.double() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -20)).all()


@pytest.mark.gpu
def test_nothing_is_changed_by_a_call_that_is_refused():
    g, wide = torch.randn(64, device="cuda"), torch.ones(1, device="cuda").expand(6)
    kept = g.clone()
    with pytest.raises(ValueError, match="several places"):
        sonicmoe.clip_gradients([g, wide], 1e-3)
    assert torch.equal(g, kept)
    o = [torch.empty(64, device="cuda"), torch.empty(6, device="cuda")]
    n = float(sonicmoe.clip_gradients([g, wide], 1e-3, out=o))
    assert abs(n - float(torch.cat([g, wide]).double().norm())) <= n * 2.0 ** -21
    assert (o[1] == o[1][0]).all() and abs(float(o[1][0]) * n / 1e-3 - 1) <= 2.0 ** -20 + 1e-6 / n
