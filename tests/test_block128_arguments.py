"""What the block-128 entry points refuse of weights that are not what they take, on the host: no call here reaches a kernel."""
import pytest
import torch


@pytest.fixture(scope="module")
def sonicmoe(built_library):
    import sonicmoe
    return sonicmoe


def test_a_weight_has_two_or_three_dimensions(sonicmoe):
    for shape in ((2, 3, 16, 64), (1, 1, 16, 64), (64,), ()):
        with pytest.raises(ValueError, match=r"\[E,N,K\]"):
            sonicmoe.quantize_weight_block128(torch.zeros(*shape, dtype=torch.bfloat16))
