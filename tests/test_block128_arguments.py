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
            sonicmoe.quantize_weight_block128(torch.zeros(shape, dtype=torch.bfloat16))


def test_a_payload_of_another_type_is_no_e4m3(sonicmoe):
    bytes_ = torch.zeros(2, 128, 64, dtype=torch.uint8)
    scales = torch.ones(2, 1, 1)
    x, efo, counts = torch.zeros(256, 64, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    idx, sc = torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2)
    w2 = (torch.zeros(2, 64, 64, dtype=torch.float8_e4m3fn), torch.ones(2, 1, 1))
    for dtype in (torch.float8_e5m2, torch.float8_e4m3fnuz, torch.float8_e5m2fnuz, torch.int8, torch.bool, torch.float8_e8m0fnu):
        bad = (bytes_.view(dtype), scales)
        with pytest.raises(ValueError, match="e4m3"):
            sonicmoe.block128_linear(x, bad, efo, counts)
        with pytest.raises(ValueError, match="e4m3"):
            sonicmoe.block128_experts(x[:4], idx, sc, bad, w2)
        with pytest.raises(ValueError, match="e4m3"):
            sonicmoe.ops.check_payload(bad[0], "payload")
    for dtype in (torch.float8_e4m3fn, torch.uint8):          # e4m3, or the bytes as the quantisers of `ops` leave them
        with pytest.raises(RuntimeError, match="CUDA"):
            sonicmoe.block128_linear(x, (bytes_.view(dtype), scales), efo, counts)
