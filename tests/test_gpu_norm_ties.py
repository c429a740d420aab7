"""Rows whose norm lies exactly on the border between two bf16 values: to the even one, as in 64 bits."""
import pytest
import torch

from oracle import norm as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32
TIES = 1 + torch.arange(1, 128, 2) * 2.0 ** -8         # between two neighbours of bf16 in [1, 2)


@pytest.fixture(scope="module")
def sonicmoe():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import sonicmoe as m
    yield m
    torch.cuda.synchronize()


def weight(H, times=1.0):
    w = TIES.repeat(-(-H // TIES.numel()))[:H] * times
    assert torch.equal(w.float().double(), w.double())
    return w.float()


def nearest(h, w, eps):
    """In 64 bits, with every step exact where the mean and its root are: h w / sqrt(sum / H + eps)."""
    h, w = h.double(), w.double()
    return O.bf16(h * w / torch.sqrt((h * h).sum(-1, keepdim=True) / h.shape[-1] + eps))


# narrow rows, several warps of them, four pieces a thread, odd widths, no power of two
@pytest.mark.parametrize("H", [8, 24, 96, 250, 256, 1000, 1001, 2048, 4096, 5120, 16384])
@pytest.mark.parametrize("residual", [None, BF, F32])
def test_constant_rows(sonicmoe, H, residual):
    """Every value 1 times a weight that is a tie."""
    c = torch.cat([torch.arange(1, 256), torch.tensor([1.0, 3.0, 49.0]) * 2.0 ** 40, torch.tensor([5.0, 77.0]) * 2.0 ** -40])
    x = c[:, None].expand(-1, H) * torch.where(torch.arange(H) % 3 == 1, -1.0, 1.0)
    x = x.to(BF)
    assert torch.equal(x[:, 0].float(), c.float())
    w = weight(H)
    res = None if residual is None else torch.zeros_like(x, dtype=residual)
    out = sonicmoe.rms_norm(x.to(DEV), w.to(DEV), None if res is None else res.to(DEV), eps=0.0)
    y = out if res is None else out[0]
    assert torch.equal(nearest(x, w, 0.0)[0].abs(), O.bf16(w.double()))
    assert torch.equal(y.cpu(), nearest(x, w, 0.0))


@pytest.mark.parametrize("H", [96, 1000, 4096, 5120])
def test_payloads(sonicmoe, H):
    x = torch.arange(1, 256).to(BF)[:, None].expand(-1, H).contiguous()
    w = weight(H)
    for scales in ("mx", "block128")[H % 32 != 0:]:
        got = sonicmoe.rms_norm_quantized(x.to(DEV), w.to(DEV), eps=0.0, scales=scales, with_output=True)
        assert torch.equal(got.y.cpu(), nearest(x, w, 0.0))
        q, s = sonicmoe.ops.quant_rows(got.y)[:2] if scales == "mx" else sonicmoe.ops.quant128_rows(got.y)
        assert torch.equal(got.payload.view(torch.uint8), q.view(torch.uint8)) and torch.equal(got.scales, s)


@pytest.mark.parametrize("H", [96, 1000, 4096])
def test_other_roots(sonicmoe, H):
    """A mean of 25 of values 1 and 7, of 16 and an eps of 9: values of a fifth, times weights that undo it."""
    x = torch.where(torch.arange(H) % 2 == 0, 1.0, 7.0)[None].to(BF)
    w = weight(H, 5.0)
    y = sonicmoe.rms_norm(x.to(DEV), w.to(DEV), eps=0.0).cpu()
    assert torch.equal(y, nearest(x, w, 0.0)) and torch.equal(y[0, ::2], O.bf16(w.double() / 5)[::2])
    x = torch.full((3, H), 4.0).to(BF)
    w = weight(H, 1.25)
    y = sonicmoe.rms_norm(x.to(DEV), w.to(DEV), eps=9.0).cpu()
    assert torch.equal(y, nearest(x, w, 9.0)) and torch.equal(y[1], O.bf16(w.double() / 1.25))
