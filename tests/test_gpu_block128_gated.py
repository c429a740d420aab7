"""The gated row quantiser against its definition in 64 bits: payloads are the same numbers, however an exponential is rounded."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def sonicmoe():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import sonicmoe as m
    return m


def definition(z):
    """Products of the activation with 448 / a in 64 bits, rounded to f32 and to e4m3, and the scales; by blocks of 128."""
    rows, K = z.shape[0], z.shape[1] // 2
    g, u = z[:, 0::2].double(), z[:, 1::2].double()
    y = g / (1 + torch.exp(-g)) * u
    pad = torch.zeros(rows, -K % 128, dtype=y.dtype, device=y.device)
    y = torch.cat([y, pad], 1).unflatten(1, (-1, 128))
    a = y.abs().amax(2).float().clamp(min=2.0 ** -100)
    top = torch.full_like(a, 448.0)                            # a quotient of tensors is rounded once
    v = (y * (top / a).double()[:, :, None]).flatten(1)[:, :K]
    return v, v.float().to(torch.float8_e4m3fn), a / top


@pytest.mark.parametrize("rows,K", [(1, 8), (3, 136), (130, 720), (4096, 768), (16384, 768)])
@pytest.mark.parametrize("spread", [1.0, 2.0])
def test_payload_of_the_definition(sonicmoe, rows, K, spread):
    g = torch.Generator(device=DEV).manual_seed(rows + K)
    for _ in range(3):
        z = torch.randn(rows, 2 * K, generator=g, device=DEV) * spread
        z[:, 1::2] *= torch.exp2(torch.randint(-20, 20, (rows, 1), generator=g, device=DEV).float())
        z = z.to(torch.bfloat16)
        q, s = sonicmoe.quantize_rows_block128(z, swiglu=True)
        v, ref, scale = definition(z)
        differ = q.float() != ref.float()
        # e4m3 has one step, 2^-9, below 2^-6; nothing looks for a border there
        assert not (differ & (v.abs() >= 2.0 ** -6)).any()
        assert ((q.float() - ref.float()).abs()[differ] <= 2.0 ** -9).all()
        # the activation of a block's largest value: 4e-7 and 8e-8 |g| with |g| <= 10, two products and a quotient of f32
        assert ((s.double() - scale.double()).abs() <= 2.0 ** -19 * scale.double()).all()


def test_blocks_of_one_value_and_without_one(sonicmoe):
    """Every value of a block is its largest; zeros; values below the floor of a maximum; infinities and NaN beside numbers."""
    z = torch.zeros(8, 2 * 256)
    z[0] = 1.0                                                 # silu(1) everywhere
    z[1, 0::2], z[1, 1::2] = -0.75, 3.0
    z[2, 0::2], z[2, 1::2] = 1.0, 2.0 ** -120
    z[3, 0::2], z[3, 1::2] = 2.0, 1.0
    z[3, 4] = float("nan")
    z[4, 0::2], z[4, 1::2] = 2.0, 1.0
    z[4, 4] = float("inf")
    z[5, 0::2], z[5, 1::2] = -100.0, 1.0
    z = z.to(torch.bfloat16).to(DEV)
    q, s = sonicmoe.quantize_rows_block128(z, swiglu=True)
    q = q.float()
    for r in (0, 1):                                           # the largest is held as 448
        assert (q[r].abs() == 448).all()
    assert (q[2] == 0).all() and (q[6:] == 0).all()
    assert torch.isnan(q[3, 2]) and (q[3, 128:] == 448).all() and torch.isfinite(s[3]).all()
    assert (q[3, :2] == 448).all() and (q[3, 3:128] == 448).all()      # NaN is no magnitude
    assert torch.isinf(s[4, 0]) and (q[4, 128:] == 448).all()
    assert torch.isfinite(q[5]).all()
