"""The norm in front of the experts against 64 bits: sums, rows, payloads, gradients."""
import pytest
import torch

from oracle import block128 as B
from oracle import norm as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24                       # half a step of f32, relative
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def sonicmoe():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import sonicmoe as m
    yield m
    torch.cuda.synchronize()


def make(T, H, tx, tr, tw, seed=0):
    g = torch.Generator().manual_seed(seed * 1000 + T * 7 + H)
    size = torch.exp2(torch.randint(-12, 12, (T, 1), generator=g).float())
    x = (torch.randn(T, H, generator=g) * size).to(tx)
    w = (1 + 0.3 * torch.randn(H, generator=g)).to(tw)
    res = None if tr is None else (torch.randn(T, H, generator=g) * size * 2).to(tr)
    dy = torch.randn(T, H, generator=g).to(tx)
    dh = None if tr is None else torch.randn(T, H, generator=g).to(tr)
    return x, w, res, dy, dh


def on(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


def within(got, want, bound):
    """Every value within its bound, NaN and infinities where they are wanted."""
    got = got.double().cpu()
    ok = ((got - want).abs() <= bound) | (got == want) | (got.isnan() & want.isnan())
    assert ok.all(), ((got - want).abs() / bound.clamp(min=1e-300))[~ok].max()


def rounded(want, dtype, err):
    """Bound of a result that was off by `err` before it was rounded to its type."""
    half = torch.finfo(dtype).eps / 2
    return err + half * (want.abs() + err) + torch.finfo(dtype).smallest_normal * half


TYPES = [(BF, None, BF), (BF, BF, BF), (BF, F32, F32), (F32, None, BF), (F32, F32, F32)]
SIZES = [(1, 1), (1, 4096), (3, 7), (130, 8), (17, 250), (33, 512), (5, 513), (9, 1001), (20, 2048), (3, 4104), (2, 8192), (3, 8200), (1, 16384)]


def check_forward(y, h, x, w, res, eps):
    want_h = O.total(x, res)
    if res is not None:
        assert h.dtype == res.dtype and torch.equal(h.cpu(), want_h)
    want, _ = O.rms_norm(want_h, w, eps)
    assert y.dtype == x.dtype and y.shape == x.shape
    if x.dtype == BF:
        assert torch.equal(y.cpu(), O.bf16(want))
    else:
        # r, and two products; below 2^-126 a product is off by up to 2^-150 instead, the first one's error times the weight
        within(y, want, 4 * U * want.abs() + (1 + w.double().abs()) * 2.0 ** -150)


@pytest.mark.parametrize("T,H", SIZES)
@pytest.mark.parametrize("tx,tr,tw", TYPES)
def test_rows_and_sums(sonicmoe, T, H, tx, tr, tw):
    x, w, res, _, _ = make(T, H, tx, tr, tw)
    out = sonicmoe.rms_norm(*on(x, w, res), eps=1e-5)
    y, h = (out, None) if res is None else out
    check_forward(y, h, x, w, res, 1e-5)


def test_many_rows_beside_borders(sonicmoe):
    """Four million values, some 500 of which an f32 product leaves on the wrong side of a border or on it."""
    x, w, res, _, _ = make(1024, 4096, BF, BF, BF, seed=3)
    y, h = sonicmoe.rms_norm(*on(x, w, res))
    check_forward(y, h, x, w, res, 1e-6)


@pytest.mark.parametrize("eps", [0.0, 1e-6, 0.5])
@pytest.mark.parametrize("size", [1e-38, 1e-30, 1e-12, 1.0, 1e15, 1e25, 3e37])
def test_magnitudes(sonicmoe, eps, size):
    g = torch.Generator().manual_seed(4)
    for tx in (BF, F32):
        x = (torch.randn(6, 320, generator=g).clamp(-3, 3) * size).to(tx)
        w = torch.randn(320, generator=g).to(BF)
        y = sonicmoe.rms_norm(*on(x, w), eps=eps)
        check_forward(y, None, x, w, None, eps)
        if size >= 1e-30:                                     # below, products of f32 that are no normal numbers lose bits
            dy = torch.randn(6, 320, generator=g).to(tx)
            check_backward(sonicmoe, x, w, None, dy, None, eps)


def test_zero_rows_nan_and_infinity(sonicmoe):
    x = torch.ones(5, 96, dtype=BF)
    x[0] = 0
    x[1, 3] = float("nan")
    x[2, 4] = float("inf")
    x[3] = -0.0
    w = torch.ones(96, dtype=BF)
    y = sonicmoe.rms_norm(*on(x, w), eps=1e-6).cpu()
    assert torch.equal(y[0], torch.zeros(96, dtype=BF)) and (y[3] == 0).all() and y[3].signbit().all()
    assert y[1].isnan().all()
    assert y[2, 4].isnan() and (y[2, :4] == 0).all()
    assert torch.equal(y[4], O.bf16(O.rms_norm(x[4:], w, 1e-6)[0])[0])
    assert sonicmoe.rms_norm(*on(x[:1], w), eps=0.0).isnan().all()          # 0 / 0


# ------------------------------------------------------------------------------------------------ gradients
def check_backward(sonicmoe, x, w, res, dy, dh, eps, main_grad=False):
    dx_, dw_, dres_ = None, None, None
    gx, gw, gres = on(x, w, res)
    for t in (gx, gw) + (() if gres is None else (gres,)):
        t.requires_grad_(True)
    if main_grad:
        gw = torch.nn.Parameter(gw.detach())
        gw.main_grad = torch.full(gw.shape, 2.0, device=DEV)
    out = sonicmoe.rms_norm(gx, gw, gres, eps=eps)
    leaves = (gx,) + (() if gres is None else (gres,))
    outs, grads = ((out,), (dy.to(DEV),)) if gres is None else (out, (dy.to(DEV), dh.to(DEV)))
    if main_grad:
        torch.autograd.backward(outs, grads)
        assert gw.grad is None
        dx_, dres_, dw_ = gx.grad, None if gres is None else gres.grad, gw.main_grad - 2
    else:
        got = torch.autograd.grad(outs, leaves + (gw,), grads)
        dx_, dres_, dw_ = got[0], got[1] if gres is not None else None, got[-1]
    h = O.total(x, res)
    want, want_w = O.rms_norm_backward(h, w, eps, dy, dh)
    H = x.shape[1]
    _, r = O.rms_norm(h, w, eps)
    g, hr = (dy.double() * w.double()).abs(), (h.double() * r).abs()
    # s sums H products in f32, at most 32 a thread and then over 5 + 16 steps; each of its terms and what it is multiplied with
    # has some roundings of its own
    err = U * (r * (6 * g + hr * (g * hr).mean(1, keepdim=True) * (32 + 21 + 12)) + 2 * want.abs()
               + (0 if dh is None else 2 * dh.double().abs()))
    assert dx_.dtype == x.dtype
    within(dx_, want, rounded(want, x.dtype, err))
    if dres_ is not None:
        assert dres_.dtype == res.dtype
        within(dres_, want, rounded(want, res.dtype, err))
    terms = (dy.double() * h.double() * r).abs().sum(0)
    err_w = U * (min(x.shape[0], 256) + 8 + 4) * terms
    tw = F32 if main_grad else w.dtype
    within(dw_, want_w, rounded(want_w, tw, err_w + (8 * U * (want_w.abs() + 2) if main_grad else 0)))


@pytest.mark.parametrize("T,H", SIZES + [(700, 72), (2500, 264), (0, 128)])
@pytest.mark.parametrize("tx,tr,tw", TYPES)
def test_gradients(sonicmoe, T, H, tx, tr, tw):
    x, w, res, dy, dh = make(T, H, tx, tr, tw, seed=1)
    check_backward(sonicmoe, x, w, res, dy, dh, 1e-5)


# rows that share a warp: from one value on, the last warp and the last block not full, more rows than one turn of all blocks
NARROW = [(1, 2), (33, 1), (7, 16), (333, 24), (50, 64), (1001, 72), (77, 95), (300, 128), (131, 136), (64, 255), (3001, 256), (90001, 8),
          (20011, 100), (13000, 256)]


@pytest.mark.parametrize("T,H", NARROW)
@pytest.mark.parametrize("tx,tr,tw", TYPES)
def test_narrow_rows(sonicmoe, T, H, tx, tr, tw):
    x, w, res, dy, dh = make(T, H, tx, tr, tw, seed=3)
    out = sonicmoe.rms_norm(*on(x, w, res), eps=1e-5)
    y, h = (out, None) if res is None else out
    check_forward(y, h, x, w, res, 1e-5)
    check_backward(sonicmoe, x, w, res, dy, dh, 1e-5)


# rows of three, five, six, seven (of eight), nine and thirteen warps, several of them a block and several turns of all blocks
@pytest.mark.parametrize("T,H", [(37, 1536), (1901, 2560), (11, 2880), (1000, 2817), (950, 3584), (601, 5120), (5, 6656), (160, 9216), (3, 13000)])
@pytest.mark.parametrize("tx,tr,tw", [(BF, BF, BF), (BF, F32, F32), (F32, None, BF), (F32, F32, F32)])
def test_rows_of_any_number_of_warps(sonicmoe, T, H, tx, tr, tw):
    x, w, res, dy, dh = make(T, H, tx, tr, tw, seed=5)
    out = sonicmoe.rms_norm(*on(x, w, res), eps=1e-5)
    check_forward(*((out, None) if res is None else out), x, w, res, 1e-5)
    check_backward(sonicmoe, x, w, res, dy, dh, 1e-5)
    if tx == BF and H % 32 == 0:
        for scales, quantise in (("mx", lambda y: sonicmoe.ops.quant_rows(y)[:2]), ("block128", sonicmoe.ops.quant128_rows)):
            got = sonicmoe.rms_norm_quantized(*on(x, w, res), eps=1e-5, scales=scales, with_output=True)
            q, s = quantise(got.y)
            assert torch.equal(got.y.cpu(), (out if res is None else out[0]).cpu())
            assert torch.equal(got.payload.view(torch.uint8), q.view(torch.uint8)) and torch.equal(got.scales, s)


@pytest.mark.parametrize("H", [24, 64, 100, 256])
def test_a_narrow_row_of_nan_is_alone(sonicmoe, H):
    """Rows of one warp share nothing, forward and backward; only the weight's gradient takes all of them in."""
    x, w, res, dy, dh = on(*make(70, H, BF, F32, F32, seed=4))
    bad = [0, 13, 38, 69]
    px = x.clone()
    px[bad] = torch.tensor([float("nan"), float("inf"), 0.0, float("nan")], device=DEV, dtype=BF)[:, None]
    keep = [i for i in range(70) if i not in bad]

    def grads(x):
        x, r = x.clone().requires_grad_(True), res.clone().requires_grad_(True)
        y, h = sonicmoe.rms_norm(x, w, r)
        return y.detach(), h.detach(), *torch.autograd.grad((y, h), (x, r), (dy, dh))

    for a, b in zip(grads(x), grads(px)):
        assert torch.equal(a[keep], b[keep])
    if H % 8 == 0:
        for scales in ("mx", "block128")[H % 32 != 0:]:
            a, b = (sonicmoe.rms_norm_quantized(v, w, res, scales=scales) for v in (x, px))
            assert torch.equal(a.payload.view(torch.uint8)[keep], b.payload.view(torch.uint8)[keep]) and torch.equal(a.scales[keep], b.scales[keep])


def test_heads_norm_in_place_of_a_view(sonicmoe):
    """Queries and keys as they lie in one projection: [tokens, heads, 128] with a stride, forward and backward."""
    T, heads, D = 45, 6, 128
    g = torch.Generator().manual_seed(8)
    qkv = torch.randn(T, 3 * heads * D, generator=g).to(BF)
    w, dy = (1 + torch.randn(D, generator=g) * 0.1).to(BF), torch.randn(T, heads, D, generator=g).to(BF)
    dq, dw = qkv.to(DEV).requires_grad_(True), w.to(DEV).requires_grad_(True)
    y = sonicmoe.rms_norm(dq[:, heads * D:2 * heads * D].view(T, heads, D), dw)
    gq, gw = torch.autograd.grad(y, (dq, dw), dy.to(DEV))
    k = qkv[:, heads * D:2 * heads * D].reshape(-1, D)
    assert torch.equal(y.cpu().view(-1, D), O.bf16(O.rms_norm(k, w, 1e-6)[0]))
    want, _ = O.rms_norm_backward(k, w, 1e-6, dy.view(-1, D), None)
    assert (gq[:, :heads * D] == 0).all() and (gq[:, 2 * heads * D:] == 0).all()
    got = gq[:, heads * D:2 * heads * D].cpu().double().reshape(-1, D)
    r = O.rms_norm(k, w, 1e-6)[1]
    gr, hr = (dy.view(-1, D).double() * w.double()).abs(), (k.double() * r).abs()
    err = U * (r * (6 * gr + hr * (gr * hr).mean(1, keepdim=True) * (32 + 21 + 12)) + 2 * want.abs())      # as in check_backward
    within(got, want, rounded(want, BF, err))


def test_weight_gradient_goes_to_main_grad(sonicmoe):
    for tw in (BF, F32):
        x, w, res, dy, dh = make(33, 520, BF, F32, tw, seed=2)
        check_backward(sonicmoe, x, w, res, dy, dh, 1e-6, main_grad=True)


def test_main_grad_where_the_sum_alone_is_used(sonicmoe):
    x, w, res, dy, dh = make(5, 136, BF, BF, F32, seed=4)
    p = torch.nn.Parameter(w.to(DEV))
    p.main_grad = torch.full((136,), 3.0, device=DEV)
    calls = []
    p._apply_backward_hook = lambda: calls.append(1)
    gx = x.to(DEV).requires_grad_(True)
    y, h = sonicmoe.rms_norm(gx, p, res.to(DEV))
    h.backward(dh.to(DEV))
    assert p.grad is None and (p.main_grad == 3).all() and calls == [1] and torch.equal(gx.grad.cpu(), dh)
    y, h = sonicmoe.rms_norm(gx, p, res.to(DEV))
    y.backward(dy.to(DEV))
    assert p.grad is None and calls == [1, 1] and (p.main_grad != 3).any()


def test_long_column_sums(sonicmoe):
    """More rows than a block adds up in one f32 sum."""
    T = 300_000
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn(T, 64, generator=g, device=DEV).to(BF)
    w = torch.ones(64, dtype=F32, device=DEV, requires_grad=True)
    dy = (torch.rand(T, 64, generator=g, device=DEV)).to(BF)
    dw, = torch.autograd.grad(sonicmoe.rms_norm(x, w), w, dy)
    _, want = O.rms_norm_backward(x, w.detach(), 1e-6, dy)
    terms = (dy.double() * x.double()).abs().sum(0) * 2
    within(dw, want.cpu(), (U * (256 + 12) * terms + U * want.abs()).cpu())


def test_gradients_one_at_a_time_and_of_the_sum_alone(sonicmoe):
    x, w, res, dy, dh = make(5, 136, BF, F32, BF, seed=5)
    want, want_w = O.rms_norm_backward(O.total(x, res), w, 1e-6, dy)
    for which in range(3):
        ts = on(x, w, res)
        ts[which].requires_grad_(True)
        y, h = sonicmoe.rms_norm(*ts)
        assert y.requires_grad
        got, = torch.autograd.grad(y, ts[which], dy.to(DEV))
        ref = (want, want_w, want)[which]
        assert got.dtype == ts[which].dtype
        assert ((got.cpu().double() - ref).norm() / ref.norm()) < 2.0 ** -8
    ts = [t.requires_grad_(True) for t in on(x, w, res)]
    y, h = sonicmoe.rms_norm(*ts)
    gx, gw, gr = torch.autograd.grad(h, ts, dh.to(DEV))
    assert torch.equal(gx.cpu(), dh.to(BF)) and torch.equal(gr.cpu(), dh) and not gw.any()


def test_gradients_are_not_differentiated_again(sonicmoe):
    x, w, _, dy, _ = make(5, 136, F32, None, F32, seed=5)
    for main_grad in (False, True):
        gx, gw, gdy = (t.requires_grad_(True) for t in on(x, w, dy))
        if main_grad:
            gw.main_grad = torch.zeros(136, device=DEV)
        dx, = torch.autograd.grad(sonicmoe.rms_norm(gx, gw), gx, gdy, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiate"):
            dx.sum().backward()


def test_gradients_against_differences(sonicmoe):
    x, w, _, dy, _ = make(4, 96, F32, None, F32, seed=6)
    x = x / x.norm(dim=1, keepdim=True) * 10
    g = torch.Generator().manual_seed(9)
    vx, vw = torch.randn(4, 96, generator=g), torch.randn(96, generator=g)
    gx, gw = (t.to(DEV).requires_grad_(True) for t in (x, w))
    dx, dw = torch.autograd.grad(sonicmoe.rms_norm(gx, gw), (gx, gw), dy.to(DEV))
    along = (dx.cpu().double() * vx).sum() + (dw.cpu().double() * vw).sum()
    d = 2.0 ** -7
    ends = [((x + s * d * vx), (w + s * d * vw)) for s in (1, -1)]          # as rounded to f32: the same for both
    kernel = [(sonicmoe.rms_norm(*on(*e)).cpu().double() * dy).sum() for e in ends]
    exact = lambda s: (O.rms_norm(x.double() + s * vx, w.double() + s * vw, 1e-6)[0] * dy).sum()
    wide, narrow = (exact(d) - exact(-d)) / (2 * d), (exact(d / 2) - exact(-d / 2)) / d
    y = O.rms_norm(x, w, 1e-6)[0]
    noise = 8 * U * (y.abs() * dy.abs()).sum() / d             # results (4 U) and rounded arguments (4 U), over 2 d, twice
    assert abs((kernel[0] - kernel[1]) / (2 * d) - along) <= noise + 2 * (wide - narrow).abs() + 64 * U * (dx.cpu() * vx).abs().sum()


# ------------------------------------------------------------------------------------------------ payloads
@pytest.mark.parametrize("T,H", [(1, 32), (3, 96), (135, 64), (77, 128), (2001, 256), (9, 288), (40, 512), (7, 1056), (64, 4096), (2, 8224), (1, 16384)])
@pytest.mark.parametrize("tr", [None, BF, F32])
def test_mx_payload_is_the_row_quantisers(sonicmoe, T, H, tr):
    x, w, res, _, _ = make(T, H, BF, tr, BF, seed=7)
    got = sonicmoe.rms_norm_quantized(*on(x, w, res), with_output=True)
    check_forward(got.y, got.h, x, w, res, 1e-6)
    assert got.payload.dtype == torch.float8_e4m3fn and got.scales.shape == (T, H // 32)
    q, s, _ = sonicmoe.ops.quant_rows(got.y)
    assert torch.equal(got.payload.view(torch.uint8), q) and torch.equal(got.scales, s)
    alone = sonicmoe.rms_norm_quantized(*on(x, w, res))
    assert alone.y is None and torch.equal(alone.payload.view(torch.uint8), q) and torch.equal(alone.scales, s)


@pytest.mark.parametrize("T,H", [(1, 8), (131, 16), (135, 64), (77, 128), (3, 136), (2001, 256), (9, 264), (40, 512), (7, 1000), (64, 4096), (2, 8208), (1, 16384)])
@pytest.mark.parametrize("tr", [None, BF, F32])
def test_block128_payload_is_that_of_64_bits(sonicmoe, T, H, tr):
    x, w, res, _, _ = make(T, H, BF, tr, F32, seed=8)
    got = sonicmoe.rms_norm_quantized(*on(x, w, res), scales="block128", with_output=True)
    check_forward(got.y, got.h, x, w, res, 1e-6)
    q, s = B.quant_rows(got.y.cpu())
    assert torch.equal(got.payload.cpu().contiguous().view(torch.uint8), q.view(torch.uint8)) and torch.equal(got.scales.cpu(), s)
    q2, s2 = sonicmoe.quantize_rows_block128(got.y)
    assert torch.equal(q2.contiguous().view(torch.uint8), got.payload.contiguous().view(torch.uint8)) and torch.equal(s2, got.scales)


def test_payload_of_zeros_nan_and_infinity(sonicmoe):
    x = torch.randn(4, 256, generator=torch.Generator().manual_seed(1)).to(BF)
    x[0] = 0
    x[1, 5] = float("nan")
    x[2, 200] = float("inf")
    for scales in ("mx", "block128"):
        got = sonicmoe.rms_norm_quantized(*on(x, torch.ones(256, dtype=BF)), scales=scales, with_output=True)
        if scales == "mx":
            q, s, _ = sonicmoe.ops.quant_rows(got.y)
        else:
            q, s = sonicmoe.ops.quant128_rows(got.y)
        assert torch.equal(got.payload.view(torch.uint8), q) and torch.equal(got.scales, s)


def test_payload_in_training(sonicmoe):
    """The payload comes with rows that carry the gradient."""
    x, w, res, dy, dh = make(24, 256, BF, BF, BF, seed=10)
    gx, gw, gres = (t.requires_grad_(True) for t in on(x, w, res))
    out = sonicmoe.rms_norm_quantized(gx, gw, gres, with_output=True)
    assert out.y.requires_grad and out.h.requires_grad and not out.payload.requires_grad
    got = torch.autograd.grad((out.y, out.h), (gx, gw, gres), on(dy, dh))
    y, h = sonicmoe.rms_norm(gx, gw, gres)
    ref = torch.autograd.grad((y, h), (gx, gw, gres), on(dy, dh))
    assert torch.equal(out.y, y) and all(torch.equal(a, b) for a, b in zip(got, ref))
    with pytest.raises(ValueError, match="with_output"):
        sonicmoe.rms_norm_quantized(gx, gw, gres)


# ------------------------------------------------------------------------------------------------ callers
def test_leading_dimensions_strides_and_offsets(sonicmoe):
    x, w, res, dy, dh = make(24, 264, BF, BF, BF, seed=11)
    y0, h0 = sonicmoe.rms_norm(*on(x, w, res))
    for lead in ((2, 3, 4), (24, 1)):
        y, h = sonicmoe.rms_norm(x.to(DEV).view(*lead, 264), w.to(DEV), res.to(DEV).view(*lead, 264))
        assert y.shape == h.shape == (*lead, 264) and torch.equal(y.view(24, 264), y0) and torch.equal(h.view(24, 264), h0)
        q = sonicmoe.rms_norm_quantized(x.to(DEV).view(*lead, 264), w.to(DEV), scales="block128")
        assert q.payload.shape == (*lead, 264) and q.scales.shape == (*lead, 3) and q.h is None
    one = sonicmoe.rms_norm(x[0].to(DEV), w.to(DEV))
    assert one.shape == (264,) and torch.equal(one, sonicmoe.rms_norm(*on(x[:1], w))[0])
    # views: rows far apart, off a 16-byte boundary, columns of a larger table, transposed, one row for all
    wide = torch.randn(24, 800, device=DEV).to(BF)
    for view in (wide[:, 3:267], wide[:, 8:272], wide[::2, 5:], wide.T[:264, :].T, wide[:1, :264].expand(24, 264)):
        ref = view.contiguous()
        wt = torch.ones(view.shape[1], device=DEV, dtype=BF)
        leaf = view.detach().requires_grad_(True)
        a, b = sonicmoe.rms_norm(leaf, wt), sonicmoe.rms_norm(ref, wt)
        assert torch.equal(a, b)
        d = torch.randn(*view.shape, device=DEV).to(BF)
        leaf2 = ref.clone().requires_grad_(True)
        assert torch.equal(torch.autograd.grad(a, leaf, d)[0], torch.autograd.grad(sonicmoe.rms_norm(leaf2, wt), leaf2, d)[0])
    # a weight off a 16-byte boundary, gradients that are views
    flat = torch.ones(1 + 264, device=DEV)
    flat[1:] = w.to(DEV)
    assert torch.equal(sonicmoe.rms_norm(x.to(DEV), flat[1:]), sonicmoe.rms_norm(*on(x, w)))
    leaf = x.to(DEV).requires_grad_(True)
    d = torch.randn(264, 24, device=DEV).to(BF)
    g1, = torch.autograd.grad(sonicmoe.rms_norm(leaf, w.to(DEV)), leaf, d.T)
    g2, = torch.autograd.grad(sonicmoe.rms_norm(leaf, w.to(DEV)), leaf, d.T.contiguous())
    assert torch.equal(g1, g2)
    empty = sonicmoe.rms_norm(x[:0].to(DEV), w.to(DEV))
    assert empty.shape == (0, 264)


def test_rows_are_left_alone_and_runs_are_equal(sonicmoe):
    x, w, res, dy, dh = make(500, 520, BF, BF, BF, seed=12)
    gx, gw, gres = (t.requires_grad_(True) for t in on(x, w, res))
    runs = []
    for _ in range(3):
        y, h = sonicmoe.rms_norm(gx, gw, gres)
        runs.append((y, h, *torch.autograd.grad((y, h), (gx, gw, gres), on(dy, dh))))
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(r, runs[0]))
    assert torch.equal(gx.detach().cpu(), x) and torch.equal(gres.detach().cpu(), res)


def test_on_another_stream_and_in_a_graph(sonicmoe):
    make_ = lambda seed: on(*make(37, 256, BF, BF, BF, seed=seed))

    def step(x, w, res, dy, dh):
        o = sonicmoe.rms_norm_quantized(x, w, res, with_output=True)
        return [o.payload.view(torch.uint8), o.scales, o.y.detach(), *torch.autograd.grad((o.y, o.h), (x, w, res), (dy, dh))]

    def leaves(seed):
        t = make_(seed)
        return [v.requires_grad_(True) for v in t[:3]] + t[3:]

    wants = [[v.clone() for v in step(*leaves(s))] for s in (20, 21)]
    static = leaves(22)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert all(torch.equal(a, b) for a, b in zip(step(*leaves(20)), wants[0]))
        step(*static)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(*static)
    for s, want in zip((20, 21), wants):
        with torch.no_grad():
            for a, b in zip(static, make_(s)):
                a.copy_(b)
        graph.replay()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_rows_beyond_32_bit_offsets(sonicmoe):
    T, H = 300_000, 8192                                     # 2.4e9 values
    x = torch.zeros(T, H, dtype=BF, device=DEV)
    picks = [0, 131_071, 131_072, 262_143, 262_144, T - 1]
    rows = torch.randn(len(picks), H, generator=torch.Generator().manual_seed(2)).to(BF)
    for i, p in enumerate(picks):
        x[p] = rows[i].to(DEV)
    w = torch.ones(H, dtype=BF, device=DEV)
    y = sonicmoe.rms_norm(x, w)
    want = O.bf16(O.rms_norm(rows, torch.ones(H), 1e-6)[0])
    assert torch.equal(y[picks].cpu(), want)
    assert not y[1:131_071:997].any()
    leaf = x.requires_grad_(True)
    d, = torch.autograd.grad(sonicmoe.rms_norm(leaf, w), leaf, y)
    ref, _ = O.rms_norm_backward(rows, torch.ones(H), 1e-6, want)
    # g = dy is nearly the unit row itself: what is left is the difference of two numbers as large as dy r
    _, r = O.rms_norm(rows, torch.ones(H), 1e-6)
    within(d[picks], ref, rounded(ref, BF, U * r * want.double().abs() * 128))
