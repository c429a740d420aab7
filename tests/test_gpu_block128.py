"""Quantisers and products with a scale per block of 128 against 64 bits."""
import pytest
import torch

from oracle import block128 as O
from oracle import group_routing as G

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = 2.0 ** -8                     # half a step of bf16, relative


@pytest.fixture(scope="module")
def sonicmoe():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import sonicmoe as m
    yield m
    torch.cuda.synchronize()
    m.ops.check_status(DEV)


def f32_tol(K, blocks):
    """Roundings of a sum of K products in f32, whatever their order, of the scales' product and of adding blocks, relative to the
    sum of the terms' magnitudes; twice 2^-24 each, for an adder that cuts instead of rounding."""
    return (min(K, 128) + blocks + 4) * 2.0 ** -23


def randn(*shape, seed=0, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(torch.bfloat16)


def spread(*shape, seed=0):
    """Values over many magnitudes, with zeros."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * torch.exp2(torch.randint(-30, 20, (shape[0],) + (1,) * (len(shape) - 1), generator=g).float())
    return torch.where(torch.rand(*shape, generator=g) < 0.1, torch.zeros(()), x).to(torch.bfloat16)


def same(q, s, ref):
    assert torch.equal(q.cpu().contiguous().view(torch.uint8), ref[0].view(torch.uint8))
    assert torch.equal(s.cpu(), ref[1])


def table(counts, tail=0):
    """Segments of 128-row multiples -> (efo, counts, rows)."""
    efo = torch.zeros(len(counts) + 1, dtype=torch.int32)
    efo[1:] = torch.tensor([-(-c // 128) * 128 for c in counts]).cumsum(0)
    return efo, torch.tensor(counts, dtype=torch.int32), int(efo[-1]) + tail


# ------------------------------------------------------------------------------------------------ quantisers
@pytest.mark.parametrize("rows,K", [(1, 8), (3, 128), (17, 136), (128, 256), (130, 720), (257, 1000), (5, 4104)])
def test_quantisers_bit_for_bit(sonicmoe, rows, K):
    for seed, make in enumerate((randn, spread)):
        x = make(rows, K, seed=seed + rows)
        q, s = sonicmoe.quantize_rows_block128(x.to(DEV))
        assert q.dtype == torch.float8_e4m3fn and s.shape == (rows, -(-K // 128))
        same(q, s, O.quant_rows(x))
        q, s, qc, sc = sonicmoe.ops.quant128_dual(x.to(DEV))
        same(q, s, O.quant_rows(x))
        same(qc.T, sc, O.quant_cols(x))
        w = make(3, rows, K, seed=seed + K)
        q, s = sonicmoe.quantize_weight_block128(w.to(DEV))
        same(q, s, O.quant_weight(w))
        q, s = sonicmoe.quantize_weight_block128(w[0].to(DEV))
        assert q.shape == (rows, K)
        same(q, s, [t[0] for t in O.quant_weight(w[:1])])


def test_quantisers_on_zeros_tiny_values_infinity_and_nan(sonicmoe):
    x = torch.zeros(4, 256, dtype=torch.bfloat16)
    x[1] = 2.0 ** -130                                        # below the floor of a maximum
    x[2, 5], x[2, 200] = float("nan"), 3.0
    x[2, :5] = torch.tensor([1.0, -2.0, 0.5, 7.0, -448.0])
    x[3] = 1.0
    x[3, 130] = float("inf")
    q, s = (t.cpu() for t in sonicmoe.quantize_rows_block128(x.to(DEV)))
    ref_q, ref_s = O.quant_rows(x)
    assert torch.equal(s, ref_s) and torch.isinf(s[3, 1])
    f, r = q.float(), ref_q.float()
    assert torch.equal(torch.isnan(f), torch.isnan(r)) and torch.equal(f[~torch.isnan(f)], r[~torch.isnan(r)])
    assert torch.isnan(f[2, 5]) and (f[2, :5] == x[2, :5].float()).all()      # NaN leaves its block alone


def test_column_form_of_segments(sonicmoe):
    efo, counts, rows = table([130, 0, 1, 128, 300], tail=128)
    x = randn(rows, 264, seed=1)
    live = O.live_rows(efo, counts, rows)
    x[~live] = float("nan")                                   # what is not live counts as zero
    q, s, qc, sc = sonicmoe.ops.quant128_dual(x.to(DEV), efo.to(DEV), counts.to(DEV))
    ref_q, ref_s = O.quant_cols(x, live)
    busy = live.view(-1, 128).any(1)
    assert torch.equal(sc.cpu()[busy], ref_s[busy])
    keep = busy.repeat_interleave(128)
    assert torch.equal(qc.cpu().T[keep], ref_q.view(torch.uint8)[keep])
    want = O.quant_rows(x[live])
    assert torch.equal(q.cpu()[live].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(s.cpu()[live], want[1])


@pytest.mark.parametrize("rows,I", [(1, 8), (33, 136), (129, 768)])
def test_gated_activation_is_quantised_within_half_a_step(sonicmoe, rows, I):
    z = randn(rows, 2 * I, seed=I, scale=3.0)
    q, s = (t.cpu() for t in sonicmoe.quantize_rows_block128(z.to(DEV), swiglu=True))
    y, got = O.swiglu(z), O.deq_rows(q, s)
    per = s.double().repeat_interleave(128, 1)[:, :I]
    # half a step of e4m3 (2^-4 of the value, 2^-10 below its normal range) and the roundings of the activation and of the scaling
    assert ((got - y).abs() <= 2.0 ** -4 * y.abs() * (1 + 1e-5) + per * 2.0 ** -10 + 1e-5 * y.abs()).all()
    amax = torch.stack([y[:, a:a + 128].abs().amax(1) for a in range(0, I, 128)], 1)
    assert ((s.double() - amax / 448).abs() <= 16 * 2.0 ** -24 * amax / 448 + 1e-33).all()


def test_listed_rows_and_scattered_tokens(sonicmoe):
    T, K, E, H = 37, 3, 8, 200
    g = torch.Generator().manual_seed(2)
    idx = torch.rand(T, E, generator=g).topk(K).indices.int()
    idx[torch.rand(T, K, generator=g) < 0.3] = -1
    md = sonicmoe.ops.topk_metadata(idx.to(DEV), torch.rand(T, K, generator=g).to(DEV), E, 128)
    x = randn(T, H, seed=3)
    q, s = sonicmoe.ops.quant128_rows_scatter(x.to(DEV), md["naept"], md["s_reverse_scatter_idx"], md["TKp_alloc"])
    n = int(md["naept"][-1])
    places = md["s_reverse_scatter_idx"][:n].long().cpu()
    tokens = md["x_gather_idx"].cpu().long()[places]
    ref = O.quant_rows(x)
    assert torch.equal(q.cpu().view(torch.uint8)[places], ref[0].view(torch.uint8)[tokens]) and torch.equal(s.cpu()[places], ref[1][tokens])
    z = randn(md["TKp_alloc"], 2 * H, seed=4).to(DEV)
    whole = sonicmoe.ops.quant128_rows(z, True)
    some = sonicmoe.ops.quant128_rows(z, True, md["s_reverse_scatter_idx"], md["naept"][-1:])
    assert torch.equal(some[0].cpu()[places], whole[0].cpu()[places]) and torch.equal(some[1].cpu()[places], whole[1].cpu()[places])


# ------------------------------------------------------------------------------------------------ products
def rows_case(sonicmoe, counts, N, K, tail=0, seed=0, make=randn, few=False, efo=None):
    e, c, rows = table(counts, tail)
    e = e if efo is None else efo
    x, w = make(rows, K, seed=seed), make(len(counts), N, K, seed=seed + 1)
    live = O.live_rows(e, c, rows)
    xq, xs = sonicmoe.ops.quant128_rows(x.to(DEV))
    wq, ws = sonicmoe.ops.quant128_weight(w.to(DEV))
    xs[~live.to(DEV)] = float("nan")                          # nobody looks at what is not live
    f = sonicmoe.ops.gemm128_few if few else sonicmoe.ops.gemm128_rows
    y = f(xq, xs, wq, ws, e.to(DEV), c.to(DEV)).cpu().double()
    ref, mag = O.rows_product(O.deq_rows(*O.quant_rows(x)), O.deq_weight(*O.quant_weight(w)), e, c)
    tol = BF16 * ref.abs() + f32_tol(K, -(-K // 128)) * mag * (1 + BF16) + 1e-38
    assert ((y - ref).abs() <= tol)[live].all()
    if not few:
        assert (y[~live] == 0).all()
    return y


@pytest.mark.parametrize("counts", [[1], [128], [129], [300, 0, 5], [0, 0, 256], [128, 700, 1, 64, 0, 257]])
@pytest.mark.parametrize("N,K", [(8, 8), (128, 128), (136, 264), (256, 512), (520, 1000), (1000, 200)])
def test_rows_by_segments(sonicmoe, counts, N, K):
    rows_case(sonicmoe, counts, N, K, tail=128 * (len(counts) % 2), seed=N + K)
    rows_case(sonicmoe, counts, N, K, seed=N + K, few=True)


def test_rows_over_many_tiles_a_pair_and_many_experts(sonicmoe):
    g = torch.Generator().manual_seed(1)
    rows_case(sonicmoe, torch.randint(0, 300, (256,), generator=g).tolist(), 264, 136, tail=256)
    rows_case(sonicmoe, torch.randint(0, 90, (256,), generator=g).tolist(), 264, 136, few=True)
    rows_case(sonicmoe, [5000, 3, 2000], 1032, 328)
    rows_case(sonicmoe, [900], 2056, 1160, make=spread)


@pytest.mark.parametrize("K", [8, 128, 1024, 4104])
@pytest.mark.parametrize("rows", [1, 2, 16, 17, 63, 64, 65, 200])
def test_few_rows_share_the_reduction_among_ctas(sonicmoe, rows, K):
    """One projection: its weight tiles are few, so that one, two, four or eight CTAs work on each."""
    for N in (128, 1000, 3200):
        x, w = randn(rows, K, seed=rows), randn(1, N, K, seed=K)
        xq, xs = sonicmoe.ops.quant128_rows(x.to(DEV))
        wq, ws = sonicmoe.ops.quant128_weight(w.to(DEV))
        y = sonicmoe.ops.gemm128_few(xq, xs, wq, ws).cpu().double()
        ref, mag = O.rows_product(O.deq_rows(*O.quant_rows(x)), O.deq_weight(*O.quant_weight(w)), None, None)
        assert ((y - ref).abs() <= BF16 * ref.abs() + f32_tol(K, -(-K // 128)) * mag * (1 + BF16)).all()


def test_few_rows_leave_the_others(sonicmoe):
    efo, counts, rows = table([3, 0, 70, 128])
    xq, xs = sonicmoe.ops.quant128_rows(randn(rows, 256).to(DEV))
    wq, ws = sonicmoe.ops.quant128_weight(randn(4, 264, 256, seed=1).to(DEV))
    from sonicmoe._lib import check, lib
    for few in (True, False):
        c = torch.full((rows, 264), 7.0, dtype=torch.bfloat16, device=DEV)
        P, ops = (lambda t: t.data_ptr()), sonicmoe.ops
        e, n = efo.to(DEV), counts.to(DEV)
        head = (P(xq), P(xs), P(wq), P(ws), P(e), P(n), P(c), rows, 264, 256, 4)
        st = torch.cuda.current_stream().cuda_stream
        if few:
            check(lib.smoe_gemm128_few(*head, 0, P(ops.status_word(DEV)), None, st), "few")
        else:
            check(lib.smoe_gemm128_rows(*head, 0, 0, P(ops.status_word(DEV)), None, st), "rows")
        dead = ~O.live_rows(efo, counts, rows)
        assert (c.cpu()[dead] == 7.0).all() and (c.cpu()[~dead] != 7.0).any()


@pytest.mark.parametrize("counts", [[1], [300, 0, 5], [128, 700, 1, 64, 0, 257]])
@pytest.mark.parametrize("N,K", [(8, 16), (136, 264), (256, 512), (1000, 200)])
def test_gradient_of_the_rows_reads_the_same_weights(sonicmoe, counts, N, K):
    efo, cnt, rows = table(counts)
    dy, w = randn(rows, N, seed=N), randn(len(counts), N, K, seed=K)
    dq, ds = sonicmoe.ops.quant128_rows(dy.to(DEV))
    wq, ws = sonicmoe.ops.quant128_weight(w.to(DEV))
    dx = sonicmoe.ops.gemm128_rows(dq, ds, wq, ws, efo.to(DEV), cnt.to(DEV), b_mn=True).cpu().double()
    wd = O.deq_weight(*O.quant_weight(w)).transpose(1, 2)
    ref, mag = O.rows_product(O.deq_rows(*O.quant_rows(dy)), wd, efo, cnt)
    assert ((dx - ref).abs() <= BF16 * ref.abs() + f32_tol(N, -(-N // 128)) * mag * (1 + BF16)).all()


@pytest.mark.parametrize("counts", [[1], [300, 0, 5], [128, 700, 1, 64, 0, 257]])
@pytest.mark.parametrize("M,N", [(8, 16), (136, 264), (512, 256), (1000, 200)])
def test_weight_gradients(sonicmoe, counts, M, N):
    efo, cnt, rows = table(counts, tail=128)
    E = len(counts)
    dy, x = randn(rows, M, seed=M), spread(rows, N, seed=N)
    live = O.live_rows(efo, cnt, rows)
    dy[~live] = float("nan")
    e, c = efo.to(DEV), cnt.to(DEV)
    a, b = (sonicmoe.ops.quant128_dual(t.to(DEV), e, c, with_rows=False)[2:] for t in (dy, x))
    ref, mag = O.cols_product(O.deq_cols(*O.quant_cols(dy, live)), O.deq_cols(*O.quant_cols(x, live)), efo, cnt, E)
    tol = f32_tol(max(counts), -(-max(counts) // 128)) * mag
    got = sonicmoe.ops.gemm128_wgrad(*a, *b, e, c)
    assert got.dtype == torch.bfloat16
    assert ((got.cpu().double() - ref).abs() <= BF16 * ref.abs() + tol * (1 + BF16)).all()
    out = torch.full((E, M, N), float("nan"), device=DEV)
    assert sonicmoe.ops.gemm128_wgrad(*a, *b, e, c, out=out) is out
    assert ((out.cpu().double() - ref).abs() <= tol).all()
    once = out.clone()
    sonicmoe.ops.gemm128_wgrad(*a, *b, e, c, out=out, accumulate=True)
    assert torch.equal(out, once + once)


# ------------------------------------------------------------------------------------------------ as they are used
def linear_reference(x, w, dy, efo, counts):
    rows = x.shape[0]
    live = O.live_rows(efo, counts, rows)
    wd = O.deq_weight(*O.quant_weight(w))
    y = O.rows_product(O.deq_rows(*O.quant_rows(x)), wd, efo, counts)
    dx = O.rows_product(O.deq_rows(*O.quant_rows(dy)), wd.transpose(1, 2), efo, counts)
    dw = O.cols_product(O.deq_cols(*O.quant_cols(dy, live)), O.deq_cols(*O.quant_cols(x, live)), efo, counts, w.shape[0])
    return y, dx, dw


def near(got, ref, K):
    v, mag = ref
    assert ((got.cpu().double() - v).abs() <= BF16 * v.abs() + f32_tol(K, -(-K // 128)) * mag * (1 + BF16)).all()


@pytest.mark.parametrize("counts,N,K", [([200, 0, 70], 264, 136), ([1], 128, 256), ([640, 129], 512, 384)])
def test_linear_and_its_gradients(sonicmoe, counts, N, K):
    efo, cnt, rows = table(counts, tail=256)
    x, w, dy = randn(rows, K, seed=1), randn(len(counts), N, K, seed=2), randn(rows, N, seed=3)
    live = O.live_rows(efo, cnt, rows)
    x[~live], dy[~live] = float("nan"), float("nan")
    e, c = efo.to(DEV), cnt.to(DEV)
    xd, wd = x.to(DEV).requires_grad_(True), w.to(DEV).requires_grad_(True)
    y = sonicmoe.block128_linear(xd, wd, e, c)
    y.backward(dy.to(DEV))
    ref = linear_reference(torch.nan_to_num(x), w, torch.nan_to_num(dy), efo, cnt)
    near(y, ref[0], K)
    near(xd.grad, ref[1], N)
    near(wd.grad, ref[2], rows)
    # constant weights: the same outputs and gradient of x
    pair = sonicmoe.quantize_weight_block128(wd)
    x2 = x.to(DEV).requires_grad_(True)
    y2 = sonicmoe.block128_linear(x2, pair, e, c)
    assert torch.equal(y2, y)
    y2.backward(dy.to(DEV))
    assert torch.equal(x2.grad, xd.grad)
    with torch.no_grad():
        assert torch.equal(sonicmoe.block128_linear(xd, wd, e, c), y)
    # an f32 accumulator on the parameter
    w3 = w.to(DEV).requires_grad_(True)
    w3.main_grad = torch.ones(len(counts), N, K, device=DEV)
    sonicmoe.block128_linear(x.to(DEV), w3, e, c).backward(dy.to(DEV))
    assert w3.grad is None
    assert ((w3.main_grad.cpu().double() - 1 - ref[2][0]).abs() <= f32_tol(rows, 8) * (ref[2][1] + 1)).all()


@pytest.mark.parametrize("rows", [0, 1, 64, 65, 300])
def test_one_projection(sonicmoe, rows):
    N, K = 392, 520
    x, w, dy = randn(rows, K, seed=1), randn(N, K, seed=2), randn(rows, N, seed=3)
    xd, wd = x.to(DEV).requires_grad_(True), w.to(DEV).requires_grad_(True)
    y = sonicmoe.block128_linear(xd, wd)
    y.backward(dy.to(DEV))
    if rows == 0:
        assert y.shape == (0, N) and (wd.grad == 0).all() and xd.grad.shape == (0, K)
        return
    ref = linear_reference(x, w[None], dy, None, None)
    near(y, ref[0], K)
    near(xd.grad, ref[1], N)
    near(wd.grad, [t[0] for t in ref[2]], rows)
    if rows % 4 == 0:                                          # leading dimensions, other strides
        with torch.no_grad():
            assert torch.equal(sonicmoe.block128_linear(xd.view(4, -1, K), wd), y.view(4, -1, N))
            assert torch.equal(sonicmoe.block128_linear(x.T.contiguous().to(DEV).T, w.T.contiguous().to(DEV).T), y)


def test_linear_gradients_against_differences(sonicmoe):
    """With payloads that e4m3 holds exactly the product is linear in its inputs: its gradients are those of the plain product."""
    g = torch.Generator().manual_seed(4)
    powers = lambda *s: torch.exp2(torch.randint(-2, 3, s, generator=g).float()).mul(torch.randint(0, 2, s, generator=g) * 2 - 1)
    x, w, dy = powers(130, 256), powers(1, 136, 256), powers(130, 136)
    xd, wd = (t.bfloat16().to(DEV).requires_grad_(True) for t in (x, w))
    y = sonicmoe.block128_linear(xd, wd)
    y.backward(dy.bfloat16().to(DEV))
    f = lambda a, b: ((a @ b[0].T) * dy.double()).sum()
    a, b = x.double(), w.double()
    for t, grad, fn in ((a, xd.grad, lambda v: f(v, b)), (b, wd.grad, lambda v: f(a, v))):
        for at in ([0, 0], [1, 7], [64, 100], [127, 255]):
            at = ([0] if t.ndim == 3 else []) + at
            d = torch.zeros_like(t)
            d[tuple(at)] = 0.5
            slope = float(fn(t + d) - fn(t - d))
            mag = 512 * 16.0                                   # terms of at most 4 * 4, 136 or 130 of them, in blocks of 128
            assert abs(float(grad[tuple(at)]) - slope) <= BF16 * abs(slope) + f32_tol(256, 2) * mag + mag * 2.0 ** -20


def experts_reference(x, idx, scores, w1, w2, bf16=True):
    """64 bits, with the definition's bf16 between the products."""
    step = (lambda t: t.to(torch.bfloat16).double()) if bf16 else (lambda t: t)
    x64 = O.deq_rows(*O.quant_rows(x))
    out = torch.zeros(x.shape[0], w2.shape[1], dtype=torch.float64)
    for t in range(x.shape[0]):
        for k in range(idx.shape[1]):
            e = int(idx[t, k])
            if e >= 0:
                y = O.swiglu(step(w1[e] @ x64[t])[None]).float()
                y = O.deq_rows(*O.quant_rows(y))[0]
                out[t] += scores[t, k].double() * step(w2[e] @ y)
    return out


@pytest.mark.parametrize("T,E,K,H,I", [(1, 8, 2, 256, 128), (7, 8, 3, 264, 72), (40, 4, 2, 128, 256), (200, 3, 2, 392, 136)])
def test_experts(sonicmoe, T, E, K, H, I):
    x, w1, w2 = randn(T, H, seed=1), randn(E, 2 * I, H, seed=2, scale=H ** -0.5), randn(E, H, I, seed=3, scale=I ** -0.5)
    g = torch.Generator().manual_seed(5)
    scores, idx = torch.rand(T, E, generator=g).topk(K)
    idx = idx.int()
    if T > 1:
        idx[torch.rand(T, K, generator=g) < 0.2] = -1
        idx[0] = -1                                            # a token without an expert
    p1, p2 = (sonicmoe.quantize_weight_block128(w.to(DEV)) for w in (w1, w2))
    out = sonicmoe.block128_experts(x.to(DEV), idx.to(DEV), scores.to(DEV), p1, p2).cpu().double()
    ref = experts_reference(x, idx, scores, *(O.deq_weight(*O.quant_weight(w)) for w in (w1, w2)))
    if T > 1:
        assert (out[0] == 0).all()
    # A rounding of z to bf16 that falls the other way moves y by 2^-8 and may move its e4m3 value by a step, 2^-3: in the sum over
    # I such moves meet at random.  Bounded by the norm: if every value moved by half a step the output would by 2^-4.
    rel = (out - ref).norm() / ref.norm()
    assert rel <= 2.0 ** -6
    # as the weights' own products without any quantisation: three roundings to e4m3, 2^-4 at most and 2^-5.2 on average each
    free = experts_reference(x.float().to(torch.bfloat16), idx, scores, w1.double(), w2.double(), False)
    assert (out - free).norm() / free.norm() <= 3 * 2.0 ** -4


@pytest.mark.parametrize("T,E,K", [(1, 4, 3), (5, 2, 6), (40, 8, 3), (2100, 16, 4)])
def test_experts_named_twice_count_twice(sonicmoe, T, E, K):
    H, I = 256, 128
    x, w1, w2 = randn(T, H, seed=1), randn(E, 2 * I, H, seed=2, scale=H ** -0.5), randn(E, H, I, seed=3, scale=I ** -0.5)
    g = torch.Generator().manual_seed(T)
    idx = torch.randint(-1, E, (T, K), generator=g, dtype=torch.int32)
    idx[-1] = E - 1                                            # the last token: one expert in every slot
    scores = torch.rand(T, K, generator=g)
    p1, p2 = (sonicmoe.quantize_weight_block128(w.to(DEV)) for w in (w1, w2))
    out = sonicmoe.block128_experts(x.to(DEV), idx.to(DEV), scores.to(DEV), p1, p2).cpu().double()
    ref = experts_reference(x, idx, scores, *(O.deq_weight(*O.quant_weight(w)) for w in (w1, w2)))
    # as in test_experts, by token: e4m3 values may be half a step off, 2^-4, and the norm is over 256 of them
    assert ((out - ref).norm(dim=1) <= 2.0 ** -4 * ref.norm(dim=1)).all()
    assert (out[(idx < 0).all(1)] == 0).all()


@pytest.mark.parametrize("T,E,K", [(1000, 16, 4), (1500, 128, 8), (300, 5, 2)])
def test_experts_of_very_different_loads(sonicmoe, T, E, K):
    """Full tiles, long and short rests of them, experts of a few rows and of none, each token against its reference."""
    H, I = 264, 136
    x, w1, w2 = randn(T, H, seed=1), randn(E, 2 * I, H, seed=2, scale=H ** -0.5), randn(E, H, I, seed=3, scale=I ** -0.5)
    g = torch.Generator().manual_seed(T)
    logits = torch.randn(T, E, generator=g) + 1.5 * torch.randn(E, generator=g)
    logits[:, 1] = -100.0
    scores, idx = logits.softmax(-1).topk(K)
    p1, p2 = (sonicmoe.quantize_weight_block128(w.to(DEV)) for w in (w1, w2))
    out = sonicmoe.block128_experts(x.to(DEV), idx.int().to(DEV), scores.to(DEV), p1, p2).cpu().double()
    n = torch.bincount(idx.flatten(), minlength=E)
    assert n[1] == 0 and ((n % 256 > 0) & (n % 256 <= 64)).any() and (n % 256 > 64).any()
    ref = experts_reference(x, idx, scores, *(O.deq_weight(*O.quant_weight(w)) for w in (w1, w2)))
    assert ((out - ref).norm(dim=1) <= 2.0 ** -4 * ref.norm(dim=1)).all()      # as above


def test_router_and_experts_in_one_step(sonicmoe):
    """Route, sort, two products with an activation between them, weighted sum; outputs and all gradients against the same step in
    f32 on the values that the operators see, and the inference chain against it."""
    T, E, K, H, I = 96, 8, 3, 256, 128
    x, w1, w2 = randn(T, H, seed=1), randn(E, 2 * I, H, seed=2, scale=H ** -0.5), randn(E, H, I, seed=3, scale=I ** -0.5)
    logits = torch.randn(T, E, generator=torch.Generator().manual_seed(4))
    logits[-5:] = -torch.inf                                   # a padded batch
    bias = torch.linspace(-0.1, 0.1, E)
    dy = randn(T, H, seed=6)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w1, w2, logits)]
    xd, w1d, w2d, ld = leaves

    scores, idx = sonicmoe.group_limited_routing(ld, K, bias=bias.to(DEV), groups=4, top_groups=2, scale=1.5)
    md = sonicmoe.ops.topk_metadata(idx, scores.detach(), E, 128)
    n = int(md["naept"][-1])
    assert n == (T - 5) * K
    places, slots = md["s_reverse_scatter_idx"][:n].long(), md["score_src_idx"][:n].long()
    xs = torch.zeros(md["TKp_alloc"], H, dtype=torch.bfloat16, device=DEV).index_put((places,), xd[slots // K])
    z = sonicmoe.block128_linear(xs, w1d, md["efo"], md["counts"])
    y = (torch.nn.functional.silu(z[:, 0::2].float()) * z[:, 1::2].float()).bfloat16()
    o = sonicmoe.block128_linear(y, w2d, md["efo"], md["counts"])
    out = torch.zeros(T, H, device=DEV).index_add(0, slots // K, o[places].float() * scores.flatten()[slots][:, None])
    out.backward(dy.to(DEV).float())

    # the same in f32 on the CPU, unquantised; the choices are those of the operator (equal by its own test)
    cpu = [t.float().requires_grad_(True) for t in (x, w1, w2, logits)]
    xc, w1c, w2c, lc = cpu
    sc = G.scores_of(lc, idx.cpu(), False, True, 1.5)
    ref = torch.zeros(T, H)
    for k in range(K):
        for e in range(E):
            t = (idx[:, k].cpu() == e).nonzero().flatten()
            zc = xc[t] @ w1c[e].T
            ref = ref.index_add(0, t, sc[t, k:k + 1] * ((torch.nn.functional.silu(zc[:, 0::2]) * zc[:, 1::2]) @ w2c[e].T))
    ref.backward(dy.float())
    # e4m3 operands: each rounding is at most 2^-4 of its value; at most five of them lie on the way to a gradient
    rel = lambda a, b: float((a.detach().cpu().double() - b.double()).norm() / b.double().norm())
    assert rel(out, ref.detach()) <= 4 * 2.0 ** -4
    for a, b in zip(leaves, cpu):
        assert torch.isfinite(a.grad).all() and rel(a.grad, b.grad) <= 5 * 2.0 ** -4
    assert (xd.grad[-5:] == 0).all() and (ld.grad[-5:] == 0).all()
    pairs = [sonicmoe.quantize_weight_block128(w) for w in (w1d, w2d)]
    served = sonicmoe.block128_experts(xd.detach(), idx, scores.detach(), *pairs)
    # the served chain does not round the activation to bf16 before it quantises it
    assert rel(served, out.detach().cpu()) <= 2.0 ** -4


def test_captured_on_another_stream_and_two_at_once(sonicmoe):
    T, E, K, H, I = 48, 8, 2, 256, 128
    w1, w2 = (sonicmoe.quantize_weight_block128(randn(*s, seed=i, scale=0.06).to(DEV)) for i, s in enumerate([(E, 2 * I, H), (E, H, I)]))
    xs = [randn(T, H, seed=7 + i).to(DEV) for i in range(2)]
    idx = torch.rand(T, E, generator=torch.Generator().manual_seed(1)).topk(K).indices.int().to(DEV)
    sc = torch.full((T, K), 0.5, device=DEV)
    want = [sonicmoe.block128_experts(x, idx, sc, w1, w2) for x in xs]
    lin = [sonicmoe.block128_linear(x, (w1[0][0], w1[1][0])) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for _ in range(3):
        for x, st in zip(xs, streams):
            with torch.cuda.stream(st):
                got.append((sonicmoe.block128_experts(x, idx, sc, w1, w2), sonicmoe.block128_linear(x, (w1[0][0], w1[1][0]))))
    torch.cuda.synchronize()
    for i, (a, b) in enumerate(got):
        assert torch.equal(a, want[i % 2]) and torch.equal(b, lin[i % 2])
    # two graphs, replayed side by side with new inputs
    graphs, outs = [], []
    for x in xs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append((sonicmoe.block128_experts(x, idx, sc, w1, w2), sonicmoe.block128_linear(x, (w1[0][0], w1[1][0]))))
        graphs.append(graph)
    xs[0].copy_(xs[1].clone())
    torch.cuda.synchronize()
    for graph, st in zip(graphs, streams):
        with torch.cuda.stream(st):
            graph.replay()
    torch.cuda.synchronize()
    for a, b in outs:
        assert torch.equal(a, want[1]) and torch.equal(b, lin[1])


def test_gradients_asked_for_one_at_a_time_and_a_matrix_with_an_accumulator(sonicmoe):
    x, w, dy = randn(70, 136, seed=1).to(DEV), randn(264, 136, seed=2).to(DEV), randn(70, 264, seed=3).to(DEV)
    both = [t.clone().requires_grad_(True) for t in (x, w)]
    sonicmoe.block128_linear(*both).backward(dy)
    one = x.clone().requires_grad_(True)
    sonicmoe.block128_linear(one, w).backward(dy)
    other = w.clone().requires_grad_(True)
    other.main_grad = torch.zeros(264, 136, device=DEV)
    sonicmoe.block128_linear(x, other).backward(dy.T.contiguous().T)          # a gradient of other strides
    assert torch.equal(one.grad, both[0].grad) and other.grad is None
    assert torch.equal(other.main_grad.to(torch.bfloat16), both[1].grad)
    other.main_grad = torch.zeros(264, 137, device=DEV)
    with pytest.raises(ValueError):
        sonicmoe.block128_linear(x, other).backward(dy)
    y = sonicmoe.block128_linear(*both)
    g, = torch.autograd.grad(y.sum(), both[0], create_graph=True)
    with pytest.raises(RuntimeError):                          # no second derivative, and it says so
        torch.autograd.grad(g.sum(), both[1])


def test_segments_without_counts_and_tables_without_rows(sonicmoe):
    efo, _, rows = table([128, 256, 0, 128])
    x, w = randn(rows, 136, seed=1), randn(4, 128, 136, seed=2)
    y = sonicmoe.block128_linear(x.to(DEV), w.to(DEV), efo.to(DEV))
    ref = O.rows_product(O.deq_rows(*O.quant_rows(x)), O.deq_weight(*O.quant_weight(w)), efo, None)
    near(y, ref, 136)
    # nothing is routed here: zeros, and gradients of zeros
    none = torch.zeros(4, dtype=torch.int32, device=DEV)
    xd, wd = x.to(DEV).requires_grad_(True), w.to(DEV).requires_grad_(True)
    for e, n in ((efo.to(DEV), none), (torch.zeros(5, dtype=torch.int32, device=DEV), none)):
        y = sonicmoe.block128_linear(xd, wd, e, n)
        gx, gw = torch.autograd.grad(y, (xd, wd), torch.ones_like(y))
        assert (y == 0).all() and (gx == 0).all() and (gw == 0).all()
    pairs = [sonicmoe.quantize_weight_block128(randn(*s, seed=4).to(DEV)) for s in ((4, 256, 136), (4, 136, 128))]
    idx, sc = torch.full((9, 2), -1, dtype=torch.int32, device=DEV), torch.ones(9, 2, device=DEV)
    out = sonicmoe.block128_experts(x[:9].to(DEV), idx, sc, *pairs)
    assert out.shape == (9, 136) and (out == 0).all()
    assert sonicmoe.block128_experts(x[:0].to(DEV), idx[:0], sc[:0], *pairs).shape == (0, 136)


def test_offsets_beyond_32_bits(sonicmoe):
    """Rows x columns, and experts x rows x columns, above 2^31: what lies at the end is what a small call gives."""
    ops = sonicmoe.ops
    rows, N, K = 300032, 8192, 128
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(rows, K, generator=g, device=DEV).to(torch.bfloat16)
    w = torch.randn(1, N, K, generator=g, device=DEV).to(torch.bfloat16)
    W = ops.quant128_weight(w)
    y = ops.gemm128_rows(*ops.quant128_rows(x), *W)
    end = slice(rows - 200, rows)
    assert torch.equal(y[end], ops.gemm128_rows(*ops.quant128_rows(x[end].contiguous()), *W))
    # y as the gradient that comes back: both forms, and a weight gradient over the last block alone
    q, s, qt, st = ops.quant128_dual(y)
    small = ops.quant128_dual(y[rows - 128:].contiguous())
    assert torch.equal(q[rows - 128:], small[0]) and torch.equal(s[rows - 128:], small[1])
    assert torch.equal(qt[:, rows - 128:], small[2]) and torch.equal(st[-1:], small[3])
    xt = ops.quant128_dual(x, with_rows=False)[2:]
    efo = torch.tensor([0, rows - 128, rows], dtype=torch.int32, device=DEV)
    counts = torch.tensor([0, 128], dtype=torch.int32, device=DEV)
    dw = ops.gemm128_wgrad(qt, st, *xt, efo, counts)
    assert (dw[0] == 0).all()
    assert torch.equal(dw[1:], ops.gemm128_wgrad(small[2], small[3], *ops.quant128_dual(x[rows - 128:].contiguous())[2:]))
    dx = ops.gemm128_rows(q, s, *W, b_mn=True)
    assert torch.equal(dx[rows - 128:], ops.gemm128_rows(small[0], small[1], *W, b_mn=True))
    z = ops.quant128_rows(y, True)
    assert torch.equal(z[0][rows - 128:], ops.quant128_rows(y[rows - 128:].contiguous(), True)[0])
    del x, y, q, s, qt, st, xt, dx, z
    E, N, K = 200, 4096, 2816
    w = torch.empty(E, N, K, dtype=torch.bfloat16, device=DEV).normal_(generator=g)
    W = ops.quant128_weight(w)
    x = torch.randn(3, K, generator=g, device=DEV).to(torch.bfloat16)
    X = ops.quant128_rows(x)
    last = ops.gemm128_few(*X, *(t[E - 1:] for t in W))
    assert torch.equal(W[0][E - 1:], ops.quant128_weight(w[E - 1:].contiguous())[0])
    efo = torch.tensor([0] * E + [3], dtype=torch.int32, device=DEV)
    counts = torch.tensor([0] * (E - 1) + [3], dtype=torch.int32, device=DEV)
    far = ops.gemm128_few(*X, *W, efo, counts)                 # (the reduction may be divided otherwise: other roundings in f32)
    ref, mag = O.rows_product(O.deq_rows(*(t.cpu().view(torch.float8_e4m3fn) if t.dtype == torch.uint8 else t.cpu() for t in X)),
                              O.deq_weight(W[0][E - 1:].cpu().view(torch.float8_e4m3fn), W[1][E - 1:].cpu()), None, None)
    tol = BF16 * ref.abs() + f32_tol(K, 22) * mag * (1 + BF16)
    for got in (last, far, ops.gemm128_rows(*X, *W, efo, counts)):
        assert ((got.cpu().double() - ref).abs() <= tol).all()


def test_repeated_calls_give_the_same_bits(sonicmoe):
    """No sum here depends on which block of threads came first."""
    efo, cnt, rows = table([300, 0, 5, 700])
    e, c = efo.to(DEV), cnt.to(DEV)
    x, w, dy = randn(rows, 264, seed=1).to(DEV), randn(4, 520, 264, seed=2).to(DEV), randn(rows, 520, seed=3).to(DEV)
    runs = []
    for _ in range(3):
        a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        y = sonicmoe.block128_linear(a, b, e, c)
        y.backward(dy)
        one = sonicmoe.block128_linear(x[:3], w[0])
        runs.append((y.detach(), a.grad, b.grad, one))
    for run in runs[1:]:
        assert all(torch.equal(p, q) for p, q in zip(run, runs[0]))


def test_views_that_begin_off_a_boundary(sonicmoe):
    """Tensors inside a larger buffer, gradients too, give what copies of them give."""
    def off(t):
        buf = torch.zeros(t.numel() + 3, dtype=t.dtype, device=DEV)
        v = buf[3:].view(t.shape)
        v.copy_(t)
        assert v.data_ptr() % 16
        return v

    x, w, dy = randn(70, 264).to(DEV), randn(1, 136, 264, seed=1).to(DEV), randn(70, 136, seed=2).to(DEV)
    got = []
    for f in (lambda t: t, off):
        a, b = f(x).requires_grad_(True), f(w).requires_grad_(True)
        y = sonicmoe.block128_linear(a, b)
        got.append([y.detach(), *torch.autograd.grad(y, (a, b), f(dy)), *sonicmoe.quantize_rows_block128(a.detach()),
                    *sonicmoe.quantize_weight_block128(b)])
    for u, v in zip(*got):
        assert torch.equal(u.float(), v.float())
    w1, w2 = (sonicmoe.quantize_weight_block128(randn(4, *s, seed=3).to(DEV)) for s in ((256, 264), (264, 128)))
    scores, idx = torch.rand(70, 4, device=DEV).topk(2)
    a, b = (sonicmoe.block128_experts(f(x), idx.int(), scores, w1, w2) for f in (lambda t: t, off))
    assert torch.equal(a, b)


@pytest.mark.parametrize("accumulate", [False, True])
def test_a_captured_training_step(sonicmoe, accumulate):
    """Router, projection and all gradients from one graph, replayed on new values, one replay after another."""
    efo, counts, rows = table([300, 0, 129, 70])
    e, n = efo.to(DEV), counts.to(DEV)
    make = lambda seed: (randn(rows, 264, seed=seed), randn(4, 136, 264, seed=seed + 1), randn(rows, 136, seed=seed + 2),
                         torch.randn(65, 16, generator=torch.Generator().manual_seed(seed + 3)))

    def step(x, w, dy, logits):
        y = sonicmoe.block128_linear(x, w, e, n)
        scores, idx = sonicmoe.group_limited_routing(logits, 3, groups=4, top_groups=2)
        # (with a main_grad w's gradient goes there on the way, and None comes back)
        grads = torch.autograd.grad((y, scores), (x, logits, w), (dy, scores.detach() * 2 + 1), allow_unused=True)
        return [y.detach(), scores.detach(), idx, *(g for g in grads if g is not None)]

    def leaves(seed):
        x, w, dy, logits = (t.to(DEV) for t in make(seed))
        x, w, logits = (t.requires_grad_(True) for t in (x, w, logits))
        if accumulate:
            w.main_grad = torch.zeros(4, 136, 264, device=DEV)
        return x, w, dy, logits

    wants = []
    for seed in (10, 20):
        t = leaves(seed)
        wants.append([v.clone() for v in step(*t)] + ([t[1].main_grad.clone()] if accumulate else []))
    static = leaves(30)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(*static)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(*static)
    for seed, want in zip((10, 20), wants):
        with torch.no_grad():
            for a, b in zip(static, make(seed)):
                a.copy_(b)
            if accumulate:
                static[1].main_grad.zero_()
        graph.replay()
        graph.replay()
        got = list(outs) + ([static[1].main_grad / 2] if accumulate else [])      # added twice: x + x is exact
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    sonicmoe.ops.check_status(DEV)
