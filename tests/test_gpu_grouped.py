"""Products of bf16 rows grouped by expert against 64 bits: segments of any lengths and places, both gradients."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32
NAN = float("nan")


@pytest.fixture(scope="module")
def sonicmoe():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import sonicmoe as m
    yield m
    torch.cuda.synchronize()
    m.ops.check_status(DEV)


def randn(*shape, seed=0, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV) * scale).to(BF)


def within(got, want, terms, n, half):
    """A sum of n products of bf16 (exact in f32) in f32, whatever their order, each addition off by up to 2^-23 of the sum of the
    terms' magnitudes (an adder that cuts instead of rounding), and half a step of the result's type."""
    err = n * 2.0 ** -23 * terms
    bound = err + half * (want.abs() + err) + 1e-38
    bad = ~((got.double() - want).abs() <= bound)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), got.double()[bad][:4].tolist(), want[bad][:4].tolist())


def segments(counts, gaps=None, first=0, padded=False, tail=0):
    """-> (efo, counts or None, first rows, rows): gaps[e] dead rows behind segment e."""
    starts, at = [], first
    for i, c in enumerate(counts):
        starts.append(at)
        at += -(-c // 128) * 128 if padded else c + (gaps[i] if gaps else 0)
    efo = torch.tensor(starts + [at], dtype=torch.int32, device=DEV)
    n = torch.tensor(counts, dtype=torch.int32, device=DEV) if gaps or padded else None
    return efo, n, starts, at + tail


def reference(x, w, dy, counts, starts):
    """-> y, dx, dw in f64 with the sums of magnitudes of each, by experts."""
    E, N, K = w.shape
    D = torch.float64
    y, ya = (torch.zeros(x.shape[0], N, dtype=D, device=DEV) for _ in range(2))
    dx, dxa = (torch.zeros(x.shape[0], K, dtype=D, device=DEV) for _ in range(2))
    dw, dwa = (torch.zeros(E, N, K, dtype=D, device=DEV) for _ in range(2))
    for e, c in enumerate(counts):
        r = slice(starts[e], starts[e] + c)
        a, b, d = x[r].double(), w[e].double(), dy[r].double()
        y[r], ya[r] = a @ b.T, a.abs() @ b.abs().T
        dx[r], dxa[r] = d @ b, d.abs() @ b.abs()
        dw[e], dwa[e] = d.T @ a, d.abs().T @ a.abs()
    return (y, ya), (dx, dxa), (dw, dwa)


def check(sonicmoe, counts, N, K, seed=0, main_grad=False, **kw):
    efo, n, starts, rows = segments(counts, **kw)
    E = len(counts)
    x, dy, w = randn(rows, K, seed=seed), randn(rows, N, seed=seed + 1), randn(E, N, K, seed=seed + 2, scale=K ** -0.5)
    live = torch.zeros(rows, dtype=torch.bool, device=DEV)
    for s, c in zip(starts, counts):
        live[s:s + c] = True
    x[~live], dy[~live] = NAN, float("inf")                  # nobody's rows
    refs = reference(x, w, dy, counts, starts)
    with torch.no_grad():
        y0 = sonicmoe.grouped_linear(x, w, efo, n)
    within(y0, *refs[0], K, 2.0 ** -8)
    assert not y0[~live].any()
    xg = x.requires_grad_(True)
    wg = torch.nn.Parameter(w) if main_grad else w.requires_grad_(True)
    if main_grad:
        wg.main_grad = torch.full((E, N, K), 3.0, device=DEV)
    y = sonicmoe.grouped_linear(xg, wg, efo, n)
    assert torch.equal(y, y0)
    y.backward(dy)
    within(xg.grad, *refs[1], N, 2.0 ** -8)
    assert not xg.grad[~live].any()
    longest = max(counts, default=0)
    if main_grad:
        assert wg.grad is None
        want = refs[2][0] + 3
        within(wg.main_grad, want, refs[2][1] + 3, longest + 1, 2.0 ** -24)
        for e, c in enumerate(counts):
            if c == 0:
                assert (wg.main_grad[e] == 3).all()
    else:
        within(wg.grad, *refs[2], longest, 2.0 ** -8)
        for e, c in enumerate(counts):
            if c == 0:
                assert not wg.grad[e].any()


@pytest.mark.parametrize("rows,N,K", [(1, 8, 8), (16, 128, 64), (17, 136, 72), (64, 256, 128), (65, 256, 256), (128, 256, 64), (300, 520, 200), (700, 1000, 720),
                                      (256, 8, 4096), (1000, 4096, 8)])
def test_one_weight(sonicmoe, rows, N, K):
    check(sonicmoe, [rows], N, K)


@pytest.mark.parametrize("counts", [
    [0], [0, 0, 5], [1, 1, 1], [64, 128, 256], [63, 65, 1, 0, 127], [257, 3, 511, 0, 0, 40], [300, 0, 299, 301], [1000, 7, 600],
    [i % 5 for i in range(128)], [(i * 7) % 41 for i in range(256)], [2000] + [0] * 30 + [1]])
@pytest.mark.parametrize("kw", [dict(), dict(padded=True, tail=200), dict(first=3, tail=5), "gaps"], ids=["packed", "padded", "offset", "gaps"])
def test_segments(sonicmoe, counts, kw):
    if kw == "gaps":
        kw = dict(gaps=[(3 * i + 1) % 70 for i in range(len(counts))], first=11, tail=33)
    check(sonicmoe, counts, 264, 136, **kw)


@pytest.mark.parametrize("N,K", [(8, 8), (64, 1000), (1000, 64), (128, 2056), (512, 1536)])
@pytest.mark.parametrize("counts", [[70, 0, 3, 400], [5, 20, 0, 9]])
def test_sizes_and_main_grad(sonicmoe, N, K, counts):
    check(sonicmoe, counts, N, K, main_grad=True)
    check(sonicmoe, counts, N, K, seed=5, padded=True)


@pytest.mark.parametrize("N,K", [(136, 72), (264, 520)])
@pytest.mark.parametrize("gaps", [False, True])
def test_every_length_of_a_segment(sonicmoe, gaps, N, K):
    """A block of the reduction ends anywhere; what lies behind it belongs to the next expert, or to nobody."""
    counts = list(range(131))
    check(sonicmoe, counts, N, K, **(dict(gaps=[(5 * i) % 37 for i in counts]) if gaps else {}))
    check(sonicmoe, counts[::-1], N, K, seed=5, main_grad=True, **(dict(gaps=[300] + [0] * 128 + [700, 1], first=40) if gaps else {}))


def test_large(sonicmoe):
    check(sonicmoe, [3000, 0, 1, 5011, 777, 64, 2500, 129], 4096, 2048)
    check(sonicmoe, [3000, 0, 1, 5011, 777, 64, 2500, 129], 2048, 1536, main_grad=True)


@pytest.mark.parametrize("counts,N,K", [([5000], 136, 72), ([5000], 64, 512), ([13001, 0, 4999], 264, 136), ([19000, 1, 700], 128, 256),
                                        ([20000], 1000, 520), ([40000], 8, 8)])
def test_weight_gradients_of_few_tiles_are_summed_in_stretches(sonicmoe, counts, N, K):
    from sonicmoe._lib import lib
    for kw in (dict(), dict(padded=True, tail=100)):
        rows = segments(counts, **kw)[3]
        assert lib.smoe_grouped_wgrad_workspace(N, K, rows, len(counts)) > 0
        check(sonicmoe, counts, N, K, **kw)
        check(sonicmoe, counts, N, K, main_grad=True, **kw)


@pytest.mark.parametrize("rows,N,K", [(600, 1024, 200), (3000, 512, 136), (5000, 128, 64), (5000, 72, 264), (300, 4096, 520)])
def test_narrow_tiles(sonicmoe, rows, N, K):
    check(sonicmoe, [rows], N, K)
    check(sonicmoe, [rows // 2, 3, 0, rows - rows // 2 - 3], N, K, main_grad=True)


@pytest.mark.parametrize("counts", [[1], [7], [16], [0, 0, 1, 0], [1] * 16, [2, 0, 5, 0, 9], [0] * 200 + [8] + [0] * 55, [0] * 100 + [3, 0, 1] + [0] * 100 + [4]])
@pytest.mark.parametrize("N,K", [(8, 8), (136, 72), (264, 1032), (1000, 720)])
def test_a_handful_of_rows(sonicmoe, counts, N, K):
    check(sonicmoe, counts, N, K)
    if sum(counts) < 12:
        check(sonicmoe, counts, N, K, first=1, tail=2)
        gaps = [0] * len(counts)
        gaps[0], gaps[-1] = 1, 1
        check(sonicmoe, counts, N, K, gaps=gaps)


def test_few_rows_of_a_wide_weight_are_shared_by_clusters(sonicmoe):
    for rows in (1, 15, 16, 17, 33, 64):
        for N, K in ((4096, 4096), (1024, 2048), (136, 8192), (4096, 760)):
            x, w = randn(rows, K, seed=rows), randn(N, K, seed=K, scale=K ** -0.5)
            y = sonicmoe.grouped_linear(x, w)
            a, b = x.double(), w.double()
            within(y, a @ b.T, a.abs() @ b.abs().T, K, 2.0 ** -8)
            dy = randn(rows, N, seed=1)
            dx, = torch.autograd.grad(sonicmoe.grouped_linear(x.requires_grad_(True), w), x, dy)
            d = dy.double()
            within(dx, d @ b, d.abs() @ b.abs(), N, 2.0 ** -8)


def test_rows_and_runs_do_not_depend_on_one_another(sonicmoe):
    """A row's result is the same whatever else is in the batch, and the same again."""
    counts = [500, 30, 700]
    efo, _, starts, rows = segments(counts)
    x, w = randn(rows, 520), randn(3, 392, 520, seed=1)
    y = sonicmoe.grouped_linear(x, w, efo)
    assert torch.equal(y, sonicmoe.grouped_linear(x, w, efo))
    x2 = x.clone()
    x2[starts[1]:starts[2]] = NAN
    y2 = sonicmoe.grouped_linear(x2, w, efo)
    assert torch.equal(y2[:starts[1]], y[:starts[1]]) and torch.equal(y2[starts[2]:], y[starts[2]:]) and y2[starts[1]:starts[2]].isnan().all()


def test_infinities_and_nan_are_carried(sonicmoe):
    efo, _, starts, rows = segments([100, 100])
    x, w, dy = randn(rows, 72), randn(2, 80, 72, seed=1), randn(rows, 80, seed=2)
    x[99, 3], x[100, 5], dy[150, 7] = float("inf"), NAN, NAN
    xg, wg = x.requires_grad_(True), w.requires_grad_(True)
    y = sonicmoe.grouped_linear(xg, wg, efo)
    dx, dw = torch.autograd.grad(y, (xg, wg), dy)
    assert torch.isinf(y[99]).all() and y[100].isnan().all() and torch.isfinite(y[:99]).all() and torch.isfinite(y[101:]).all()
    assert dx[150].isnan().all() and torch.isfinite(dx[:150]).all() and torch.isfinite(dx[151:]).all()
    assert torch.isinf(dw[0, :, 3]).all() and torch.isfinite(dw[0, :, :3]).all() and torch.isfinite(dw[0, :, 4:]).all()
    assert dw[1, :, 5].isnan().all() and dw[1, 7].isnan().all() and torch.isfinite(dw[1, :7, :5]).all()


def test_one_gradient_at_a_time_and_leading_dimensions(sonicmoe):
    x, w, dy = randn(6, 50, 72), randn(1, 136, 72, seed=1), randn(6, 50, 136, seed=2)
    for weight in (w, w[0]):
        y = sonicmoe.grouped_linear(x, weight)
        assert y.shape == (6, 50, 136)
        assert torch.equal(y.view(300, 136), sonicmoe.grouped_linear(x.view(300, 72), weight))
        xg, wg = x.clone().requires_grad_(True), weight.clone().requires_grad_(True)
        both = torch.autograd.grad(sonicmoe.grouped_linear(xg, wg), (xg, wg), dy)
        assert torch.equal(torch.autograd.grad(sonicmoe.grouped_linear(xg, weight), xg, dy)[0], both[0])
        assert torch.equal(torch.autograd.grad(sonicmoe.grouped_linear(x, wg), wg, dy)[0], both[1])
        assert both[0].shape == x.shape and both[1].shape == weight.shape
    assert sonicmoe.grouped_linear(x[0, 0], w).shape == (136,)
    empty = x[:0].clone().requires_grad_(True)
    wg = w.clone().requires_grad_(True)
    y = sonicmoe.grouped_linear(empty, wg)
    dx, dw = torch.autograd.grad(y, (empty, wg), dy[:0])
    assert y.shape == (0, 50, 136) and dx.shape == empty.shape and not dw.any()


def test_views(sonicmoe):
    """Rows apart, off a boundary, columns of a larger table; gradients and weights that are views; an accumulator off a boundary."""
    wide, w = randn(90, 800), randn(3, 72, 264, seed=3)
    efo, _, _, _ = segments([40, 7, 43])
    for view in (wide[:, :264], wide[:, 8:272], wide[:, 3:267], randn(90, 264, seed=4).repeat_interleave(2, 0)[::2], randn(264, 90).T,
                 wide[:1, :264].expand(90, 264)):
        dy = randn(90, 100, seed=5)[:, 16:88]
        grads = []
        for x in (view.detach(), view.contiguous()):
            xg = x.requires_grad_(True)
            wg = w.clone().requires_grad_(True)
            y = sonicmoe.grouped_linear(xg, wg, efo)
            grads.append((y, *torch.autograd.grad(y, (xg, wg), dy)))
        assert all(torch.equal(a, b) for a, b in zip(*grads))
    flat = torch.zeros(3 * 72 * 264 + 1, dtype=BF, device=DEV)
    flat[1:] = w.flatten()
    x = wide[:, :264]
    assert torch.equal(sonicmoe.grouped_linear(x, flat[1:].view(3, 72, 264), efo), sonicmoe.grouped_linear(x, w, efo))
    assert torch.equal(sonicmoe.grouped_linear(x, w.transpose(1, 2).contiguous().transpose(1, 2), efo), sonicmoe.grouped_linear(x, w, efo))
    p = torch.nn.Parameter(w.clone())
    p.main_grad = torch.zeros(3 * 72 * 264 + 1, device=DEV)[1:].view(3, 72, 264)
    dy = randn(90, 72, seed=6)
    sonicmoe.grouped_linear(x, p, efo).backward(dy)
    p2 = torch.nn.Parameter(w.clone())
    p2.main_grad = torch.zeros(3, 72, 264, device=DEV)
    sonicmoe.grouped_linear(x, p2, efo).backward(dy)
    assert torch.equal(p.main_grad, p2.main_grad)


def test_a_weight_changed_between_the_passes_is_noticed(sonicmoe):
    x, w = randn(40, 72).requires_grad_(True), randn(2, 80, 72).requires_grad_(True)
    y = sonicmoe.grouped_linear(x, w, segments([20, 20])[0])
    with torch.no_grad():
        w.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(torch.ones_like(y))


def test_gradients_are_not_differentiated_again(sonicmoe):
    for main_grad in (False, True):
        x, w, dy = (t.requires_grad_(True) for t in (randn(40, 72), randn(80, 72), randn(40, 80)))
        if main_grad:
            w.main_grad = torch.zeros(80, 72, device=DEV)
        dx, = torch.autograd.grad(sonicmoe.grouped_linear(x, w), x, dy, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiate"):
            dx.sum().backward()


def test_the_hook_of_a_parameter_with_main_grad(sonicmoe):
    p = torch.nn.Parameter(randn(2, 72, 136))
    p.main_grad = torch.zeros(2, 72, 136, device=DEV)
    calls = []
    p._apply_backward_hook = lambda: calls.append(1)
    sonicmoe.grouped_linear(randn(30, 136), p, segments([10, 20])[0]).sum().backward()
    assert calls == [1] and p.main_grad.any()
    p.main_grad = torch.zeros(2, 72, 135, device=DEV)
    with pytest.raises(ValueError, match="main_grad"):
        sonicmoe.grouped_linear(randn(30, 136), p, segments([10, 20])[0]).sum().backward()


@pytest.mark.parametrize("main_grad", [False, True])
@pytest.mark.parametrize("rows", [40, 900])
def test_in_a_graph_and_on_another_stream(sonicmoe, rows, main_grad):
    counts = ([rows // 2, 0, rows - rows // 2], [3, rows - 4, 1])

    def make(i):
        return randn(rows, 136, seed=i), randn(3, 264, 136, seed=i + 1), randn(rows, 264, seed=i + 2), segments(counts[i % 2])[0]

    def leaves(i):
        x, w, dy, efo = make(i)
        x, w = x.requires_grad_(True), w.requires_grad_(True)
        if main_grad:
            w.main_grad = torch.zeros(3, 264, 136, device=DEV)
        return x, w, dy, efo

    def step(x, w, dy, efo):
        y = sonicmoe.grouped_linear(x, w, efo)
        return [y.detach(), *(g for g in torch.autograd.grad(y, (x, w), dy, allow_unused=True) if g is not None)]

    wants = []
    for i in (10, 11):
        t = leaves(i)
        wants.append([v.clone() for v in step(*t)] + ([t[1].main_grad.clone()] if main_grad else []))
    static = leaves(12)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        t = leaves(10)
        got = step(*t) + ([t[1].main_grad] if main_grad else [])
        assert all(torch.equal(a, b) for a, b in zip(got, wants[0]))
        step(*static)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(*static)
    for i, want in zip((10, 11), wants):
        with torch.no_grad():
            for a, b in zip(static, make(i)):
                a.copy_(b)
            if main_grad:
                static[1].main_grad.zero_()
        graph.replay()
        graph.replay()
        got = list(outs) + ([static[1].main_grad / 2] if main_grad else [])      # added twice: x + x is exact
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_gradients_against_differences(sonicmoe):
    """The product is linear in either operand: a difference of two products is the product of the difference, up to their roundings."""
    counts = [30, 0, 41]
    efo, _, starts, rows = segments(counts)
    x, w, dy = randn(rows, 72), randn(3, 80, 72, seed=1), randn(rows, 80, seed=2)
    vx, vw = randn(rows, 72, seed=3), randn(3, 80, 72, seed=4)
    xg, wg = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    dx, dw = torch.autograd.grad(sonicmoe.grouped_linear(xg, wg, efo), (xg, wg), dy)
    total = lambda a, b: (sonicmoe.grouped_linear(a, b, efo).double() * dy.double()).sum()
    for lo, hi, g, v in (((x, w), ((x + vx), w), dx, x), ((x, w), (x, (w + vw)), dw, w)):
        moved = (hi[0].double() - x.double()) if g is dx else (hi[1].double() - w.double())
        want = (g.double() * moved).sum()
        ys = [sonicmoe.grouped_linear(*p, efo).double().abs() for p in (lo, hi)]
        bound = 2.0 ** -8 * (((ys[0] + ys[1]) * dy.double().abs()).sum() + (g.double() * moved).abs().sum()) * 1.01
        assert abs(total(*hi) - total(*lo) - want) <= bound


def test_offsets_beyond_32_bits(sonicmoe):
    """Rows and columns whose product passes 2^31, and an expert whose weights lie beyond."""
    rows, K, N = 600_000, 4096, 16
    x = torch.zeros(rows, K, dtype=BF, device=DEV)
    at = [0, 524_287, 524_288, rows - 1]
    x[at] = randn(4, K, seed=1)
    w = randn(2, N, K, seed=2, scale=1 / 64)
    efo = torch.tensor([0, 524_288, rows], dtype=torch.int32, device=DEV)
    y = sonicmoe.grouped_linear(x, w, efo)
    for i, r in enumerate(at):
        a, b = x[r].double(), w[int(r >= 524_288)].double()
        within(y[r], b @ a, b.abs() @ a.abs(), K, 2.0 ** -8)
    del x, y
    E = 130
    w = torch.zeros(E, 4096, 4096, dtype=BF, device=DEV)
    w[129] = randn(4096, 4096, seed=3, scale=1 / 64)
    counts = [0] * 129 + [5]
    efo = segments(counts)[0]
    x = randn(5, 4096, seed=4).requires_grad_(True)
    y = sonicmoe.grouped_linear(x, w, efo)
    b = w[129].double()
    within(y, x.double() @ b.T, x.double().abs() @ b.abs().T, 4096, 2.0 ** -8)
    dy = randn(5, 4096, seed=5)
    dx, = torch.autograd.grad(y, x, dy)
    within(dx, dy.double() @ b, dy.double().abs() @ b.abs(), 4096, 2.0 ** -8)
    dw = sonicmoe.ops.grouped_wgrad(dy, x.detach(), efo, None, E)
    within(dw[129], dy.double().T @ x.double(), dy.double().abs().T @ x.double().abs(), 5, 2.0 ** -8)
    assert not dw[128].any()
