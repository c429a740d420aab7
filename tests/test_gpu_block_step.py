"""The norm, the router, the experts, their gradients and clipping as one pre-norm block uses them: FP8 experts on the norm's payload,
bf16 experts by ragged segments, one token and a captured step."""
import pytest
import torch

from oracle import norm as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16
T, H, I, E, K = 320, 256, 128, 8, 2


@pytest.fixture(scope="module")
def sonicmoe():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import sonicmoe as m
    yield m
    torch.cuda.synchronize()
    m.ops.check_status(DEV)


def randn(*shape, seed=0, scale=1.0, dtype=BF):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).to(DEV)


def params():
    return dict(g=torch.nn.Parameter(1 + randn(H, seed=1, scale=0.2, dtype=torch.float32)),
                router=torch.nn.Parameter(randn(H, E, seed=2, scale=H ** -0.5)),
                w1=torch.nn.Parameter(randn(E, 2 * I, H, seed=3, scale=H ** -0.5)),
                w2=torch.nn.Parameter(randn(E, H, I, seed=4, scale=I ** -0.5)))


def relative(got, want):
    got, want = got.detach().double(), want.detach().double()
    return float((got - want).norm() / want.norm())


# Each bf16 tensor of a chain is off by some 0.0017 of its norm (a rounding of up to 2^-8 of each value), and products pass a relative
# error on: six of them in a row, as independent errors add up, stay below 2^-7
CHAIN = 2.0 ** -7


def fp8_block(m, p, x, res):
    """-> (out, residual stream)"""
    n = m.rms_norm_quantized(x, p["g"], res, with_output=True)
    logits = n.y @ p["router"]
    scores, idx = m.group_limited_routing(logits.float(), K, score="softmax", groups=4, top_groups=2)
    return m.run_sonic_moe(n.payload, idx, scores, K, E, p["w1"], p["w2"], fp8=True, fp8_scale=n.scales, grad_holder=n.y), n, idx, scores


def accumulators(p):
    """As the FP8 layer has them: that of W2 lies the other way round."""
    p["w1"].main_grad = torch.zeros(E, 2 * I, H, device=DEV)
    p["w2"].main_grad = torch.zeros(E, I, H, device=DEV)


def test_fp8_experts_on_the_payload_of_the_norm(sonicmoe):
    m, p = sonicmoe, params()
    accumulators(p)
    x, res, dout, dh = randn(T, H, seed=5), randn(T, H, seed=6, scale=2), randn(T, H, seed=7), randn(T, H, seed=8)
    gx, gres = x.clone().requires_grad_(True), res.clone().requires_grad_(True)
    out, n, idx, scores = fp8_block(m, p, gx, gres)
    torch.autograd.backward((out, n.h), (dout, dh))
    # the same step by step, the norm in 64 bits
    h = O.total(x.cpu(), res.cpu()).to(DEV)
    y = O.bf16(O.rms_norm(h.cpu(), p["g"].detach().cpu(), 1e-6)[0]).to(DEV).requires_grad_(True)
    assert torch.equal(n.h, h) and torch.equal(n.y, y)
    q = params()
    accumulators(q)
    payload, raw, _ = m.ops.quant_rows(y.detach())
    logits = y @ q["router"]
    scores2, idx2 = m.group_limited_routing(logits.float(), K, score="softmax", groups=4, top_groups=2)
    out2 = m.run_sonic_moe(payload.view(torch.float8_e4m3fn), idx2, scores2, K, E, q["w1"], q["w2"], fp8=True, fp8_scale=raw, grad_holder=y)
    out2.backward(dout)
    assert torch.equal(out, out2) and torch.equal(idx, idx2)
    assert torch.equal(p["w1"].main_grad, q["w1"].main_grad) and torch.equal(p["w2"].main_grad, q["w2"].main_grad)
    want, want_g = O.rms_norm_backward(h.cpu(), q["g"].detach().cpu(), 1e-6, y.grad.cpu(), dh.cpu())
    assert relative(gx.grad.cpu(), want) < 2.0 ** -8 and torch.equal(gx.grad, gres.grad)
    assert relative(p["g"].grad.cpu(), want_g) < 512 * 2.0 ** -24
    assert torch.equal(p["router"].grad, q["router"].grad)
    # gradients of all kinds, clipped together
    grads = [v.main_grad if hasattr(v, "main_grad") else v.grad for v in p.values()]
    before = [g.cpu().clone() for g in grads]
    norm = m.clip_gradients(p.values(), 0.5)
    assert abs(float(norm) / float(O.gradient_norm(before)) - 1) < 6 * 2.0 ** -24 and float(norm) > 0.5
    for g, r in zip(grads, O.clipped(before, 0.5)):
        assert ((g.cpu().double() - r).abs() <= r.abs() * (12 * 2.0 ** -24 + torch.finfo(g.dtype).eps / 2 * 1.01) + 1e-45).all()


def bf16_block(m, p, x, res):
    """Experts in bf16 over segments that follow one another: token rows sorted by expert, two products, a weighted sum."""
    y, h = m.rms_norm(x, p["g"], res)
    scores, idx = m.group_limited_routing((y @ p["router"]).float(), K, score="softmax", groups=4, top_groups=2)
    flat = idx.flatten()
    order = flat.argsort(stable=True)
    _, ends = m.count_cumsum(flat.contiguous(), E)
    efo = torch.cat([ends.new_zeros(1), ends])
    rows = y[order // K]
    z = m.grouped_linear(rows, p["w1"], efo)
    a = (torch.nn.functional.silu(z[:, 0::2].float()) * z[:, 1::2].float()).to(BF)
    o = m.grouped_linear(a, p["w2"], efo)
    weighted = o.float() * scores.flatten()[order][:, None]
    return torch.zeros(x.shape, device=x.device).index_add(0, order // K, weighted).to(BF), h, idx


def exact_block(p, x, res, idx):
    """The same in 64 bits, for the same choice of experts."""
    g, router, w1, w2 = (p[k].double() for k in ("g", "router", "w1", "w2"))
    h = x + res
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-6) * g
    s = torch.softmax(y @ router, -1).gather(1, idx.long())
    s = s / s.sum(-1, keepdim=True)
    out = torch.zeros_like(x)
    for e in range(E):
        t, k = (idx == e).nonzero(as_tuple=True)
        z = y[t] @ w1[e].T
        out = out.index_add(0, t, ((torch.nn.functional.silu(z[:, 0::2]) * z[:, 1::2]) @ w2[e].T) * s[t, k][:, None])
    return out, h


@pytest.mark.parametrize("accumulate", [False, True])
def test_bf16_experts_forward_and_backward(sonicmoe, accumulate):
    m, p = sonicmoe, params()
    if accumulate:
        for k in ("g", "w1", "w2"):
            p[k].main_grad = torch.zeros(p[k].shape, device=DEV)
    x, res, dout, dh = randn(T, H, seed=5), randn(T, H, seed=6, scale=2), randn(T, H, seed=7), randn(T, H, seed=8)
    gx, gres = x.clone().requires_grad_(True), res.clone().requires_grad_(True)
    out, h, idx = bf16_block(m, p, gx, gres)
    torch.autograd.backward((out, h), (dout, dh))
    q = {k: v.detach().double().requires_grad_(True) for k, v in p.items()}
    ex, er = x.double().requires_grad_(True), res.double().requires_grad_(True)
    want, want_h = exact_block(q, ex, er, idx)
    torch.autograd.backward((want, want_h), (dout.double(), dh.double()))
    assert relative(out, want) < CHAIN
    assert relative(gx.grad, ex.grad) < CHAIN and relative(gres.grad, er.grad) < CHAIN
    for k, v in p.items():
        got = v.main_grad if hasattr(v, "main_grad") else v.grad
        assert relative(got, q[k].grad) < CHAIN, k
    norm = m.gradient_norm(p.values())
    whole = torch.cat([(v.main_grad if hasattr(v, "main_grad") else v.grad).double().flatten() for v in p.values()]).norm()
    assert abs(float(norm) / float(whole) - 1) < 6 * 2.0 ** -24


def test_one_token(sonicmoe):
    """Decoding: the rows of one token are those it has in a batch, through the norm, the payload and the experts of either kind."""
    m, p = sonicmoe, params()
    x, res = randn(T, H, seed=5), randn(T, H, seed=6, scale=2)
    with torch.no_grad():
        out, n, idx, _ = fp8_block(m, p, x, res)
        one, n1, idx1, _ = fp8_block(m, p, x[7:8], res[7:8])
        assert torch.equal(n1.payload.view(torch.uint8), n.payload[7:8].view(torch.uint8)) and torch.equal(n1.scales, n.scales[7:8])
        assert torch.equal(idx1, idx[7:8]) and relative(one, out[7:8]) < CHAIN
        b, _, _ = bf16_block(m, p, x, res)
        b1, h1, _ = bf16_block(m, p, x[7:8], res[7:8])
        assert torch.equal(h1, O.total(x[7:8].cpu(), res[7:8].cpu()).to(DEV)) and relative(b1, b[7:8]) < CHAIN


def test_a_captured_step(sonicmoe):
    """Forward, backward and clipping into other tensors, replayed on new values."""
    m = sonicmoe
    p = params()
    dest = {k: torch.empty(v.shape, dtype=BF, device=DEV) for k, v in p.items()}

    def step(x, res, dout):
        out, h, _ = bf16_block(m, p, x, res)
        grads = torch.autograd.grad((out, h), list(p.values()), (dout, dout))
        return [out.detach(), m.clip_gradients(grads, 1.0, out=list(dest.values()))]

    def batch(i):
        return randn(T, H, seed=20 + i), randn(T, H, seed=30 + i), randn(T, H, seed=40 + i)

    wants = []
    for i in range(2):
        wants.append([v.clone() for v in step(*batch(i))] + [d.clone() for d in dest.values()])
    static = batch(2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*static)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(*static)
    for i, want in enumerate(wants):
        for a, b in zip(static, batch(i)):
            a.copy_(b)
        graph.replay()
        for a, b in zip(outs[1:] + list(dest.values()), want[1:]):
            assert torch.equal(a, b)
        # (the weighted sum is torch's, whose order varies)
        assert relative(outs[0], want[0]) < 2.0 ** -7


def calls(m, rows):
    """The calls whose kernels are made ready while what is ahead of them ends, each as the first of its kind behind it."""
    x, w, dy = randn(rows, 136, seed=1), randn(3, 264, 136, seed=2), randn(rows, 264, seed=3)
    efo = torch.tensor([0, rows // 2, rows // 2, rows], dtype=torch.int32, device=DEV)
    grads, outs, norm = [randn(500, 33, seed=4), randn(7, seed=5)], [torch.empty(500, 33, device=DEV), torch.empty(7, device=DEV)], torch.full(
        (), 40.0, device=DEV)
    return [(x, lambda: [m.grouped_linear(x, w, efo)]), (dy, lambda: [m.ops.grouped_rows(dy, w, efo, None, True)]),
            (dy, lambda: [m.ops.grouped_wgrad(dy, x, efo, None, 3)]),
            (grads[0], lambda: [m.clip_gradients(grads, 10.0, norm=norm, out=outs), *outs]), (grads[0], lambda: [m.gradient_norm(grads)])]


@pytest.mark.parametrize("rows", [3, 60, 3000])
@pytest.mark.parametrize("ahead", ["copy", "join", "copy of another stream", "fill"])
def test_calls_right_behind_what_makes_their_input(sonicmoe, rows, ahead):
    """A copy, a kernel of another stream, a fill: eager and captured, the call sees what they leave."""
    m = sonicmoe
    for value, call in calls(m, rows):
        fresh = [torch.randn(value.shape, generator=torch.Generator(device=DEV).manual_seed(i), device=DEV).to(BF) for i in range(3)]
        source, scratch = fresh[0].clone(), torch.empty(1 << 24, device=DEV)
        other = torch.cuda.Stream()

        def run():
            here = torch.cuda.current_stream()
            if ahead == "copy":
                value.copy_(source)
            elif ahead == "fill":
                value.zero_()
                value.add_(source)
            else:
                other.wait_stream(here)
                with torch.cuda.stream(other):
                    scratch.fill_(1.0)                        # takes a while
                    if ahead == "join":
                        torch.mul(source, 1, out=value)
                    else:
                        value.copy_(source)
                here.wait_stream(other)
            return call()

        wants = []
        for f in fresh[:2]:
            value.copy_(f)
            torch.cuda.synchronize()
            wants.append([v.clone() for v in call()])
        for f, want in zip(fresh[:2], wants):
            source.copy_(f)
            value.fill_(float("nan"))
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(run(), want))
        value.copy_(fresh[2])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = run()
        for f, want in zip(fresh[:2], wants):
            source.copy_(f)
            value.fill_(float("nan"))
            torch.cuda.synchronize()
            graph.replay()
            assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_two_streams_at_once(sonicmoe):
    """Calls of two streams overlap: each has outputs and workspaces of its own."""
    m = sonicmoe
    sets = [calls(m, rows) for rows in (2500, 40)]
    wants = [[[v.clone() for v in call()] for _, call in s] for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[] for _ in sets]
    for turn in range(20):
        for i, (stream, s) in enumerate(zip(streams, sets)):
            with torch.cuda.stream(stream):
                got[i].append([[v.clone() for v in call()] for _, call in s])
    torch.cuda.synchronize()
    for want, runs in zip(wants, got):
        for run in runs:
            assert all(torch.equal(a, b) for x, y in zip(run, want) for a, b in zip(x, y))


def test_the_graph_kept_for_a_second_backward_pass(sonicmoe):
    m = sonicmoe
    x, w, g = (t.requires_grad_(True) for t in (randn(50, 136, seed=1), randn(264, 136, seed=2), randn(136, seed=3)))
    y = m.grouped_linear(m.rms_norm(x, g), w)
    dy = randn(50, 264, seed=4)
    first = torch.autograd.grad(y, (x, w, g), dy, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(y, (x, w, g), dy)))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, (x, w, g), dy)


def test_one_weight_for_all_experts(sonicmoe):
    """A weight that is expanded over the experts gets the sum of their gradients."""
    m = sonicmoe
    x, w, dy = randn(90, 72, seed=1), randn(1, 80, 72, seed=2).requires_grad_(True), randn(90, 80, seed=3)
    efo = torch.tensor([0, 40, 47, 90], dtype=torch.int32, device=DEV)
    y = m.grouped_linear(x, w.expand(3, 80, 72), efo)
    dw, = torch.autograd.grad(y, w, dy)
    parts = sum((dy[a:b].double().T @ x[a:b].double() for a, b in ((0, 40), (40, 47), (47, 90))))
    assert torch.equal(y, m.grouped_linear(x, w.detach()[0].expand(3, 80, 72), efo)) and relative(dw[0], parts) < 2.0 ** -7


def test_recorded_calls_are_the_same_calls(sonicmoe):
    """With a recorder the calls go kernel by kernel: the same results and gradients, each launch named."""
    m = sonicmoe
    rows, efo = 77, torch.tensor([0, 30, 30, 61, 77], dtype=torch.int32, device=DEV)

    def step():
        x, g, w = randn(rows, 96, seed=1).requires_grad_(True), randn(96, seed=2).requires_grad_(True), randn(4, 40, 96, seed=3).requires_grad_(True)
        res = randn(rows, 96, seed=4).float().requires_grad_(True)
        n = m.rms_norm_quantized(x, g, res, scales="block128", with_output=True)
        y = m.grouped_linear(n.y, w, efo)
        grads = torch.autograd.grad([y, n.h], [x, g, res, w], [randn(rows, 40, seed=5), randn(rows, 96, seed=6).float()])
        total = m.clip_gradients(grads, 1.0)
        with torch.no_grad():
            alone = m.grouped_linear(m.rms_norm(x, g), w, efo)
        return [n.payload.view(torch.uint8), n.scales, n.y, n.h, y, *grads, total, m.gradient_norm(grads), alone]

    want, record = step(), []
    m.ops.set_recorder(record)
    try:
        got = step()
    finally:
        m.ops.set_recorder(None)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert [n for n, _, _ in record] == ["rms_norm", "grouped_rows", "grouped_rows", "grouped_wgrad", "rms_norm_bwd", "clip_gradients",
                                         "rms_norm", "grouped_rows", "gradient_norm"]
