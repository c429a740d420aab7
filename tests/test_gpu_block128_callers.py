"""Block-128 operators on what callers hold: parts of stacked checkpoints, accumulators inside a flat buffer, a first call that is being
captured, bounds that were too low."""
import os
import subprocess
import sys

import pytest
import torch

from oracle import block128 as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = 2.0 ** -8                     # half a step of bf16, relative
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def sonicmoe():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import sonicmoe as m
    yield m
    torch.cuda.synchronize()
    m.ops.check_status(DEV)


def f32_tol(K):
    """Roundings of a sum of K products in f32 by blocks of 128, whatever their order, relative to the sum of the terms' magnitudes;
    twice 2^-24 each, for an adder that cuts instead of rounding."""
    return (min(K, 128) + -(-K // 128) + 4) * 2.0 ** -23


def randn(*shape, seed=0, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(torch.bfloat16)


def table(counts):
    efo = torch.zeros(len(counts) + 1, dtype=torch.int32)
    efo[1:] = torch.tensor([-(-c // 128) * 128 for c in counts]).cumsum(0)
    return efo, torch.tensor(counts, dtype=torch.int32), int(efo[-1])


@pytest.mark.parametrize("N,K", [(384, 384), (520, 328), (328, 1400)])
def test_parts_of_stacked_weights(sonicmoe, N, K):
    """An odd number of scales a matrix: every expert's but the first start off a 16-byte boundary."""
    E, rows = 5, 200
    x, w, dy = randn(rows, K, seed=1), randn(E, N, K, seed=2), randn(rows, N, seed=3)
    q, s = sonicmoe.quantize_weight_block128(w.to(DEV))
    xs = x.to(DEV)
    for e in (1, 2, 3):
        assert s[e].data_ptr() % 16
        for n in (1, 70, rows):                               # the kernel for few rows, and tiles
            got, want = [], []
            for part, out in (((q[e], s[e]), got), ((q[e], s[e].clone()), want)):
                a = xs[:n].clone().requires_grad_(True)
                y = sonicmoe.block128_linear(a, part)
                out += [y.detach(), *torch.autograd.grad(y, a, dy[:n].to(DEV))]
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    efo, counts, n = table([130, 0, 40])
    x = randn(n, K, seed=4).to(DEV)
    y = sonicmoe.block128_linear(x, (q[1:4], s[1:4]), efo.to(DEV), counts.to(DEV))
    assert torch.equal(y, sonicmoe.block128_linear(x, (q[1:4], s[1:4].clone()), efo.to(DEV), counts.to(DEV)))


@pytest.mark.parametrize("T", [3, 200])
def test_an_expert_parallel_rank_of_stacked_layers(sonicmoe, T):
    E, H, I, K = 6, 384, 192, 2                               # 3 x 3 and 3 x 2 scales an expert
    w1 = sonicmoe.quantize_weight_block128(randn(E, 2 * I, H, seed=1, scale=H ** -0.5).to(DEV))
    w2 = sonicmoe.quantize_weight_block128(randn(E, H, I, seed=2, scale=I ** -0.5).to(DEV))
    x = randn(T, H, seed=3).to(DEV)
    scores, idx = torch.rand(T, 3, generator=torch.Generator().manual_seed(4)).topk(K)
    part = [tuple(t[3:] for t in w) for w in (w1, w2)]
    assert part[0][1].data_ptr() % 16 and part[1][1].data_ptr() % 16
    a = sonicmoe.block128_experts(x, idx.int().to(DEV), scores.to(DEV), *part)
    b = sonicmoe.block128_experts(x, idx.int().to(DEV), scores.to(DEV), *(tuple(t.clone() for t in w) for w in part))
    assert torch.equal(a, b)


def test_kernel_by_kernel_on_scales_off_a_boundary(sonicmoe):
    ops = sonicmoe.ops
    off = lambda t: torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape)
    xq, xs = ops.quant128_rows(randn(70, 264).to(DEV))
    wq, ws = ops.quant128_weight(randn(1, 136, 264, seed=1).to(DEV))
    dq, ds = ops.quant128_rows(randn(70, 136, seed=2).to(DEV))
    col = [ops.quant128_dual(randn(70, n, seed=3).to(DEV), with_rows=False)[2:] for n in (136, 264)]
    assert off(xs).data_ptr() % 16 and off(ws).data_ptr() % 16
    for f in (ops.gemm128_rows, ops.gemm128_few):
        assert torch.equal(f(xq, off(xs), wq, off(ws)), f(xq, xs, wq, ws))
    assert torch.equal(ops.gemm128_rows(dq, off(ds), wq, off(ws), b_mn=True), ops.gemm128_rows(dq, ds, wq, ws, b_mn=True))
    (a, s), (b, t) = col
    assert torch.equal(ops.gemm128_wgrad(a, off(s), b, off(t)), ops.gemm128_wgrad(a, s, b, t))


def test_an_accumulator_inside_a_flat_buffer(sonicmoe):
    """A main_grad that starts at any element is added to like one that starts on a boundary."""
    E, N, K = 2, 136, 264
    efo, counts, rows = table([130, 70])
    x, dy = randn(rows, K, seed=1).to(DEV), randn(rows, N, seed=2).to(DEV)
    start = torch.randn(E, N, K, generator=torch.Generator().manual_seed(3)).to(DEV)
    got = []
    for pad in (0, 1):
        w = randn(E, N, K, seed=4).to(DEV).requires_grad_(True)
        flat = torch.full((E * N * K + 9,), 5.0, device=DEV)
        w.main_grad = flat[pad:pad + E * N * K].view(E, N, K)
        w.main_grad.copy_(start)
        a = x.clone().requires_grad_(True)
        sonicmoe.block128_linear(a, w, efo.to(DEV), counts.to(DEV)).backward(dy)
        assert w.grad is None and (flat[:pad] == 5).all() and (flat[pad + E * N * K:] == 5).all()
        got.append((w.main_grad.clone(), a.grad))
    assert w.main_grad.data_ptr() % 16
    assert torch.equal(got[0][1], got[1][1])
    assert torch.equal(got[0][0], got[1][0])


def test_more_rows_than_a_few_row_product_was_told(sonicmoe):
    """`live_rows` only divides the work: told too few, clusters of CTAs that share a tile's reduction take several tiles each."""
    ops = sonicmoe.ops
    counts = [70, 0, 129, 64, 1, 200]
    efo, cnt, rows = table(counts)
    live = O.live_rows(efo, cnt, rows)
    # blocks of the reduction and weight tiles for clusters of 2, of 4 and of 8 where one row is expected on some 148 SMs
    for N, K in ((5120, 1536), (4608, 1536), (1000, 6152)):
        x, w = randn(rows, K, seed=N), randn(len(counts), N, K, seed=K)
        xq, xs = ops.quant128_rows(x.to(DEV))
        wq, ws = ops.quant128_weight(w.to(DEV))
        y = ops.gemm128_few(xq, xs, wq, ws, efo.to(DEV), cnt.to(DEV), live_rows=1)
        again = ops.gemm128_few(xq, xs, wq, ws, efo.to(DEV), cnt.to(DEV), live_rows=1)
        assert torch.equal(y[live.to(DEV)], again[live.to(DEV)])
        ref, mag = O.rows_product(O.deq_rows(*O.quant_rows(x)), O.deq_weight(*O.quant_weight(w)), efo, cnt)
        err = (y.cpu().double() - ref).abs()
        assert (err <= BF16 * ref.abs() + f32_tol(K) * mag * (1 + BF16))[live].all()
    ops.check_status(DEV)


def test_live_rows_of_products_that_leave_the_others(sonicmoe):
    """Every live row is written, with the product, where tiles are laid over live rows only."""
    ops = sonicmoe.ops
    from sonicmoe._lib import check, lib
    N, K = 264, 256
    for counts in ([3, 0, 70, 128], [257, 1, 0, 64], [0, 0, 513, 128]):
        efo, cnt, rows = table(counts)
        x, w = randn(rows, K), randn(4, N, K, seed=1)
        xq, xs = ops.quant128_rows(x.to(DEV))
        wq, ws = ops.quant128_weight(w.to(DEV))
        ref, mag = O.rows_product(O.deq_rows(*O.quant_rows(x)), O.deq_weight(*O.quant_weight(w)), efo, cnt)
        live = O.live_rows(efo, cnt, rows)
        e, n = efo.to(DEV), cnt.to(DEV)
        for few in (True, False):
            c = torch.full((rows, N), float("nan"), dtype=torch.bfloat16, device=DEV)
            P = lambda t: t.data_ptr()
            head = (P(xq), P(xs), P(wq), P(ws), P(e), P(n), P(c), rows, N, K, 4)
            tail = (P(ops.status_word(DEV)), None, torch.cuda.current_stream().cuda_stream)
            if few:
                check(lib.smoe_gemm128_few(*head, 0, *tail), "few")
            else:
                check(lib.smoe_gemm128_rows(*head, 0, 0, *tail), "rows")
            c = c.cpu()
            assert torch.isnan(c[~live]).all()
            assert ((c.double() - ref).abs() <= BF16 * ref.abs() + f32_tol(K) * mag * (1 + BF16))[live].all()


CAPTURED_FIRST = """
import sys
import torch
sys.path[:0] = [{root!r}, {root!r} + "/supersonic-moe_b200"]
import sonicmoe
x = torch.randn(40, 256, device="cuda").bfloat16()
w = torch.randn(136, 256, device="cuda").bfloat16()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = sonicmoe.block128_linear(x, w)
    word, host = sonicmoe.ops.failure_words(x.device)
status = sonicmoe.ops.status_word("cuda")
assert status.data_ptr() == word and host
assert int(status.item()) == 0, "before the first replay"
status.fill_(503)
graph.replay()
torch.cuda.synchronize()
assert int(status.item()) == 503, "a replay took a recorded failure back"
status.zero_()
assert torch.equal(y, sonicmoe.block128_linear(x, w))
assert sonicmoe.ops.failure_words(x.device) == (word, host)
sonicmoe.ops._posted[0][1].value = 502
try:
    sonicmoe.block128_linear(x, w)
    raise SystemExit("a failure that a replay posted did not surface")
except RuntimeError as e:
    assert "502" in str(e)
sonicmoe.ops.check_status("cuda")
print("captured first: ok")
"""


def test_the_first_call_of_a_process_is_captured(sonicmoe):
    """The word that kernels report failures in is no part of the graph, and the host sees it from a replay too."""
    run = subprocess.run([sys.executable, "-c", CAPTURED_FIRST.format(root=ROOT)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "captured first: ok" in run.stdout, run.stderr[-2000:]


def test_router_of_groups_into_the_layer(sonicmoe):
    """The router's tables are what the layer takes: its outputs and gradients are those of the same tables handed over as leaves."""
    T, E, K, H, I = 256, 8, 2, 256, 128
    x, w1, w2 = randn(T, H, seed=1).to(DEV), randn(E, 2 * I, H, seed=2, scale=H ** -0.5), randn(E, H, I, seed=3, scale=I ** -0.5)
    logits = torch.randn(T, E, generator=torch.Generator().manual_seed(4))
    logits[-9:] = -torch.inf                                  # a padded batch
    dy = randn(T, H, seed=5).to(DEV)
    outs = []
    for leaves in (False, True):
        a, b, c = (t.to(DEV).clone().requires_grad_(True) for t in (x, w1, w2))
        ld = logits.to(DEV).requires_grad_(True)
        scores, idx = sonicmoe.group_limited_routing(ld, K, groups=4, top_groups=2, scale=1.5)
        s = scores.detach().requires_grad_(True) if leaves else scores
        out = sonicmoe.run_sonic_moe(a, idx, s, K, E, b, c, fp8=True)
        out.backward(dy)
        if leaves:
            ld.grad, = torch.autograd.grad(scores, ld, s.grad)
        outs.append((out.detach(), a.grad, b.grad, c.grad, ld.grad))
    for u, v in zip(*outs):
        assert torch.isfinite(u).all() and torch.equal(u, v)
    assert (outs[0][0][-9:] == 0).all() and (outs[0][1][-9:] == 0).all() and (outs[0][4][-9:] == 0).all()
    assert outs[0][4].abs().max() > 0
