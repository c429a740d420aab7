"""The norm and the products by expert where their forward pass is made again inside a backward pass (activation recomputation): the
gradients are those of the plain call, however the backward pass is asked for."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16
ROWS, K, N, E = 77, 96, 136, 3


@pytest.fixture(scope="module")
def sonicmoe():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import sonicmoe as m
    yield m
    torch.cuda.synchronize()
    m.ops.check_status(DEV)


def randn(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(BF).to(DEV)


class Recomputed(torch.autograd.Function):
    """Keeps the inputs alone and makes the forward pass again in the backward pass."""

    @staticmethod
    def forward(ctx, call, *inputs):
        ctx.call, ctx.inputs = call, inputs
        return call(*inputs)

    @staticmethod
    def backward(ctx, dy):
        again = []
        for t in ctx.inputs:
            a = t.detach().requires_grad_(t.requires_grad)
            if hasattr(t, "main_grad"):
                a.main_grad = t.main_grad
            again.append(a)
        with torch.enable_grad():
            out = ctx.call(*again)
        torch.autograd.backward(out, dy)
        return None, *(a.grad for a in again)


WAYS = {"plain": lambda call, *ts: call(*ts), "function": lambda call, *ts: Recomputed.apply(call, *ts),
        "checkpoint": lambda call, *ts: checkpoint(call, *ts, use_reentrant=False),
        "reentrant checkpoint": lambda call, *ts: checkpoint(call, *ts, use_reentrant=True)}


def leaves(wants, main_grad):
    """x, the norm's weight, the residual, the experts' weight: gradients of those that are named in `wants`."""
    ts = dict(x=randn(ROWS, K, seed=1), g=randn(K, seed=2), res=randn(ROWS, K, seed=3).float(), w=randn(E, N, K, seed=4))
    for n, t in ts.items():
        t.requires_grad_(n in wants)
        if main_grad and n in ("g", "w") and n in wants:
            t.main_grad = torch.full(t.shape, 2.0, device=DEV)
    return ts


def gradients(m, way, drive, wants, main_grad, quantized):
    efo = torch.tensor([0, 30, 30, ROWS], dtype=torch.int32, device=DEV)

    def call(x, g, res, w):
        y = m.rms_norm_quantized(x, g, res, with_output=True).y if quantized else m.rms_norm(x, g, res)[0]
        return m.grouped_linear(y, w, efo)

    ts = leaves(wants, main_grad)
    y = WAYS[way](call, *ts.values())
    dy = randn(ROWS, N, seed=5)
    asked = [ts[n] for n in wants]
    if drive == "grad":
        got = torch.autograd.grad(y, asked, dy, allow_unused=main_grad)
    else:
        y.backward(dy, **(dict(inputs=asked) if drive == "inputs" else {}))
        got = [t.grad for t in asked]
    return [y.detach()] + [t.main_grad if hasattr(t, "main_grad") else g for t, g in zip(asked, got)]


def drives(way, main_grad, wants):
    if way == "reentrant checkpoint":            # which drives a backward pass of its own, and hands copies on that have no accumulator
        return ["backward"] if not main_grad or wants == "x" else []
    return ["backward", "grad", "inputs"] if not main_grad or "x" in wants else ["backward", "inputs"]


@pytest.mark.parametrize("quantized", [False, True], ids=["rows", "payload"])
@pytest.mark.parametrize("way,main_grad,wants,drive", [
    (way, main_grad, wants, drive) for way in ("function", "checkpoint", "reentrant checkpoint") for main_grad in (False, True)
    for wants in ("x g res w", "x", "w", "g w", "x w") for drive in drives(way, main_grad, wants)])
def test_gradients_are_those_of_the_plain_call(sonicmoe, way, main_grad, wants, drive, quantized):
    wants = wants.split()
    want = gradients(sonicmoe, "plain", drive, wants, main_grad, quantized)
    got = gradients(sonicmoe, way, drive, wants, main_grad, quantized)
    assert all(g is not None for g in got)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("drive", ["backward", "grad", "inputs"])
def test_products_alone_one_gradient_at_a_time(sonicmoe, drive):
    """Nothing is saved that no gradient needs, and what one needs is."""
    efo = torch.tensor([0, 30, 30, ROWS], dtype=torch.int32, device=DEV)
    dy = randn(ROWS, N, seed=5)
    for want in ("x", "w"):
        results = []
        for way in ("plain", "function", "checkpoint"):
            x, w = randn(ROWS, K, seed=1), randn(E, N, K, seed=4)
            leaf = (x if want == "x" else w).requires_grad_(True)
            y = WAYS[way](lambda a, b: sonicmoe.grouped_linear(a, b, efo), x, w)
            if drive == "grad":
                g, = torch.autograd.grad(y, leaf, dy)
            else:
                y.backward(dy, **(dict(inputs=[leaf]) if drive == "inputs" else {}))
                g = leaf.grad
            results.append(g)
        assert all(r is not None and torch.equal(r, results[0]) for r in results)
