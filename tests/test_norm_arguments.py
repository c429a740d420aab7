"""Refusals of the norm and of gradient clipping: on the host, before anything is launched."""
import pytest
import torch

import sonicmoe

BF = torch.bfloat16


@pytest.mark.parametrize("x,w,res,kw", [
    (torch.zeros(2, 8, dtype=torch.float16), torch.zeros(8), None, {}),
    (torch.zeros(2, 8, dtype=BF), torch.zeros(7), None, {}),
    (torch.zeros(2, 8, dtype=BF), torch.zeros(8, dtype=torch.float16), None, {}),
    (torch.zeros(2, 8, dtype=BF), torch.zeros(1, 8), None, {}),
    (torch.zeros(2, 8, dtype=BF), torch.zeros(8), torch.zeros(2, 9, dtype=BF), {}),
    (torch.zeros(2, 8, dtype=BF), torch.zeros(8), torch.zeros(1, 8, dtype=BF), {}),
    (torch.zeros(2, 8), torch.zeros(8), torch.zeros(2, 8, dtype=BF), {}),
    (torch.zeros(2, 8, dtype=BF), torch.zeros(8), None, dict(eps=-1e-6)),
    (torch.zeros(2, 8, dtype=BF), torch.zeros(8), None, dict(eps=float("nan"))),
    (torch.zeros(2, 8, dtype=BF), torch.zeros(8), None, dict(eps=float("inf"))),
    (torch.zeros(1, 16385, dtype=BF), torch.zeros(16385), None, {}),
    (torch.zeros(3, 0, dtype=BF), torch.zeros(0), None, {}),
    (torch.zeros((), dtype=BF), torch.zeros(1), None, {}),
])
def test_norm_refusals(x, w, res, kw):
    for call in (sonicmoe.rms_norm, sonicmoe.rms_norm_quantized):
        with pytest.raises(ValueError):
            call(x, w, res, **kw)


def test_quantized_refusals():
    x, w = torch.zeros(2, 40, dtype=BF), torch.zeros(40)
    for bad in (dict(scales="mx"), dict(scales="fp8"), dict(scales=None)):
        with pytest.raises(ValueError):
            sonicmoe.rms_norm_quantized(x, w, **bad)
    with pytest.raises(ValueError):
        sonicmoe.rms_norm_quantized(x[:, :36], w[:36], scales="block128")
    with pytest.raises(ValueError):
        sonicmoe.rms_norm_quantized(torch.zeros(2, 64), torch.zeros(64))
    with pytest.raises(ValueError, match="with_output"):
        sonicmoe.rms_norm_quantized(x[:, :32].requires_grad_(True), w[:32])


def test_there_is_no_cpu_path():
    with pytest.raises(RuntimeError, match="CUDA"):
        sonicmoe.rms_norm(torch.zeros(2, 8, dtype=BF), torch.zeros(8))
    with pytest.raises(RuntimeError, match="CUDA"):
        sonicmoe.gradient_norm([torch.zeros(8)])
    with pytest.raises(RuntimeError, match="CUDA"):
        sonicmoe.clip_gradients([torch.zeros(8)], 1.0)


def test_clipping_refusals():
    g = torch.zeros(8)
    p = torch.nn.Parameter(torch.zeros(3))
    for call in (lambda: sonicmoe.gradient_norm([]), lambda: sonicmoe.gradient_norm([p]), lambda: sonicmoe.clip_gradients([p], 1.0),
                 lambda: sonicmoe.clip_gradients([g], -1.0), lambda: sonicmoe.clip_gradients([g], float("nan")),
                 lambda: sonicmoe.clip_gradients([g, g], 1.0), lambda: sonicmoe.clip_gradients([g, g[:4]], 1.0),
                 lambda: sonicmoe.clip_gradients([g], 1.0, norm=torch.zeros(2)),
                 lambda: sonicmoe.clip_gradients([g], 1.0, norm=torch.zeros((), dtype=torch.float64)),
                 lambda: sonicmoe.clip_gradients([g], 1.0, out=[]),
                 lambda: sonicmoe.clip_gradients([g], 1.0, out=[torch.zeros(7)]),
                 lambda: sonicmoe.clip_gradients([g], 1.0, out=[torch.zeros(16)[::2]]),
                 lambda: sonicmoe.clip_gradients([g, torch.zeros(8)], 1.0, out=[torch.zeros(8), g])):
        with pytest.raises(ValueError):
            call()
    o = torch.zeros(8)
    with pytest.raises(ValueError, match="twice"):
        sonicmoe.clip_gradients([g, torch.zeros(8)], 1.0, out=[o, o])


def test_clipping_refuses_memory_that_it_writes_twice():
    """Also where the tensors only overlap: the order of reads and writes would make the result."""
    g, other = torch.zeros(64), torch.zeros(64)
    bf = g.view(torch.bfloat16)
    for grads, kw in (([g, g[8:16]], {}), ([g[:40], other, g[32:]], {}), ([g[:8], bf[15:]], {}), ([g.view(8, 8).T, g.view(8, 8).T], {}),
                      ([g.view(8, 8)[:, :4], g], {}),
                      ([other, other.clone()], dict(out=[g, g])),
                      ([other[:8], other[8:16]], dict(out=[g[:8], g[4:12]])),
                      ([g[:8], other[:8]], dict(out=[other[8:16], g[7:15]])),          # another gradient's end
                      ([g[:8]], dict(out=[g[4:12]])), ([g[4:12]], dict(out=[g[:8]])),       # its own, shifted
                      ([g[:8]], dict(out=[bf[:8]])), ([bf[:8]], dict(out=[g[:8]])), ([g[:8]], dict(out=[bf[8:16]])),
                      ([g], dict(norm=g[3])), ([g[:8]], dict(out=[other[:8]], norm=other[7:8]))):
        with pytest.raises(ValueError, match="twice|lies"):
            sonicmoe.clip_gradients(grads, 1.0, **kw)
    # beside one another, within one another's gaps, over themselves, empty ones anywhere: these pass the checks and want a GPU
    for grads, kw in (([g[:8], g[8:]], {}), ([g.view(8, 8)[:, :4], g.view(8, 8)[:, 4:]], {}), ([g, g[8:8], g[8:8]], {}),
                      ([g[:8], g[8:16]], dict(out=[g[:8], g[8:16]])), ([g[:8], g[8:16]], dict(out=[g[16:24], g[8:16]])),
                      ([g[:8]], dict(norm=g[8])), ([g[:8]], dict(out=[other[:8]], norm=g[0])),
                      ([g.view(8, 8).T], dict(out=[g.view(8, 8)]))):
        with pytest.raises(RuntimeError, match="CUDA"):
            sonicmoe.clip_gradients(grads, 1.0, **kw)


def test_c_entry_points_check_their_arguments():
    from sonicmoe._lib import lib
    SHAPE, ALIGN, ARG = 1, 2, 6
    norm = lambda **k: lib.smoe_rms_norm(*({**dict(x=16, x32=0, ldx=64, res=None, r32=0, ldr=64, w=16, w32=0, T=2, H=64, eps=1e-6, y=16,
                                                   h=None, rstd=None, kind=0, q=None, s=None, stream=None), **k}.values()))
    assert norm(H=0) == norm(H=16385) == norm(ldx=63) == norm(T=-1) == norm(kind=1, H=40, q=16, s=16) == SHAPE
    assert norm(x=None) == norm(w=None) == norm(y=None) == norm(res=16) == norm(kind=3) == norm(kind=1) == norm(eps=-1.0) == ARG
    assert norm(x32=1, kind=1, q=16, s=16) == norm(x32=1, res=16, h=16) == ARG
    assert norm(kind=1, q=8, s=16) == ALIGN
    assert norm(T=0, x=None) == 0
    bwd = lambda **k: lib.smoe_rms_norm_bwd(*({**dict(dy=16, x32=0, h=16, h32=0, ldh=64, w=16, w32=0, rstd=16, dh=None, T=2, H=64, dx=16,
                                                      dres=None, dw=16, dw32=0, acc=0, ws=None, stream=None), **k}.values()))
    assert bwd(H=0) == bwd(ldh=1) == SHAPE and bwd() == bwd(x32=1) == bwd(acc=1) == bwd(dy=None) == ARG
    assert lib.smoe_rms_norm_bwd_workspace(4, 0) == -1 and lib.smoe_rms_norm_bwd_workspace(0, 8) == 0
    from array import array
    t = array("q", [18, 18, 4, 1 | 1 << 32])
    at = t.buffer_info()[0]
    assert lib.smoe_gradient_norm(at, 1, 16, 16, None) == ALIGN
    assert lib.smoe_gradient_norm(None, 1, 16, 16, None) == lib.smoe_gradient_norm(None, -1, 16, 16, None) == ARG
    assert lib.smoe_gradient_clip(None, 0, -1.0, None, 16, 16, None) == ARG
    assert lib.smoe_gradient_workspace(-1) == -1
