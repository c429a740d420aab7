"""What group-limited routing and the block-128 products refuse, on the host: no call here reaches a kernel.  And the oracles' own
rules, against loops and differences."""
import math

import pytest
import torch

from oracle import block128 as O
from oracle import group_routing as G

SHAPE, ALIGN, ARG = 1, 2, 6
P = 4096          # an address that is never looked at


@pytest.fixture(scope="module")
def lib(built_library):
    from sonicmoe._lib import lib
    return lib


@pytest.fixture(scope="module")
def sonicmoe(built_library):
    import sonicmoe
    return sonicmoe


def test_routing_refuses(lib):
    def call(T=4, E=64, K=4, groups=8, top=4, score=2, logits=P, scores=P, idx=P):
        return lib.smoe_group_routing(logits, 0, None, T, E, K, groups, top, score, 0, 1, 1.0, scores, idx, None)
    for kw in (dict(E=0), dict(E=1025), dict(K=0), dict(K=33), dict(K=65), dict(groups=0), dict(groups=7), dict(groups=64),
               dict(top=0), dict(top=9), dict(K=9, top=1), dict(T=-1)):
        assert call(**kw) == SHAPE, kw
    for kw in (dict(score=0), dict(score=3), dict(logits=None), dict(scores=None), dict(idx=None)):
        assert call(**kw) == ARG, kw
    assert call(T=0, logits=None, scores=None, idx=None) == 0
    bwd = lambda T=4, E=64, K=4, p=P: lib.smoe_group_routing_bwd(p, 0, P, P, T, E, K, 0, 1, 1.0, P, None)
    assert bwd(E=1025) == bwd(K=33) == bwd(T=-1) == SHAPE and bwd(p=None) == ARG and bwd(T=0, p=None) == 0


def test_quantisers_refuse(lib):
    rows = lambda x=P, n=4, K=128, q=P, s=P: lib.smoe_quant128_rows(x, n, K, 0, None, None, 0, q, s, None)
    assert rows(K=0) == rows(K=12) == rows(n=-1) == rows(n=1 << 31) == SHAPE
    assert rows(x=None) == rows(q=None) == rows(s=None) == ARG
    assert rows(x=P + 8) == rows(q=P + 8) == rows(s=P + 2) == ALIGN
    assert rows(n=0, x=None, q=None, s=None) == 0
    assert lib.smoe_quant128_rows(P, 4, 128, 0, P, None, 4, P, P, None) == ARG             # a list without its length
    dual = lambda efo=None, counts=None, E=1, st=P, K=128: lib.smoe_quant128_dual(P, 4, K, efo, counts, E, P, P, P, st, None)
    assert dual(K=4) == SHAPE and dual(counts=P) == ARG and dual(efo=P, E=0) == ARG and dual(st=P + 4) == ALIGN
    weight = lambda E=1, N=4, K=128, w=P: lib.smoe_quant128_weight(w, E, N, K, P, P, None)
    assert weight(K=4) == weight(E=-1) == weight(E=65536) == SHAPE and weight(w=P + 2) == ALIGN and weight(E=0) == 0
    assert lib.smoe_quant128_rows_scatter(P, 4, 128, None, P, 128, P, P, None) == ARG


def test_products_refuse(lib):
    def rows(a=P, s=P, b=P, efo=None, counts=None, c=P, n=4, N=128, K=128, E=1, status=P, few=False):
        if few:
            return lib.smoe_gemm128_few(a, s, b, P, efo, counts, c, n, N, K, E, 0, status, None, None)
        return lib.smoe_gemm128_rows(a, s, b, P, efo, counts, c, n, N, K, E, 0, 1, status, None, None)
    for few in (False, True):
        for kw in (dict(n=-1), dict(n=1 << 31), dict(N=0), dict(N=12), dict(K=20), dict(K=0), dict(E=0), dict(E=257, efo=P)):
            assert rows(few=few, **kw) == SHAPE, kw
        for kw in (dict(E=2), dict(counts=P), dict(a=None), dict(b=None), dict(c=None), dict(s=None), dict(status=None)):
            assert rows(few=few, **kw) == ARG, kw
        for kw in (dict(a=P + 8), dict(b=P + 4), dict(c=P + 8), dict(s=P + 4)):
            assert rows(few=few, **kw) == ALIGN, kw
        assert rows(few=few, n=0, a=None, b=None, c=None, s=None) == 0
    wgrad = lambda M=128, N=128, n=128, bf16=0, acc=0, c=P, E=1: lib.smoe_gemm128_wgrad(P, P, P, P, None, None, c, M, N, n, E, bf16, acc,
                                                                                      P, None, None)
    assert wgrad(M=12) == wgrad(N=0) == wgrad(n=-1) == wgrad(E=0) == SHAPE
    assert wgrad(bf16=1, acc=1) == wgrad(c=None) == wgrad(E=2) == ARG and wgrad(c=P + 4) == ALIGN
    assert wgrad(n=0, acc=1) == 0


def test_whole_passes_refuse_and_say_what_they_need(lib):
    size = lambda rows=256, N=128, K=384, E=2, flags=7, which=0: lib.smoe_block128_bytes(rows, N, K, E, flags, which)
    assert size(N=4) == size(K=12) == size(E=0) == size(E=257) == size(rows=-1) == -1
    assert size(flags=0) == 0 and size(flags=4, which=2) < size(flags=6, which=2)
    # payload and scales of the weight and of x by columns; of x by rows; of dy in both forms, each part on 256 bytes
    up = lambda n: -(-n // 256) * 256
    assert size() == up(2 * 128 * 384) + up(4 * 2 * 3) + up(256 * 384) + up(4 * 2 * 384)
    assert size(which=1) == up(256 * 384) + up(4 * 256 * 3)
    assert size(which=2) == 2 * up(256 * 128) + up(4 * 256) + up(4 * 2 * 128)
    assert size(rows=0) > 0 and size(rows=0, which=1) == 0
    assert lib.smoe_block128_linear(P, P, P, None, None, P, None, None, 4, 128, 128, 1, 0, P, None, None) == ARG        # no scratch
    assert lib.smoe_block128_linear(P, P, P, None, None, P, None, P, 4, 128, 128, 1, 2, P, None, None) == ARG           # nowhere to save
    assert lib.smoe_block128_linear_bwd(P, P, P, None, None, None, P, P, P, 4, 128, 128, 1, 6, 0, P, None, None) == ARG
    experts = lambda T=4, H=128, I=64, E=8, K=2: lib.smoe_block128_experts_bytes(T, H, I, E, K)
    assert experts(K=17) == experts(K=0) == experts(E=257) == experts(H=4) == experts(I=12) == experts(T=-1) == experts(T=1 << 30) == -1
    assert experts() > 0 and lib.smoe_block128_experts(None, P, P, P, P, P, P, P, P, 4, 128, 64, 8, 2, P, None, None) == ARG
    assert lib.smoe_block128_experts(*[None] * 9, 0, 128, 64, 8, 2, None, None, None) == 0


def test_python_entry_points_refuse(sonicmoe):
    route = sonicmoe.group_limited_routing
    logits = torch.zeros(4, 64)
    for bad in (dict(score="tanh"), dict(groups=7), dict(groups=33), dict(groups=0), dict(groups=8, top_groups=9),
                dict(groups=8, top_groups=0), dict(group_score=3), dict(bias=torch.zeros(63)), dict(bias=torch.zeros(1, 64))):
        with pytest.raises(ValueError):
            route(logits, 4, **bad)
    for bad, K in ((logits, 0), (logits, 33), (logits, 65), (logits[0], 4), (logits.half(), 4), (torch.zeros(4, 1025), 4)):
        with pytest.raises(ValueError):
            route(bad, K)
    with pytest.raises(ValueError):
        route(logits, 9, groups=8, top_groups=1)
    with pytest.raises(RuntimeError, match="CUDA"):
        route(logits, 4)

    linear = sonicmoe.block128_linear
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)
    e4 = lambda *s: torch.zeros(*s, dtype=torch.uint8).view(torch.float8_e4m3fn)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)
    x, w, efo, cnt = bf(256, 64), bf(2, 128, 64), i32(3), i32(2)
    for bad in ((x.float(), w, efo, cnt), (x, w.float(), efo, cnt), (x, w[0, 0], None, None), (bf(256, 72), w, efo, cnt),
                (x, w, None, None), (x, w, None, cnt), (x, w, i32(2), cnt), (x, w, efo, i32(3)), (x, w, efo.long(), cnt),
                (x, w, efo, cnt.long()), (bf(2, 128, 64), w, efo, cnt), (x, w[0], None, cnt),
                (x, (w, torch.zeros(2, 1, 1)), efo, cnt), (x, (e4(2, 128, 64), torch.zeros(2, 2, 1)), efo, cnt),
                (x, (e4(2, 128, 64), torch.zeros(2, 1, 1, dtype=torch.float64)), efo, cnt),
                (x, (e4(2, 128, 80)[..., :64], torch.zeros(2, 1, 1)), efo, cnt)):
        with pytest.raises(ValueError):
            linear(*bad)
    with pytest.raises(RuntimeError, match="CUDA"):
        linear(x, w, efo, cnt)

    experts = sonicmoe.block128_experts
    pair = lambda E, N, K: (e4(E, N, K), torch.zeros(E, -(-N // 128), -(-K // 128)))
    good = dict(x=bf(4, 64), idx=i32(4, 2), sc=torch.zeros(4, 2), w1=pair(8, 256, 64), w2=pair(8, 64, 128))
    for bad in (dict(x=bf(4, 2, 64)), dict(x=torch.zeros(4, 64)), dict(w1=pair(8, 256, 72)), dict(w2=pair(8, 64, 136)),
                dict(w2=pair(7, 64, 128)), dict(idx=i32(3, 2)), dict(sc=torch.zeros(4, 3)), dict(idx=i32(4))):
        a = {**good, **bad}
        with pytest.raises(ValueError):
            experts(a["x"], a["idx"], a["sc"], a["w1"], a["w2"])
    with pytest.raises(RuntimeError, match="CUDA"):
        experts(good["x"], good["idx"], good["sc"], good["w1"], good["w2"])
    for f in (sonicmoe.quantize_rows_block128, sonicmoe.quantize_weight_block128):
        with pytest.raises(RuntimeError, match="CUDA"):
            f(x)


def test_the_oracle_of_a_scale(built_library):
    """Block by block as the rule reads."""
    x = torch.randn(3, 300, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    q, s = O.quant_rows(x)
    for r in range(3):
        for b in range(3):
            v = x[r, 128 * b:128 * b + 128].float()
            a = v.abs().max()
            assert s[r, b] == torch.tensor([a.item()]).div(torch.tensor([448.0]))[0]
            step = torch.maximum(2.0 ** -3 * v.abs(), s[r, b] * 2.0 ** -9)              # e4m3: three bits behind the first
            assert ((q[r, 128 * b:128 * b + 128].float() * s[r, b] - v).abs() <= step * 0.5 * (1 + 1e-6)).all()
    wq, ws = O.quant_weight(torch.randn(1, 130, 136, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16))
    cq, cs = O.quant_cols(x)
    assert ws.shape == (1, 2, 2) and cs.shape == (1, 300) and torch.equal(cq.float().abs().amax(0), torch.full((300,), 448.0))


def test_the_oracle_of_a_choice():
    logits = torch.tensor([[0.0, 2.0, 1.0, 2.0, -math.inf, 3.0, 0.5, 0.5]])
    assert G.choose(logits[0], None, 3, 1, 1, 2, False) == [5, 1, 3]
    # groups {0,1} {2,3} {4,5} {6,7}: sums of two scores; the third has one open expert
    assert G.choose(logits[0], None, 3, 4, 2, 2, False) == [1, 3, 2]
    assert G.choose(logits[0], None, 3, 4, 1, 1, False) == [5, -1, -1]
    bias = torch.tensor([9.0, 0, 0, 0, 9.0, 0, 0, 0])
    assert G.choose(logits[0], bias, 3, 1, 1, 2, True) == [0, 5, 1]
    g = torch.tensor([[1.0, -2.0, 0.5]])
    idx = torch.tensor([[5, 1, -1]], dtype=torch.int32)
    for softmax in (False, True):
        grad, x = G.route_grad(logits, idx, g, softmax, True, 1.5), logits.double()
        for e in (0, 1, 5, 7):
            d = torch.zeros_like(x)
            d[0, e] = 1e-5
            slope = sum(w * (G.scores_of(x + w * d, idx, softmax, True, 1.5) * g.double()).sum() for w in (1, -1)) / 2e-5
            assert abs(float(slope - grad[0, e])) < 1e-8
        assert grad[0, 4] == 0
