"""The norm of a list of gradients and their clipping against 64 bits."""
import pytest
import torch

from oracle import norm as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
BF, F32 = torch.bfloat16, torch.float32
# f32 sums of eight squares (each rounded, seven additions), f64 beyond, a root that halves the error, a rounding to f32
NORM = (8 / 2 + 1) * U


@pytest.fixture(scope="module")
def sonicmoe():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import sonicmoe as m
    yield m
    torch.cuda.synchronize()


def make(shapes, types, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(*s, generator=g) * scale).to(types[i % len(types)]) for i, s in enumerate(shapes)]


def on(ts):
    return [t.to(DEV) for t in ts]


LISTS = [
    [(1,)], [(7,)], [(8,)], [(4096,)], [(4097,)], [(3, 5, 7), (0,), (2, 0, 3), (16, 8)], [(1 << 20,), (1,)],
    [(i % 37 + 1, i % 11 + 1) for i in range(48)], [(i % 37 + 1,) for i in range(49)], [(5, i % 900) for i in range(640)],
    [(i % 300,) for i in range(641)], [(3000, 1111), (17,), (2048, 2048)], [(33, 1001)] * 1300,
]


@pytest.mark.parametrize("shapes", LISTS, ids=range(len(LISTS)))
@pytest.mark.parametrize("types", [(F32,), (BF,), (F32, BF)], ids=["f32", "bf16", "mixed"])
def test_norm_and_clipping(sonicmoe, shapes, types):
    grads = make(shapes, types)
    want = O.gradient_norm(grads)
    dev = on(grads)
    n = sonicmoe.gradient_norm(dev)
    assert n.shape == () and n.dtype == F32
    assert abs(float(n) - float(want)) <= NORM * float(want)
    assert torch.equal(n, sonicmoe.gradient_norm(dev))                      # one order
    for max_norm in (float(want) / 3, float(want) * 2, 0.0):
        refs = O.clipped(grads, max_norm)
        for outs in (None, [torch.full(g.shape, 9.0, dtype=BF, device=DEV) for g in dev],
                     [torch.full(g.shape, 9.0, dtype=F32, device=DEV) for g in dev]):
            src = [g.clone() for g in dev]
            m = sonicmoe.clip_gradients(src, max_norm, out=outs)
            assert torch.equal(m, n)
            for g, o, ref, old in zip(grads, src if outs is None else outs, refs, src):
                half = torch.finfo(o.dtype).eps / 2
                # the factor: the norm's error, its quotient and its rounding; one product; the result's type
                bound = ref.abs() * (NORM + 3 * U + half * 1.01) + 1e-45
                assert ((o.cpu().double() - ref).abs() <= bound).all()
                if outs is not None:
                    assert torch.equal(old.cpu(), g)
            if max_norm > float(want) and outs is None:
                assert all(torch.equal(a, b) for a, b in zip(src, dev))


@pytest.mark.parametrize("value", [1e-40, 1e-30, 1e-20, 1e-15, 1e10, 1e17, 1e20, 1e30, 3e38])
def test_squares_beyond_the_range_of_f32(sonicmoe, value):
    for n in (1, 9, 5000):
        g = torch.full((n,), value)
        want = O.gradient_norm([g])
        got = sonicmoe.gradient_norm(on([g]))
        if float(want) > 3.4028e38:
            assert torch.isinf(got)
        else:
            assert abs(float(got) - float(want)) <= NORM * float(want) + 1e-45
    mixed = [torch.tensor([1e-25, 1e30, 1.0] * 11), torch.tensor([1e-30] * 100)]
    assert abs(float(sonicmoe.gradient_norm(on(mixed))) / float(O.gradient_norm(mixed)) - 1) <= NORM


def test_nan_and_infinity(sonicmoe):
    g = make([(100,), (3, 40)], (F32,))
    bad = [t.clone() for t in g]
    bad[1][2, 7] = float("nan")
    dev = on(bad)
    assert sonicmoe.clip_gradients(dev, 1.0).isnan() and all(t.isnan().all() for t in dev)
    bad[1][2, 7] = -float("inf")
    dev = on(bad)
    assert torch.isinf(sonicmoe.clip_gradients(dev, 1.0))
    assert not dev[0].any() and dev[1][2, 7].isnan() and dev[1].nan_to_num().eq(0).all()
    dev = on(g)
    n = sonicmoe.clip_gradients(dev, float("inf"))
    assert all(torch.equal(a.cpu(), b) for a, b in zip(dev, g)) and torch.isfinite(n)


def test_parameters_stand_for_their_gradients(sonicmoe):
    p = [torch.nn.Parameter(torch.randn(4, 8, device=DEV).to(BF)) for _ in range(4)]
    p[0].main_grad = torch.randn(4, 8, device=DEV)
    p[0].grad = torch.randn(4, 8, device=DEV).to(BF)
    p[1].grad = torch.randn(4, 8, device=DEV).to(BF)
    p[3].main_grad = torch.randn(4, 8, device=DEV)
    kept = p[0].grad.clone()
    loose = torch.randn(5, device=DEV)
    grads = [p[0].main_grad, p[1].grad, p[3].main_grad, loose]
    refs = O.clipped([g.cpu() for g in grads], 0.5)
    version = p[1].grad._version
    n = sonicmoe.clip_gradients(iter(p + [loose]), 0.5)
    assert torch.isfinite(n)
    for g, r in zip(grads, refs):
        assert ((g.cpu().double() - r).abs() <= r.abs() * (2.0 ** -8 if g.dtype == BF else 10 * U)).all()
    assert torch.equal(p[0].grad, kept) and p[1].grad._version > version


class OwnAccumulator(torch.nn.Parameter):
    """A parameter that keeps its accumulator elsewhere."""
    @property
    def main_grad(self):
        return self.kept[0]


def test_wherever_an_accumulator_is_kept(sonicmoe):
    def parameter(cls=torch.nn.Parameter):
        p = cls(torch.zeros(40, device=DEV))
        p.grad = torch.full_like(p, 100.0)
        return p

    plain, none, attribute, own, frozen = parameter(), parameter(), parameter(), parameter(OwnAccumulator), parameter()
    none.main_grad = None
    attribute.main_grad = torch.full((40,), 2.0, device=DEV)
    own.kept = [torch.full((40,), 3.0, device=DEV)]
    frozen.grad = None
    buffer = torch.full((40,), 4.0, device=DEV).requires_grad_(False)
    items = [plain, none, attribute, own, frozen, buffer]
    total = (40 * (2 * 100.0 ** 2 + 4 + 9 + 16)) ** 0.5
    assert abs(float(sonicmoe.gradient_norm(items)) / total - 1) <= NORM
    versions = [t._version for t in (plain.grad, attribute.main_grad, own.kept[0], buffer)]
    assert abs(float(sonicmoe.clip_gradients(iter(items), total / 2)) / total - 1) <= NORM
    for t, v, was in zip((plain.grad, attribute.main_grad, own.kept[0], buffer), (100.0, 2.0, 3.0, 4.0), versions):
        assert torch.allclose(t, torch.full_like(t, v / 2), rtol=8 * U) and t._version == was + 1
    assert abs(float(sonicmoe.gradient_norm(attribute)) / (160 ** 0.5 / 2) - 1) <= NORM + 8 * U      # alone, without a list


def test_a_given_norm(sonicmoe):
    g = make([(1000,), (7, 9)], (F32, BF))
    dev = on(g)
    norm = torch.tensor(40.0, device=DEV)
    out = sonicmoe.clip_gradients(dev, 10.0, norm=norm)
    assert out is norm
    for a, b in zip(dev, g):
        r = b.double() * (10 / (40 + 1e-6))
        assert ((a.cpu().double() - r).abs() <= r.abs() * (3 * U + torch.finfo(a.dtype).eps / 2 * 1.01)).all()


def test_views_and_strides(sonicmoe):
    base = torch.randn(4000, device=DEV)
    views = [base[1:514], base[600:1001], base[1100:1500].view(20, 20).T, base[2000:4000:2]]
    refs = O.clipped([v.cpu() for v in views], 1.0)
    untouched = base.clone()
    n = sonicmoe.clip_gradients(views, 1.0)
    assert abs(float(n) / float(O.gradient_norm([v.cpu() for v in (untouched[1:514], untouched[600:1001], untouched[1100:1500],
                                                                   untouched[2000:4000:2])])) - 1) <= NORM
    for v, r in zip(views, refs):
        assert ((v.cpu().double() - r).abs() <= r.abs() * 12 * U).all()
    for a, b in ((0, 1), (514, 600), (1001, 1100), (1500, 2000)):
        assert torch.equal(base[a:b], untouched[a:b])
    assert torch.equal(base[2001:4000:2], untouched[2001:4000:2])
    # outputs off a 16-byte boundary, of another type
    flat = torch.full((1030,), 7.0, dtype=BF, device=DEV)
    outs = [flat[1:514], flat[515:916]]
    srcs = [untouched[1:514], untouched[600:1001]]
    sonicmoe.clip_gradients(srcs, 1.0, out=outs)
    for o, r in zip(outs, O.clipped([s.cpu() for s in srcs], 1.0)):
        assert ((o.cpu().double() - r).abs() <= r.abs() * 2.0 ** -8 * 1.01).all()
    assert (flat[0] == 7) and (flat[514] == 7) and (flat[916:] == 7).all()


def test_in_a_graph_and_on_another_stream(sonicmoe):
    shapes = [(100, 33), (5,), (4096, 16)]
    static, outs = on(make(shapes, (F32, BF))), [torch.empty(s, dtype=BF, device=DEV) for s in shapes]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        sonicmoe.clip_gradients(static, 1.0, out=outs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        n = sonicmoe.clip_gradients(static, 1.0, out=outs)
        sonicmoe.clip_gradients(static, 1.0)
    for seed in (1, 2):
        fresh = on(make(shapes, (F32, BF), seed=seed, scale=3.0))
        for a, b in zip(static, fresh):
            a.copy_(b)
        ref_outs = [torch.empty_like(o) for o in outs]
        ref_n = sonicmoe.clip_gradients(fresh, 1.0, out=ref_outs)
        graph.replay()
        assert torch.equal(n, ref_n) and all(torch.equal(a, b) for a, b in zip(outs, ref_outs))
        sonicmoe.clip_gradients(fresh, 1.0)
        assert all(torch.equal(a, b) for a, b in zip(static, fresh))


def test_more_than_32_bits_of_values(sonicmoe):
    n = (1 << 31) + 12345
    g = torch.zeros(n, dtype=BF, device=DEV)
    at = [0, 1 << 30, (1 << 31) - 1, 1 << 31, n - 1]
    for i, p in enumerate(at):
        g[p] = float(i + 1)
    norm = sonicmoe.clip_gradients([g], 1.0)
    want = sum((i + 1) ** 2 for i in range(5)) ** 0.5
    assert abs(float(norm) - want) <= NORM * want
    for i, p in enumerate(at):
        assert abs(float(g[p]) - (i + 1) / want) <= (i + 1) / want * 2.0 ** -8 * 1.01
