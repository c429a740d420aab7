"""Routing metadata of rows that name an expert twice: every entry that a reader follows is written, whatever the buffers held."""
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


@pytest.mark.parametrize("order", [0, 1])
@pytest.mark.parametrize("N,E,K", [(1, 4, 2), (1, 2, 8), (33, 8, 3), (700, 5, 8), (3000, 16, 4), (5000, 200, 16)])
def test_entries_of_repeated_experts(sonicmoe, N, E, K, order):
    from sonicmoe._lib import check, lib
    idx = torch.randint(-1, E, (N, K), generator=torch.Generator().manual_seed(N + K), dtype=torch.int32)
    idx[-1] = E - 1                                            # the last row: one expert in every slot
    probs = torch.rand(N, K, generator=torch.Generator().manual_seed(1))
    TK, TKp = N * K, -(-N * K // 128) * 128 + E * 128
    make = lambda n, dtype=torch.int32: torch.full((n,), -7, dtype=dtype, device=DEV)
    efo, x_gather, s_scatter, s_rev, naept, src, counts = (make(n) for n in (E + 1, TKp, TKp, TK, N + 1, TK, E))
    scores = make(TKp, torch.float32)
    ws = torch.empty(lib.smoe_topk_metadata_workspace(N, E), dtype=torch.uint8, device=DEV)
    di, dp = idx.to(DEV), probs.to(DEV)
    P = lambda t: t.data_ptr()
    check(lib.smoe_topk_metadata(P(di), P(dp), N, K, E, 128, TK, TKp, order, 0, P(efo), P(x_gather), P(s_scatter), P(s_rev), P(naept),
                                 P(scores), P(src), P(counts), P(ws), torch.cuda.current_stream().cuda_stream), "topk_metadata")
    rows, rev, of, at, first, sc, gather = (t.cpu().tolist() for t in (counts, s_rev, src, naept, efo, scores, x_gather))
    chosen = [[(e, k) for k, e in enumerate(r) if e >= 0] for r in idx.tolist()]
    assert rows == [sum(any(e == c for c, _ in r) for r in chosen) for e in range(E)]          # a row counts once for an expert
    seen = [0] * E
    n = 0
    for t, r in enumerate(chosen):
        assert at[t] == n
        place = {}
        for e in sorted({e for e, _ in r}):
            place[e] = first[e] + seen[e]
            seen[e] += 1
        for e, k in sorted(r) if order == 0 else r:
            assert rev[n] == place[e] and gather[place[e]] == t and of[n] == t * K + k and sc[n] == probs[t, k]
            n += 1
    assert at[N] == n
    assert all(v == 0 for v in rev[n:] + of[n:]) and all(v == 0 for v in sc[n:])
