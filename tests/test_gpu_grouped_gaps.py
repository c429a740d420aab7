"""Products by expert over segments with counts that begin and end anywhere, of too many rows for the kernels of few: no tile of rows or
block of a reduction takes in what lies behind a segment's live rows, and those become zero."""
import random

import pytest
import torch

from test_gpu_grouped import check

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sonicmoe():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import sonicmoe as m
    yield m
    torch.cuda.synchronize()
    m.ops.check_status("cuda")


def layout(E, lo, hi, gap, seed):
    r = random.Random(seed)
    counts = [r.randint(lo, hi) for _ in range(E)]
    gaps = [r.choice((0, 1, r.randint(2, gap))) for _ in range(E)]
    if (sum(counts) + sum(gaps) + 5 + 33) % 128 == 0:      # (a multiple of 128 stands for padded segments)
        gaps[0] += 1
    return counts, dict(gaps=gaps, first=5, tail=33)


def for_many_rows(rows, E, *columns):
    """Above an eighth over 128 rows an expert, and with more tiles of 64 x 128 than two an SM of 148, columns of either product."""
    assert rows > 144 * E and all(rows // 64 * -(-c // 128) > 2 * 148 for c in columns)


@pytest.mark.parametrize("E,lo,hi,gap,N,K", [(20, 130, 320, 70, 1032, 520), (8, 512, 900, 300, 1032, 520), (40, 0, 500, 40, 264, 648),
                                             (3, 3000, 5000, 700, 264, 520), (64, 256, 420, 9, 128, 72), (2, 9000, 13000, 1000, 136, 136)])
@pytest.mark.parametrize("main_grad", [False, True])
def test_gaps(sonicmoe, E, lo, hi, gap, N, K, main_grad):
    counts, kw = layout(E, lo, hi, gap, E + N)
    for_many_rows(sum(counts), E, N, K)
    check(sonicmoe, counts, N, K, seed=int(main_grad), main_grad=main_grad, **kw)


def test_every_end_of_a_tile(sonicmoe):
    """Live rows of every remainder of 256 and 64, behind starts of any."""
    counts = [300 + (i * 5) % 257 for i in range(100)]
    gaps = [(i * 7) % 23 for i in range(100)]
    for_many_rows(sum(counts), 100, 136, 72)
    check(sonicmoe, counts, 136, 72, gaps=gaps, first=1, tail=1)


@pytest.mark.parametrize("alloc,E", [(80, 64), (96, 30), (136, 64), (144, 30), (200, 20)])
def test_the_kernels_of_few_and_many_rows_agree(sonicmoe, alloc, E):
    """About as many rows an expert as divide the two, with gaps and padded to a multiple of 128 in all."""
    r = random.Random(alloc)
    counts = [r.randint(0, min(alloc, 128)) for _ in range(E)]
    gaps = [alloc - c for c in counts]
    rows = alloc * E
    check(sonicmoe, counts, 1032, 520, gaps=gaps, tail=-rows % 128)
    check(sonicmoe, counts, 1032, 520, gaps=gaps, tail=-rows % 128 + 1)
    full = [alloc] * E
    check(sonicmoe, full, 1032, 520, gaps=[0] * E, tail=-rows % 128 + 1)
