"""Refusals of the products grouped by expert: on the host, before anything is launched."""
import pytest
import torch

import sonicmoe

BF = torch.bfloat16


def t(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


def i32(*v):
    return torch.tensor(v, dtype=torch.int32)


@pytest.mark.parametrize("x,w,efo,counts", [
    (t(4, 16, dtype=torch.float32), t(1, 8, 16), None, None),
    (t(4, 16), t(1, 8, 16, dtype=torch.float32), None, None),
    (t(4, 16), t(8), None, None),
    (t(4, 16), t(1, 1, 8, 16), None, None),
    (t(4, 16), t(1, 8, 24), None, None),
    (t(4, 12), t(1, 8, 12), None, None),
    (t(4, 16), t(1, 12, 16), None, None),
    (t(4, 16), t(1, 0, 16), None, None),
    (t(4, 0), t(1, 8, 0), None, None),
    (t(4, 16), t(2, 8, 16), None, None),
    (t(4, 16), t(1, 8, 16), None, i32(4)),
    (t(4, 16), t(2, 8, 16), i32(0, 4), None),
    (t(4, 16), t(2, 8, 16), i32(0, 2, 4).long(), None),
    (t(4, 16), t(2, 8, 16), i32(0, 2, 4), i32(2)),
    (t(4, 16), t(2, 8, 16), i32(0, 2, 4), i32(2, 2).long()),
    (t(2, 2, 16), t(2, 8, 16), i32(0, 2, 4), None),
    (t(4, 16), t(257, 8, 16), torch.zeros(258, dtype=torch.int32), None),
    (t(4, 16), t(0, 8, 16), i32(0), None),
])
def test_refusals(x, w, efo, counts):
    with pytest.raises(ValueError):
        sonicmoe.grouped_linear(x, w, efo, counts)


def test_there_is_no_cpu_path():
    with pytest.raises(RuntimeError, match="CUDA"):
        sonicmoe.grouped_linear(t(4, 16), t(1, 8, 16))


def test_c_entry_points_check_their_arguments():
    from sonicmoe._lib import lib
    SHAPE, ALIGN, ARG = 1, 2, 6
    rows = lambda **k: lib.smoe_grouped_rows(*({**dict(x=16, ldx=64, w=16, tr=0, efo=16, counts=None, y=16, rows=4, N=8, K=64, E=2, status=16,
                                                       host=None, stream=None), **k}.values()))
    assert rows(N=12) == rows(K=0) == rows(E=0) == rows(E=257) == rows(ldx=56) == rows(ldx=68) == rows(rows=-1) == rows(rows=1 << 30) == SHAPE
    assert rows(efo=None) == rows(status=None) == rows(x=None) == rows(w=None) == rows(y=None) == ARG
    assert rows(E=1, efo=None, counts=16) == ARG
    assert rows(x=8) == rows(w=24) == rows(y=2) == ALIGN
    assert rows(rows=0, x=None, y=None) == 0
    wg = lambda **k: lib.smoe_grouped_wgrad(*({**dict(dy=16, ldy=8, x=16, ldx=64, efo=16, counts=None, dw=16, N=8, K=64, rows=4, E=2, bf16=1, acc=0, ws=None,
                                                      status=16, host=None, stream=None), **k}.values()))
    assert wg(N=4) == wg(ldy=0) == wg(ldx=65) == SHAPE
    assert wg(acc=1) == wg(dw=None) == wg(dy=None) == wg(efo=None) == ARG
    assert wg(dw=8) == wg(dy=2) == wg(x=8) == ALIGN
    assert wg(rows=0, bf16=0, acc=1) == 0
    assert lib.smoe_grouped_wgrad_workspace(8, 64, 4, 2) == 0 and lib.smoe_grouped_wgrad_workspace(8, 60, 4, 2) == -1
