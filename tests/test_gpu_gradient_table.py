"""The list of gradients as a program that calls the C entry points hands it over."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu


class Gradient(ctypes.Structure):
    _fields_ = [("grad", ctypes.c_void_p), ("out", ctypes.c_void_p), ("numel", ctypes.c_int64), ("grad_f32", ctypes.c_int32),
                ("out_f32", ctypes.c_int32)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_norm_does_not_look_at_outputs(dtype):
    """Whatever stands in their place: the same sums in the same order.  (Of 1 and of three squares of 2^-12 in one f32 sum nothing is left
    of the latter, in f64 they are.)"""
    from sonicmoe._lib import check, lib
    g = torch.zeros(4096, device="cuda", dtype=dtype)
    g[0], g[2:8:2] = 1.0, 2.0 ** -12
    norms, ws = torch.zeros(4, device="cuda"), torch.empty(lib.smoe_gradient_workspace(1), dtype=torch.uint8, device="cuda")
    for i, out in enumerate((None, g.data_ptr(), 3, 0xDEADBEEF1)):
        row = Gradient(g.data_ptr(), out, g.numel(), dtype == torch.float32, 1)
        check(lib.smoe_gradient_norm(ctypes.addressof(row), 1, norms[i:].data_ptr(), ws.data_ptr(), torch.cuda.current_stream().cuda_stream),
              "gradient_norm")
    assert len(set(norms.tolist())) == 1
