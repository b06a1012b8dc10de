"""What sd3_layer_norm and sd3_layer_norm_backward refuse, before any CUDA call (no GPU needed)."""
from ctypes import c_void_p

import pytest

from conftest import load_binding

P = c_void_p(4096)  # never read: every call here is refused


def forward(s, x=P, ldx=64, dtype=0, eps=1e-5, y=c_void_p(8192), rows=2, C=64):
    return s.lib().sd3_layer_norm(x, ldx, dtype, None, None, eps, y, None, None, rows, C, None)


def backward(s, dy=P, lddy=64, x=P, ldx=64, dtype=0, mean=P, rstd=P, dx=c_void_p(8192), rows=2, C=64, scratch=P, nbytes=1 << 30):
    return s.lib().sd3_layer_norm_backward(dy, lddy, x, ldx, dtype, None, mean, rstd, dx, None, None, rows, C, scratch, nbytes,
                                           None)


@pytest.mark.parametrize("bad", [dict(dtype=2), dict(rows=-1), dict(C=0), dict(C=1 << 25), dict(ldx=63), dict(ldx=-64), dict(eps=-1.0),
                                 dict(eps=float("nan")), dict(x=None), dict(y=None), dict(y=P, ldx=80)])
def test_forward(bad):
    s = load_binding()
    assert forward(s, **bad) == -1
    assert b"sd3_layer_norm" in s.lib().sd3_last_error()


@pytest.mark.parametrize("bad", [dict(dtype=7), dict(rows=-1), dict(C=0), dict(ldx=63), dict(lddy=1), dict(x=None), dict(dy=None),
                                 dict(mean=None), dict(rstd=None), dict(dx=None), dict(scratch=None), dict(nbytes=8),
                                 dict(scratch=c_void_p(4098)), dict(dx=P, ldx=80), dict(dx=P, lddy=80)])
def test_backward(bad):
    s = load_binding()
    assert backward(s, **bad) == -1
    assert b"sd3_layer_norm_backward" in s.lib().sd3_last_error()


def test_no_rows_need_nothing():
    s = load_binding()
    assert forward(s, x=None, y=None, rows=0) == 0


@pytest.mark.parametrize("dtype,at", [(0, 4098), (1, 4097)])
def test_addresses_inside_an_element(dtype, at):
    s = load_binding()
    for name in ("x", "y"):
        assert forward(s, dtype=dtype, **{name: c_void_p(at)}) == -1
    for name in ("x", "dy", "dx"):
        assert backward(s, dtype=dtype, **{name: c_void_p(at)}) == -1
    for name in ("mean", "rstd"):
        assert backward(s, dtype=dtype, **{name: c_void_p(4098)}) == -1


class Wide:
    """stands for a CUDA tensor of one row that is too long for a 32-bit number"""
    dtype, device, is_cuda, shape = None, "cuda:0", True, (1, 2 ** 32 + 8)

    def dim(self):
        return 2

    def stride(self, d):
        return (2 ** 32 + 8, 1)[d]


def test_rows_too_long_for_an_int():
    s = load_binding()
    with pytest.raises(s.Sd3Error, match="2\\^31"):
        s.layer_norm(Wide())
    with pytest.raises(s.Sd3Error, match="2\\^31"):
        s.layer_norm_backward(Wide(), Wide(), None, None, None)
    with pytest.raises(s.Sd3Error, match="2\\^31"):
        s.linear_residual(Wide(), Wide())


@pytest.mark.gpu
def test_rows_too_long_for_an_int_in_the_extension(sd3):
    import os
    import sys
    import torch
    sys.path.insert(0, os.path.dirname(sd3.LIB_PATH))
    import custom_modules as F
    x, w = torch.empty(1, 2 ** 32 + 8, device="cuda", dtype=torch.bfloat16), torch.empty(8, device="cuda")
    with pytest.raises(RuntimeError, match="2\\^31"):
        F.layer_norm(x, w, w, 1e-5, True)
    with pytest.raises(RuntimeError, match="2\\^31"):
        F.layer_norm_backward(x, x, w, w, w)
    with pytest.raises(RuntimeError, match="2\\^31"):
        F.linear_residual(x, x)
