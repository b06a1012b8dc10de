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
