"""What sd3_attention_packed refuses, before any CUDA call (no GPU needed)."""
from ctypes import c_void_p

import pytest

from conftest import load_binding

Q, K, V, O, N = (c_void_p(1 << n) for n in (12, 16, 20, 24, 28))  # never read: every call here is refused


def call(s, q=Q, ldq=512, k=K, ldk=256, v=V, ldv=256, out=O, ldo=512, offsets=N, count=2, rows=10, heads=8, kv_heads=4, D=64,
         causal=1, scale=0.125):
    return s.lib().sd3_attention_packed(q, ldq, k, ldk, v, ldv, out, ldo, offsets, count, rows, heads, kv_heads, D, causal, scale,
                                        None)


@pytest.mark.parametrize("bad,code", [
    (dict(count=-1), -1), (dict(rows=-1), -1), (dict(heads=0), -1), (dict(kv_heads=0), -1), (dict(kv_heads=3), -1),
    (dict(kv_heads=16), -1), (dict(scale=0.0), -1), (dict(scale=-1.0), -1), (dict(scale=float("nan")), -1),
    (dict(scale=float("inf")), -1), (dict(D=32), -2), (dict(D=96), -2), (dict(D=256), -2), (dict(q=None), -1), (dict(k=None), -1),
    (dict(v=None), -1), (dict(out=None), -1), (dict(offsets=None), -1), (dict(offsets=c_void_p(4098)), -1), (dict(ldq=504), -1),
    (dict(ldk=248), -1), (dict(ldv=128), -1), (dict(ldo=504), -1), (dict(out=Q), -1), (dict(out=K), -1), (dict(out=V), -1),
    (dict(ldq=516), -2), (dict(ldk=260), -2), (dict(ldv=257), -2), (dict(ldo=513), -2), (dict(q=c_void_p(4104)), -2),
    (dict(out=c_void_p((1 << 24) + 2)), -2), (dict(rows=2147483647, count=2147483647, heads=65536, kv_heads=65536, ldq=1 << 23,
                                                   ldk=1 << 23, ldv=1 << 23, ldo=1 << 23), -2)])
def test_refusals(bad, code):
    s = load_binding()
    assert call(s, **bad) == code
    assert b"attention_packed" in s.lib().sd3_last_error()


def test_nothing_needs_nothing():
    s = load_binding()
    assert call(s, q=None, count=0) == 0 and call(s, q=None, rows=0) == 0
