"""linear_residual: act(x w^T + bias) + residual against the same in 64 bits.

Tolerances.  Products of bf16 values are exact in fp32; a sum of K of them is off by at most K steps of the tensor core's
accumulation, 2^-23 each, of the sum of absolute products, which is sqrt(K) times smaller for the random signs here: 2^-23 *
(16 + sqrt(K)) * sum |x w| covers it.  Activations have slopes of at most 1.13 and their own error of 1e-6 |y| + 2e-7.  One
rounding to bf16: half a step, 2^-8 of the value."""
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
NAMES = ["none", "gelu_tanh", "gelu", "silu", "relu"]


def oracle(x, w, bias, act, residual):
    y = x.double() @ w.double().t()
    if bias is not None:
        y = y + bias.double()
    pre = y
    if act == 1:
        y = 0.5 * y * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (y + 0.044715 * y ** 3)))
    elif act == 2:
        y = 0.5 * y * torch.special.erfc(-y * 0.5 ** 0.5)
    elif act == 3:
        y = y * torch.sigmoid(y)
    elif act == 4:
        y = y.clamp(min=0)
    return (y + residual.double() if residual is not None else y), pre


def check(sd3, M, N, K, act=0, with_bias=True, with_residual=True, dtype=torch.bfloat16, pads=(0, 0, 0, 0), seed=0, inplace=False):
    g = torch.Generator(device="cuda").manual_seed(seed + 7 * M + N + K)

    def rows(m, n, pad, dt, scale=1.0):
        t = torch.full((m, n + pad), float("nan"), device="cuda", dtype=dt)
        t[:, :n] = torch.randn(m, n, device="cuda", generator=g) * scale
        return t[:, :n]

    x, w = rows(M, K, pads[0], torch.bfloat16), rows(N, K, pads[1], torch.bfloat16, K ** -0.5)
    bias = torch.randn(N, device="cuda", generator=g) if with_bias else None
    residual = rows(M, N, pads[2], dtype) if with_residual else None
    want, pre = oracle(x, w, bias, act, residual)
    wide = torch.full((M, N + pads[3]), 17.0, device="cuda", dtype=dtype)
    out = residual if inplace else wide[:, :N]
    got = sd3.linear_residual(x, w, bias, act, residual, out=out)
    assert got.data_ptr() == out.data_ptr()
    torch.cuda.synchronize()
    sd3.assert_healthy()
    # accumulation, bias and residual additions (one step each of the larger operand), the activation's own error
    terms = x.double().abs() @ w.double().abs().t()
    tol = 2.0 ** -23 * (16 + K ** 0.5) * terms * 1.13 + 1e-6 * pre.abs() + 2e-7 + 2.0 ** -23 * (want.abs() + pre.abs())
    off = (got.double() - want).abs() - tol - (2.0 ** -8 * want.abs() if dtype == torch.bfloat16 else 0)
    assert torch.isfinite(got).all() and (off <= 0).all(), "off by %g" % off.max().item()
    if pads[3] and not inplace:
        assert (wide[:, N:] == 17).all()  # what lies between the rows stays as it was
    if not inplace:
        again = torch.empty_like(wide)[:, :N]  # the same bits again
        assert torch.equal(sd3.linear_residual(x, w, bias, act, residual, out=again), got)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N,K", [(1, 1, 8), (1, 6144, 1536), (2, 64, 64), (5, 100, 40), (8, 333, 136), (77, 1536, 6144), (127, 129, 1032),
                                   (128, 128, 512), (154, 1536, 768), (255, 1000, 72), (300, 5, 2048), (129, 1001, 1544)])
def test_few_rows_and_odd_widths(sd3, M, N, K, dtype):
    check(sd3, M, N, K, act=(M + N) % 5, dtype=dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N,K", [(256, 256, 64), (257, 256, 128), (333, 1536, 1536), (1000, 136, 200), (4429, 1544, 512),
                                   (2048, 4608, 1536), (300, 1537, 768), (1111, 999, 1000), (8192, 64, 64), (700, 130, 64)])
def test_many_rows(sd3, M, N, K, dtype):
    check(sd3, M, N, K, act=(M + K // 8) % 5, dtype=dtype)


@pytest.mark.parametrize("act", range(5))
@pytest.mark.parametrize("M,N", [(20, 264), (600, 512)])
@pytest.mark.parametrize("with_bias,with_residual", [(True, True), (False, False), (True, False), (False, True)])
def test_parts(sd3, act, M, N, with_bias, with_residual):
    check(sd3, M, N, 192, act, with_bias, with_residual, torch.float32)
    check(sd3, M, N, 192, act, with_bias, with_residual, torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N,K,pads", [(50, 300, 64, (8, 16, 4, 12)), (50, 300, 64, (8, 16, 1, 3)), (600, 512, 256, (8, 64, 8, 24)),
                                        (600, 512, 256, (0, 0, 3, 8)), (600, 512, 256, (0, 0, 8, 5)), (40, 80, 61, (3, 11, 0, 0)),
                                        (500, 200, 61, (3, 11, 0, 0))])
def test_rows_with_a_stride(sd3, M, N, K, pads, dtype):
    check(sd3, M, N, K, 1, dtype=dtype, pads=pads)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N", [(3, 100), (129, 130), (700, 768), (4429, 256)])
def test_onto_the_residual(sd3, M, N, dtype):
    check(sd3, M, N, 320, 3, dtype=dtype, inplace=True)


def test_activations_far_from_zero(sd3):
    """Values from -200 to 200 through every activation: no overflow, zeros and identities where they belong."""
    v = torch.linspace(-200, 200, 401, device="cuda").bfloat16()
    x = torch.zeros(401, 64, device="cuda", dtype=torch.bfloat16)
    x[:, 0] = v
    w = torch.zeros(72, 64, device="cuda", dtype=torch.bfloat16)
    w[:, 0] = 1
    for rows in (100, 401):
        for act in range(5):
            got = sd3.linear_residual(x[:rows], w, None, act, out_dtype=torch.float32)
            want, pre = oracle(x[:rows], w, None, act, None)
            assert ((got.double() - want).abs() <= 1e-6 * pre.abs() + 2e-7).all(), act


def test_not_a_number_stays_in_its_row(sd3):
    for M in (100, 600):
        x, w = torch.randn(M, 128, device="cuda").bfloat16(), torch.randn(256, 128, device="cuda").bfloat16()
        clean = sd3.linear_residual(x, w, act=sd3.ACT_RELU)
        x[70, 3] = float("nan")
        got = sd3.linear_residual(x, w, act=sd3.ACT_RELU)
        assert got[70].isnan().all() and torch.equal(got[:70], clean[:70]) and torch.equal(got[71:], clean[71:])


def test_no_rows(sd3):
    x, w = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16), torch.ones(8, 64, device="cuda", dtype=torch.bfloat16)
    assert sd3.linear_residual(x, w).shape == (0, 8)


def test_captured_and_on_another_stream(sd3):
    for M in (4, 512):
        x, w = torch.randn(M, 256, device="cuda").bfloat16(), torch.randn(320, 256, device="cuda").bfloat16()
        r = torch.randn(M, 320, device="cuda")
        want = sd3.linear_residual(x, w, None, 2, r)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = sd3.linear_residual(x, w, None, 2, r)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = sd3.linear_residual(x, w, None, 2, r)
        x.mul_(-0.5)
        graph.replay()
        assert torch.equal(got, sd3.linear_residual(x, w, None, 2, r))


def test_extension(sd3):
    sys.path.insert(0, os.path.dirname(sd3.LIB_PATH))
    import custom_modules as F
    x, w = torch.randn(2, 30, 192, device="cuda").bfloat16(), torch.randn(100, 192, device="cuda").bfloat16()
    bias, r = torch.randn(100, device="cuda"), torch.randn(2, 30, 100, device="cuda")
    for act, name in enumerate(NAMES):
        want = sd3.linear_residual(x.view(60, 192), w, bias, act, r.view(60, 100))
        got = F.linear_residual(x, w, bias, r, name)
        assert got.shape == r.shape and got.dtype == torch.float32 and torch.equal(got.view(60, 100), want)
    assert F.linear_residual(x, w).dtype == torch.bfloat16
    stream = r.clone()
    assert F.linear_residual(x, w, bias, stream, "silu", out=stream) is stream
    assert torch.equal(stream, F.linear_residual(x, w, bias, r, "silu"))
    for bad in (dict(activation="tanh"), dict(dtype=torch.float16), dict(residual=r[:1]), dict(residual=r.bfloat16(), dtype=torch.float32),
                dict(bias=bias[:50]), dict(w=w.float()), dict(w=w[:, :96]), dict(x=x.cpu()), dict(out=r[:, :, :50])):
        with pytest.raises(RuntimeError):
            F.linear_residual(**dict(dict(x=x, w=w), **bad))
    with pytest.raises(RuntimeError, match="16-byte aligned"):
        F.linear_residual(x[..., :61].contiguous(), w[:, :61].contiguous())
