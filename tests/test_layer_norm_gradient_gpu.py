"""Layer norm with weight and bias and its gradient, against the formulas in 64 bits.

Tolerances.  fp32 outputs: the kernel's sums are trees of at most 16 terms a thread, 5 shuffles and 16 warps, so a row's
statistics are off by less than 40 half steps, 40 * 2^-24 = 2.4e-6 of the largest term; 1e-5 of the row's largest value
covers y and dx, which are a few products of them.  dw and db add rows one after the other (at most rows / 148 + 1 of them a
thread) and then up to 148 partial rows: 2^-24 times that many terms, times the largest column sum of absolute values.
bf16 outputs: half a step of bf16, 2^-8 of the value, on top."""
import pytest
import torch

pytestmark = pytest.mark.gpu

EPS = 1e-5


def oracle(x, w, b, dy):
    x = x.double()
    mean = x.mean(1)
    var = (x - mean[:, None]).square().mean(1)
    rstd = (var + EPS).rsqrt()
    u = (x - mean[:, None]) * rstd[:, None]
    g = dy.double() * w.double()
    dx = rstd[:, None] * (g - g.mean(1, keepdim=True) - u * (g * u).mean(1, keepdim=True))
    return u * w.double() + b.double(), mean, rstd, dx, (dy.double() * u).sum(0), dy.double().sum(0), u


def make(rows, C, dtype, seed=0, pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, C + pad, device="cuda", generator=g)[:, :C] * 2 + torch.randn(rows, 1, device="cuda", generator=g)
    dy = torch.randn(rows, C + pad, device="cuda", generator=g)
    wide_x, wide_dy = torch.empty(rows, C + pad, device="cuda", dtype=dtype), dy.to(dtype)
    wide_x.fill_(float("nan"))  # what lies between the rows belongs to nobody
    wide_x[:, :C] = x
    wide_dy[:, C:] = float("nan")
    w = 1 + 0.3 * torch.randn(C, device="cuda", generator=g)
    b = 0.3 * torch.randn(C, device="cuda", generator=g)
    return wide_x[:, :C], w, b, wide_dy[:, :C]


def close(got, want, tol, half):
    """|got - want| <= tol + half |want|, everywhere"""
    off = (got.double() - want).abs() - half * want.abs()
    assert torch.isfinite(got).all()
    assert (off <= tol).all(), "off by %g" % off.max().item()


def check(sd3, x, w, b, dy):
    rows, C = x.shape
    y, mean, rstd = sd3.layer_norm(x, w, b, EPS)
    dx, dw, db = sd3.layer_norm_backward(dy, x, w, mean, rstd)
    torch.cuda.synchronize()
    ry, rmean, rrstd, rdx, rdw, rdb, u = oracle(x, w, b, dy)
    half = 2.0 ** -8 if x.dtype == torch.bfloat16 else 0.0
    assert y.dtype == x.dtype and dx.dtype == x.dtype and dw.dtype == torch.float32
    size = x.double().abs().amax(1)
    assert ((mean.double() - rmean).abs() <= 40 * 2.0 ** -24 * size).all()
    # the variance's relative error: that of the sum of squares, and the mean's error squared
    assert ((rstd.double() / rrstd - 1).abs() <= 1e-5).all()
    close(y, ry, 1e-5 * ry.abs().amax(1, keepdim=True).clamp(min=1) * (1 + (size * rrstd)[:, None]), half)
    scale = rrstd[:, None] * (dy.double().abs() * w.double().abs()).amax(1, keepdim=True) * (1 + u.abs().amax(1, keepdim=True)) ** 2
    close(dx, rdx, 1e-5 * scale, half)
    terms = rows / 148 + 150 + 16
    close(dw, rdw, (terms * 2.0 ** -24 + 1e-5) * (dy.double() * u).abs().sum(0) + 1e-6, 0)
    close(db, rdb, terms * 2.0 ** -24 * dy.double().abs().sum(0) + 1e-30, 0)
    again = sd3.layer_norm_backward(dy, x, w, mean, rstd)
    for p, q in zip((dx, dw, db), again):
        assert torch.equal(p, q)
    sd3.assert_healthy()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,C", [(1, 1), (1, 8), (3, 16), (5, 31), (2, 64), (40, 100), (7, 128), (300, 256), (33, 264), (149, 500),
                                    (1357, 777), (77, 768), (154, 1536), (1000, 1544), (5, 2047), (600, 4096), (9, 5000),
                                    (3, 8192), (2, 8191), (4, 10007), (5, 20000), (70, 9000)])
def test_widths_and_rows(sd3, rows, C, dtype):
    check(sd3, *make(rows, C, dtype, seed=rows + C))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,C,pad", [(50, 1536, 8), (50, 1536, 3), (50, 100, 28), (3, 9000, 5)])
def test_rows_with_a_stride(sd3, rows, C, pad, dtype):
    check(sd3, *make(rows, C, dtype, seed=1, pad=pad))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_addresses_that_are_not_aligned(sd3, dtype):
    x, w, b, dy = make(20, 512, dtype, seed=2)
    shifted = torch.empty(20 * 512 + 1, device="cuda", dtype=dtype)[1:].view(20, 512)
    shifted.copy_(x)
    check(sd3, shifted, w, b, dy)


def carved(t, at, pad):
    """t's rows, `pad` elements apart, `at` elements into a buffer of NaN"""
    rows, C = t.shape
    flat = torch.full((at + rows * (C + pad) + 64,), float("nan"), device="cuda", dtype=t.dtype)
    view = flat[at:at + rows * (C + pad)].view(rows, C + pad)[:, :C]
    view.copy_(t)
    return view


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,C", [(1, 777), (2, 777), (3, 300), (40, 257), (149, 1001), (700, 333), (3, 8191), (400, 2047), (60, 4098)])
@pytest.mark.parametrize("at_x,at_dy,pad", [(0, 0, 0), (1, 3, 0), (6, 0, 1), (7, 2, 2), (5, 5, 9)])
def test_rows_between_other_values(sd3, rows, C, at_x, at_dy, pad, dtype):
    x, w, b, dy = make(rows, C, dtype, seed=rows + C + at_x)
    check(sd3, carved(x, at_x, pad), w, b, carved(dy, at_dy, pad))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("onto", ["x", "dy"])
@pytest.mark.parametrize("rows,C", [(1, 777), (700, 777), (30, 8191), (900, 1024)])
def test_gradient_onto_its_operands(sd3, rows, C, onto, dtype):
    x, w, b, dy = (t.contiguous() for t in make(rows, C, dtype, seed=rows))
    _, mean, rstd = sd3.layer_norm(x, w, b, EPS)
    want = sd3.layer_norm_backward(dy, x, w, mean, rstd)
    dw, db = torch.empty_like(w), torch.empty_like(w)
    nbytes = sd3.lib().sd3_layer_norm_backward_scratch_bytes(rows, C)
    scratch = torch.empty(nbytes, device="cuda", dtype=torch.uint8)
    dx = x if onto == "x" else dy
    sd3.check(sd3.lib().sd3_layer_norm_backward(*(sd3.ptr(dy), C, sd3.ptr(x), C, sd3.dtype_tag(x)), sd3.ptr(w), sd3.ptr(mean),
                                                sd3.ptr(rstd), sd3.ptr(dx), sd3.ptr(dw), sd3.ptr(db), rows, C, sd3.ptr(scratch),
                                                nbytes, sd3.stream_ptr()), "sd3_layer_norm_backward")
    for p, q in zip((dx, dw, db), want):
        assert torch.equal(p, q)


def test_no_rows(sd3):
    x = torch.empty(0, 96, device="cuda")
    y, mean, rstd = sd3.layer_norm(x, None, None)
    assert y.shape == (0, 96) and mean.numel() == 0
    dx, dw, db = sd3.layer_norm_backward(x, x, None, mean, rstd)
    assert dx.shape == (0, 96) and (dw == 0).all() and (db == 0).all()


def test_a_row_of_equal_values_and_values_far_from_zero(sd3):
    x = torch.full((2, 1536), 3.0, device="cuda")
    y, mean, rstd = sd3.layer_norm(x, None, None, EPS)
    assert (y == 0).all() and (mean == 3).all() and torch.allclose(rstd, torch.full_like(rstd, EPS ** -0.5), rtol=1e-6)
    # a mean of 4096 standard deviations: the deviations are formed from x - mean, not from the sum of squares.
    # x is exact to 2^-12 there, the mean off by 40 * 2^-24 * 4096 = 0.01 at most
    x = torch.randn(3, 1536, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5)) + 4096
    y = sd3.layer_norm(x, None, None, EPS)[0]
    ref = torch.nn.functional.layer_norm(x.double(), (1536,), eps=EPS)
    assert (y.double() - ref).abs().max() <= 0.01


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("C", [200, 333, 777, 1024, 1538])
def test_rows_of_one_huge_value(sd3, C, dtype):
    # mean * rstd is no fp32 number, every deviation is 0: u = 0, dx = rstd (g - mean(g)) with rstd = eps^-1/2
    x = torch.full((5, C), 2.0 ** 124, device="cuda", dtype=dtype)
    dy = torch.ones(5, C, device="cuda", dtype=dtype)
    mean = torch.full((5,), 2.0 ** 124, device="cuda")
    rstd = torch.full((5,), EPS ** -0.5, device="cuda")
    w = torch.ones(C, device="cuda")
    dx, dw, db = sd3.layer_norm_backward(dy, x, w, mean, rstd)
    assert dx.float().abs().max() <= C * 2.0 ** -24 * EPS ** -0.5 and (dw == 0).all() and (db == 5).all()


def test_infinities_stay_in_their_row(sd3):
    x = torch.randn(9, 640, device="cuda").bfloat16()
    clean = sd3.layer_norm(x, None, None)[0]
    x[4, 7] = float("inf")
    got = sd3.layer_norm(x, None, None)[0]
    assert torch.equal(got[:4], clean[:4]) and torch.equal(got[5:], clean[5:]) and not torch.isfinite(got[4]).any()


def test_gradient_against_differences(sd3):
    rows, C, h = 3, 40, 1e-3
    x, w, b, dy = make(rows, C, torch.float32, seed=8)
    _, mean, rstd = sd3.layer_norm(x, w, b, EPS)
    dx, dw, db = sd3.layer_norm_backward(dy, x, w, mean, rstd)

    def loss(x, w, b):
        return (oracle(x, w, b, dy)[0] * dy.double()).sum().item()

    for i, j in ((0, 0), (1, 17), (2, 39)):
        e = torch.zeros(rows, C, device="cuda", dtype=torch.float64)
        e[i, j] = h
        # the third derivative of a row's loss is at most a few times rstd^3 |g|, so h^2 / 6 of it stays below 1e-4
        assert abs((loss(x.double() + e, w, b) - loss(x.double() - e, w, b)) / (2 * h) - dx[i, j].item()) < 1e-4
        v = torch.zeros(C, device="cuda", dtype=torch.float64)
        v[j] = h
        assert abs((loss(x, w.double() + v, b) - loss(x, w.double() - v, b)) / (2 * h) - dw[j].item()) < 1e-4
        assert abs((loss(x, w, b.double() + v) - loss(x, w, b.double() - v)) / (2 * h) - db[j].item()) < 1e-4


def test_extension(sd3):
    import os
    import sys
    sys.path.insert(0, os.path.join(os.path.dirname(sd3.LIB_PATH)))
    import custom_modules as F
    x, w, b, dy = make(60, 384, torch.bfloat16, seed=3)
    y, mean, rstd = sd3.layer_norm(x, w, b, EPS)
    got = F.layer_norm(x.view(3, 20, 384), w, b, EPS, True)
    assert got[0].shape == (3, 20, 384) and torch.equal(got[0].view(60, 384), y)
    assert torch.equal(got[1], mean) and torch.equal(got[2], rstd)
    for p, q in zip(F.layer_norm_backward(dy, x, w, mean, rstd), sd3.layer_norm_backward(dy, x, w, mean, rstd)):
        assert torch.equal(p, q)
    # without statistics the call is what it was
    plain = F.layer_norm(x, w, b, EPS, False)
    assert len(plain) == 1 and (plain[0].double() - y.double()).abs().max() <= 2.0 ** -7 * y.double().abs().max()
    with pytest.raises(RuntimeError, match="one shape"):
        F.layer_norm_backward(dy[:30], x, w, mean, rstd)
    with pytest.raises(RuntimeError, match="384 values"):
        F.layer_norm_backward(dy, x, w[:100], mean, rstd)
    with pytest.raises(RuntimeError, match="float32 or bfloat16"):
        F.layer_norm(x.half(), w, b, EPS, True)


def test_library_errors_reach_the_extensions_caller(sd3):
    import os
    import sys
    sys.path.insert(0, os.path.join(os.path.dirname(sd3.LIB_PATH)))
    import custom_modules as F
    x = torch.zeros(4, 12, device="cuda", dtype=torch.bfloat16)  # 24-byte rows: no operand of the tensor cores
    with pytest.raises(RuntimeError, match="sd3_linear failed"):
        F.linear(x, torch.zeros(12, 8, device="cuda", dtype=torch.bfloat16), torch.zeros(8, device="cuda"))


def test_captured_and_on_another_stream(sd3):
    x, w, b, dy = make(500, 1536, torch.bfloat16, seed=4)
    y, mean, rstd = sd3.layer_norm(x, w, b, EPS)
    want = sd3.layer_norm_backward(dy, x, w, mean, rstd)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = sd3.layer_norm_backward(dy, x, w, mean, rstd)
    torch.cuda.current_stream().wait_stream(side)
    for p, q in zip(got, want):
        assert torch.equal(p, q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gy, gm, gr = sd3.layer_norm(x, w, b, EPS)
        got = sd3.layer_norm_backward(dy, x, w, gm, gr)
    x.mul_(1.5)
    dy.add_(0.25)
    graph.replay()
    y, mean, rstd = sd3.layer_norm(x, w, b, EPS)
    for p, q in zip((gy, gm, gr) + got, (y, mean, rstd) + sd3.layer_norm_backward(dy, x, w, mean, rstd)):
        assert torch.equal(p, q)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,C", [(7, 64), (700, 777), (3, 8191), (900, 1024), (5, 20000)])
def test_forward_onto_its_operand(sd3, rows, C, dtype):
    x, w, b, _ = (t.contiguous() for t in make(rows, C, dtype, seed=rows))
    y, mean, rstd = sd3.layer_norm(x, w, b, EPS)
    m, r = torch.empty_like(mean), torch.empty_like(rstd)
    sd3.check(sd3.lib().sd3_layer_norm(sd3.ptr(x), C, sd3.dtype_tag(x), sd3.ptr(w), sd3.ptr(b), EPS, sd3.ptr(x), sd3.ptr(m), sd3.ptr(r),
                                       rows, C, sd3.stream_ptr()), "sd3_layer_norm")
    assert torch.equal(x, y) and torch.equal(m, mean) and torch.equal(r, rstd)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,C", [(40, 96), (700, 778), (300, 777), (2000, 1536), (6, 9001)])
def test_one_row_for_all(sd3, rows, C, dtype):
    x, w, b, dy = make(rows, C, dtype, seed=C)
    check(sd3, x[:1].contiguous().expand(rows, C), w, b, dy)
    check(sd3, x, w, b, dy[:1].contiguous().expand(rows, C))
