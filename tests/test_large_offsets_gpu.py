"""The operators of a layer over packed prompts on tensors of more than 2^31 elements: the last rows against a call on them alone
(the same rows of smaller tensors, which the other tests compare with 64 bits)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def fill(t):
    """cheap values that repeat every 1009 elements, which no power of two divides"""
    flat, period = t.view(-1), torch.linspace(-2, 2, 1009, device="cuda").to(t.dtype)
    whole = flat.numel() // 1009 * 1009
    flat[:whole].view(-1, 1009).copy_(period.expand(whole // 1009, 1009))
    flat[whole:].copy_(period[:flat.numel() - whole])
    return t


@pytest.mark.parametrize("N", [32768, 32767])
def test_linear(sd3, N):
    M, K = 66000, 64
    g = torch.Generator(device="cuda").manual_seed(0)
    x, w = (torch.randn(n, K, device="cuda", generator=g).bfloat16() for n in (M, N))
    r = fill(torch.empty(M, N, device="cuda", dtype=torch.bfloat16))
    out = sd3.linear_residual(x, w, None, sd3.ACT_RELU, r)
    tail = M - 300
    want = (x[tail:].float() @ w.float().T).relu() + r[tail:].float()
    off = (out[tail:].float() - want).abs() - 2.0 ** -8 * want.abs() - 1e-4  # fp32 sums of 64 products below 20: 64 * 2^-24 * 20
    assert (off <= 0).all()
    sd3.assert_healthy()


@pytest.mark.parametrize("C", [1536, 1538, 1537])
def test_layer_norm(sd3, C):
    rows = 2 ** 31 // C + 1000
    x = fill(torch.empty(rows, C, device="cuda"))
    dy = x.roll(1, 1)
    w = torch.linspace(0.5, 1.5, C, device="cuda")
    y, mean, rstd = sd3.layer_norm(x, w)
    dx, dw, db = sd3.layer_norm_backward(dy, x, w, mean, rstd)
    tail = rows - 500
    xs, ds = x[tail:].double(), dy[tail:].double()
    u = (xs - xs.mean(1, keepdim=True)) * (xs.var(1, unbiased=False, keepdim=True) + 1e-5).rsqrt()
    gr = ds * w.double()
    want = (xs.var(1, unbiased=False, keepdim=True) + 1e-5).rsqrt() * (gr - gr.mean(1, keepdim=True) - u * (gr * u).mean(1, keepdim=True))
    # values below 2, statistics off by less than 40 half steps: some products of them stay below 2e-5
    assert (y[tail:].double() - u * w.double()).abs().max() < 2e-5 and (dx[tail:].double() - want).abs().max() < 2e-5
    assert torch.isfinite(dw).all() and torch.isfinite(db).all()
    sd3.assert_healthy()


@pytest.mark.parametrize("D", [64, 128])
def test_attention(sd3, D):
    heads, kv_heads, n, count = 4096 // D, 1, 1000, 530
    T = n * count
    q = fill(torch.empty(T, heads, D, device="cuda", dtype=torch.bfloat16))
    k = fill(torch.empty(T, kv_heads, D, device="cuda", dtype=torch.bfloat16))
    v = fill(torch.empty(T, kv_heads, D, device="cuda", dtype=torch.bfloat16))
    o = torch.arange(count + 1, device="cuda", dtype=torch.int32) * n
    got = sd3.attention_packed(q, k, v, o, True)
    a, b, c = (t[T - n:].contiguous() for t in (q, k, v))
    one = torch.tensor([0, n], device="cuda", dtype=torch.int32)
    want = sd3.attention_packed(a, b, c, one, True).float()
    # the two calls may take different variants: each is off by half a step of P and of the output, of values below 2
    assert (got[T - n:].float() - want).abs().max() <= 2 * 2 * (2.0 ** -8 + 8.5e-4 + 2.0 ** -8)
    sd3.assert_healthy()
