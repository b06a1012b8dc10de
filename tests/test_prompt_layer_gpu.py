"""The operators together: a pre-norm transformer layer over a packed batch of prompts, as a text encoder runs it, through the
extension, eagerly and as one captured graph, against the same layer in 64 bits; and the gradient of its last norm in a chain.

Tolerance: every operator rounds its bf16 output once (2^-8 of a value), eight of them on the way through both sublayers, each
carried on by maps of norm about one; 2-norm errors of roundings add up in squares: sqrt(8) * 2^-9 (uniform rounding errors are
1 / sqrt(3) of the largest) < 0.006 of the residual branch."""
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu


def reference(x, p, lengths, heads, kv_heads, D, causal):
    def norm(x, w, b):
        return torch.nn.functional.layer_norm(x, x.shape[-1:], w, b, 1e-5)

    x = x.double()
    p = {k: v.double() for k, v in p.items()}
    h = norm(x, p["w1"], p["b1"]) @ p["qkv"].t() + p["qkv_b"]
    qkv = h.view(x.shape[0], heads + 2 * kv_heads, D)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
    out, begin = torch.zeros_like(q), 0
    for n in lengths:
        a, b, c = (t[begin:begin + n].transpose(0, 1) for t in (q, k, v))
        b, c = b.repeat_interleave(heads // kv_heads, 0), c.repeat_interleave(heads // kv_heads, 0)
        s = a @ b.transpose(1, 2) * D ** -0.5
        if causal:
            s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=s.device).triu(1), float("-inf"))
        out[begin:begin + n] = (s.softmax(-1) @ c).transpose(0, 1)
        begin += n
    x1 = x + out.reshape(x.shape[0], heads * D) @ p["out"].t() + p["out_b"]
    m = torch.nn.functional.gelu(norm(x1, p["w2"], p["b2"]) @ p["up"].t() + p["up_b"])
    return x1 + m @ p["down"].t() + p["down_b"], x1


def layer(F, x, p, offsets, heads, kv_heads, D, causal):
    """x (tokens, E) float32, updated in place: the residual stream"""
    T = x.shape[0]
    h = F.layer_norm(x, p["w1"], p["b1"], 1e-5, True)[0].bfloat16()
    qkv = F.linear_residual(h, p["qkv"], p["qkv_b"]).view(T, heads + 2 * kv_heads, D)
    o = F.mha_packed(qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:], offsets, causal)
    F.linear_residual(o.view(T, heads * D), p["out"], p["out_b"], x, out=x)
    h = F.layer_norm(x, p["w2"], p["b2"], 1e-5, True)[0].bfloat16()
    m = F.linear_residual(h, p["up"], p["up_b"], None, "gelu")
    return F.linear_residual(m, p["down"], p["down_b"], x, out=x)


def params(E, heads, kv_heads, D, hidden):
    g = torch.Generator(device="cuda").manual_seed(1)

    def mat(n, k):
        return (torch.randn(n, k, device="cuda", generator=g) * k ** -0.5).bfloat16()

    def vec(n, scale=0.1, at=0.0):
        return at + scale * torch.randn(n, device="cuda", generator=g)

    N = (heads + 2 * kv_heads) * D
    return dict(w1=vec(E, at=1.0), b1=vec(E), w2=vec(E, at=1.0), b2=vec(E), qkv=mat(N, E), qkv_b=vec(N), out=mat(E, heads * D), out_b=vec(E),
                up=mat(hidden, E), up_b=vec(hidden), down=mat(E, hidden), down_b=vec(E))


@pytest.mark.parametrize("E,heads,kv_heads,D,causal,lengths", [(768, 12, 12, 64, True, [77, 77]), (512, 8, 2, 128, True, [300, 1, 600, 64]),
                                                               (256, 4, 4, 64, False, [12, 333, 1, 0, 150])])
def test_layer(sd3, E, heads, kv_heads, D, causal, lengths):
    sys.path.insert(0, os.path.dirname(sd3.LIB_PATH))
    import custom_modules as F
    T = sum(lengths)
    o = [0]
    for n in lengths:
        o.append(o[-1] + n)
    offsets = torch.tensor(o, dtype=torch.int32, device="cuda")
    p = params(E, heads, kv_heads, D, 4 * E)
    x = torch.randn(T, E, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    want, _ = reference(x, p, lengths, heads, kv_heads, D, causal)
    got = layer(F, x.clone(), p, offsets, heads, kv_heads, D, causal)
    torch.cuda.synchronize()
    sd3.assert_healthy()
    added = want - x.double()
    assert (got.double() - want).norm() <= 0.006 * added.norm()
    # the same bits as one graph, on a stream of its own
    static = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer(F, static, p, offsets, heads, kv_heads, D, causal)
    static.copy_(x)
    graph.replay()
    assert torch.equal(static, got)


def test_gradient_of_a_norm_in_a_chain(sd3):
    """loss = sum(c * (gelu-free linear of layer_norm(x))): the gradient through the norm against autograd in 64 bits."""
    sys.path.insert(0, os.path.dirname(sd3.LIB_PATH))
    import custom_modules as F
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(200, 320, device="cuda", generator=g)
    w, b = 1 + 0.1 * torch.randn(320, device="cuda", generator=g), 0.1 * torch.randn(320, device="cuda", generator=g)
    m = torch.randn(64, 320, device="cuda", generator=g) * 320 ** -0.5
    c = torch.randn(200, 64, device="cuda", generator=g)
    X, W, B = (t.double().requires_grad_() for t in (x, w, b))
    (torch.nn.functional.layer_norm(X, (320,), W, B, 1e-5) @ m.double().t() * c.double()).sum().backward()
    y, mean, rstd = F.layer_norm(x, w, b, 1e-5, True)
    dx, dw, db = F.layer_norm_backward(c @ m, x, w, mean, rstd)
    # fp32 throughout: a few hundred half steps of 2^-24 of the largest values
    for got, want in ((dx, X.grad), (dw, W.grad), (db, B.grad)):
        assert (got.double() - want).abs().max() <= 2e-5 * want.abs().max()


def test_two_streams_at_once(sd3):
    """Each operator in small and large sizes (clusters that share K, CTA pairs, two heads a CTA) in two streams that run at the same
    time, in opposite orders: the same bits as alone."""
    g = torch.Generator(device="cuda").manual_seed(11)

    def normal(*shape, dtype=torch.bfloat16):
        return torch.randn(*shape, device="cuda", generator=g).to(dtype)

    calls = []
    for M, N, K, out in ((1, 1536, 6144, torch.bfloat16), (64, 512, 1536, torch.float32), (300, 1001, 520, torch.float32),
                         (2000, 1536, 768, torch.float32), (1500, 1000, 1024, torch.bfloat16), (40, 64, 4096, torch.float32)):
        x, w, r = normal(M, K), normal(N, K), normal(M, N, dtype=out)
        calls.append(lambda x=x, w=w, r=r: sd3.linear_residual(x, w, None, sd3.ACT_SILU, r))
    for heads, kv, D, lengths in ((12, 12, 64, [77, 77]), (8, 2, 128, [1500]), (4, 4, 128, [3, 200, 64])):
        q, k, v = normal(sum(lengths), heads, D), normal(sum(lengths), kv, D), normal(sum(lengths), kv, D)
        o = torch.tensor([sum(lengths[:i]) for i in range(len(lengths) + 1)], device="cuda", dtype=torch.int32)
        calls.append(lambda q=q, k=k, v=v, o=o: sd3.attention_packed(q, k, v, o, True))
    for rows, C, dtype in ((5, 777, torch.float32), (1000, 1536, torch.float32), (1000, 777, torch.bfloat16), (400, 4098, torch.float32)):
        x, dy, w = normal(rows, C, dtype=dtype), normal(rows, C, dtype=dtype), normal(C, dtype=torch.float32)
        _, mean, rstd = sd3.layer_norm(x, w)
        calls.append(lambda x=x, dy=dy, w=w, m=mean, r=rstd: torch.cat([t.flatten().float() for t in sd3.layer_norm_backward(dy, x, w, m, r)]))
    want = [c() for c in calls]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(10):
        for i in range(len(calls)):
            for s, order in ((0, i), (1, len(calls) - 1 - i)):
                with torch.cuda.stream(streams[s]):
                    got[s].append((order, calls[order]()))
    torch.cuda.synchronize()
    sd3.assert_healthy()
    for results in got:
        for i, t in results:
            assert torch.equal(t, want[i])
