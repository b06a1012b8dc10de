"""Timed cases of the operators of a transformer layer over packed prompts: attention over packed sequences, the matrix
product with bias, activation and residual in its epilogue, and layer norm with its gradient.

`run` computes them with elementary torch operations in 32 bits, or, with `own` set, through this repository's extension.
"""
import math
import os
import sys

import torch

own = False

EPS = 1e-5
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"bf16": 2, "f32": 4, "none": 0}
MAX_TOKENS = 8192  # of a drawn attention
MAX_LINEAR = 16384 * 6144 * 1536  # products of a drawn linear
MAX_NORM = 32768 * 1536  # elements of a drawn layer norm


def _extension():
    here = os.path.join(os.getcwd(), "sd3.c_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    import custom_modules
    return custom_modules


def _attention(name, lengths, heads, kv_heads, dim, causal):
    return {"name": name, "op": "attention", "lengths": lengths, "heads": heads, "kv_heads": kv_heads, "dim": dim, "causal": causal}


def _linear(name, M, N, K, act, residual, out):
    return {"name": name, "op": "linear", "M": M, "N": N, "K": K, "act": act, "residual": residual, "out": out}


def _norm(name, op, rows, width, dtype):
    return {"name": name, "op": op, "rows": rows, "width": width, "dtype": dtype}


def listed():
    return [
        # a prompt and its negative prompt, padded to the usual 77 tokens, in a text encoder of width 768
        _attention("attention prompt pair", "77,77", 12, 12, 64, True),
        # a serving batch of captions of different lengths, every token sees its whole caption, 24 heads of 64
        _attention("attention captions", "333,77,12,256,154,1,333,40,77,201,19,333,128,64,300,90", 24, 24, 64, False),
        # prompts from one token to a few thousand before a language model's first answer, grouped heads
        _attention("attention ragged grouped", "1,2048,77,1023,333,129,64,640", 32, 8, 128, True),
        # one long document
        _attention("attention long grouped", "8192", 32, 8, 128, True),
        # one token through the first half of an MLP: the weights are all there is to read
        _linear("linear one token", 1, 6144, 1536, "gelu_tanh", "none", "bf16"),
        # odd widths: an adapter between two encoders, onto a 32-bit stream
        _linear("linear odd", 333, 1001, 1544, "silu", "f32", "f32"),
        # sixteen thousand rows through the first half of an MLP, and through the second half onto the 32-bit stream
        _linear("linear rows up", 16384, 6144, 1536, "gelu", "none", "bf16"),
        _linear("linear rows down", 16384, 1536, 6144, "none", "f32", "f32"),
        # layer norm of the prompts' rows, and of eight images' rows in 32 bits
        _norm("norm prompt pair", "norm", 154, 1536, "bf16"),
        _norm("norm rows f32", "norm", 32768, 1536, "f32"),
        # its gradient: a small odd width, and eight images' rows
        _norm("norm gradient odd", "norm_gradient", 1357, 777, "f32"),
        _norm("norm gradient rows", "norm_gradient", 32768, 1536, "bf16"),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(["attention", "linear", "norm", "norm_gradient"])
    if op == "attention":
        dim, kv = rng.choice([64, 128]), rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([g for g in (1, 2, 3, 4, 8) if g * kv <= 32])
        total, lengths = _log(rng, 16, MAX_TOKENS), []
        for _ in range(rng.randint(1, 24)):
            if total > 0:
                lengths.append(_log(rng, 1, total))
                total -= lengths[-1]
        rng.shuffle(lengths)
        return {k: v for k, v in _attention("", ",".join(map(str, lengths)), heads, kv, dim, rng.random() < 0.7).items() if k != "name"}
    if op == "linear":
        N, K = _log(rng, 64, 6144), 8 * _log(rng, 8, 768)
        if rng.random() < 0.6:
            N = max(64, N // 64 * 64)
        M = _log(rng, 1, min(16384, MAX_LINEAR // (N * K)))
        out = rng.choice(["bf16", "f32"])
        act = rng.choice(["none", "gelu_tanh", "gelu", "silu", "relu"])
        return {k: v for k, v in _linear("", M, N, K, act, rng.choice(["none", out]), out).items() if k != "name"}
    width = _log(rng, 64, 8192)
    if rng.random() < 0.6:
        width = max(64, width // 64 * 64)
    rows = _log(rng, 1, min(32768, MAX_NORM // width))
    return {k: v for k, v in _norm("", op, rows, width, rng.choice(["bf16", "f32"])).items() if k != "name"}


def _lengths(case):
    return [int(n) for n in case["lengths"].split(",")]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    s = {"case": case}
    if case["op"] == "attention":
        lengths, total = _lengths(case), sum(_lengths(case))
        hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
        # what a projection leaves: the q, k and v of a token next to each other in one row
        qkv = normal(total, hq + 2 * hk, d, dtype=torch.bfloat16)
        s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
        offsets = [0]
        for n in lengths:
            offsets.append(offsets[-1] + n)
        s["offsets"] = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    elif case["op"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        s["x"] = normal(M, K, dtype=torch.bfloat16)
        s["w"] = normal(N, K, dtype=torch.bfloat16, scale=K ** -0.5)
        s["bias"] = normal(N, scale=0.1)
        s["residual"] = None if case["residual"] == "none" else normal(M, N, dtype=TYPES[case["residual"]])
    else:
        rows, width, dt = case["rows"], case["width"], TYPES[case["dtype"]]
        # rows of different means and sizes, as a residual stream has them
        x = normal(rows, width) * (0.5 + normal(rows, 1).abs()) + normal(rows, 1, scale=0.5)
        s["x"] = x.to(dt)
        s["w"], s["b"] = 1.0 + normal(width, scale=0.1), normal(width, scale=0.1)
        if case["op"] == "norm_gradient":
            s["dy"] = normal(rows, width, dtype=dt)
            wide = s["x"].double()  # the statistics that a forward pass has left
            s["mean"] = wide.mean(1).float()
            s["rstd"] = ((wide - wide.mean(1, keepdim=True)).square().mean(1) + EPS).rsqrt().float()
    return s


def _padded(x, start, count, longest):
    at = (start[:, None] + torch.arange(longest, device=x.device)).clamp(max=x.shape[0] - 1)
    x = x.float()[at]  # (sequences, longest, heads, dim)
    return x * (torch.arange(longest, device=x.device) < count[:, None])[:, :, None, None]


def _attention_plain(s):
    case, lengths = s["case"], _lengths(s["case"])
    q, k, v = s["q"], s["k"], s["v"]
    offsets = s["offsets"].long()
    total, groups = q.shape[0], case["heads"] // case["kv_heads"]
    if len(lengths) * max(lengths) ** 2 <= total ** 2:  # one padded batch entry per sequence
        longest, start, count = max(lengths), offsets[:-1], offsets[1:] - offsets[:-1]
        q, k, v = (_padded(t, start, count, longest) for t in (q, k, v))
        place = torch.arange(longest, device=q.device)
        seen = (place < count[:, None])[:, None, :].expand(-1, longest, -1)
        if case["causal"]:
            seen = seen & (place[None, :] <= place[:, None])
    else:  # one batch entry with a mask of blocks
        q, k, v = (t.float()[None] for t in (q, k, v))
        place = torch.arange(total, device=q.device)
        which = torch.searchsorted(offsets[1:], place, right=True)
        seen = which[:, None] == which[None, :]
        if case["causal"]:
            seen = seen & (place[None, :] <= place[:, None])
        seen = seen[None]
    q = q.unflatten(2, (case["kv_heads"], groups))  # (batch, tokens, kv_heads, groups, dim)
    scores = torch.einsum("bikgd,bjkd->bkgij", q, k) * case["dim"] ** -0.5
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = (scores - top.clamp(min=-1e30)).exp()
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    out = torch.einsum("bkgij,bjkd->bikgd", p, v).flatten(2, 3)
    if out.shape[0] > 1 or out.shape[1] != total:
        out = out[(torch.arange(out.shape[1], device=out.device) < count[:, None])]
    return out.reshape(total, case["heads"], case["dim"]).to(torch.bfloat16)


def _activate(y, act):
    if act == "gelu_tanh":
        return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    if act == "gelu":
        return 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    if act == "silu":
        return y / (1 + torch.exp(-y))
    return y.clamp(min=0) if act == "relu" else y


def _linear_plain(s):
    y = _activate(s["x"].float() @ s["w"].float().t() + s["bias"], s["case"]["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(TYPES[s["case"]["out"]])


def _norm_plain(s):
    x = s["x"].float()
    mean = x.mean(1)
    off = x - mean[:, None]
    rstd = 1 / torch.sqrt((off * off).mean(1) + EPS)
    return [(off * rstd[:, None] * s["w"] + s["b"]).to(s["x"].dtype), mean, rstd]


def _norm_gradient_plain(s):
    dy, rstd = s["dy"].float(), s["rstd"][:, None]
    unit = (s["x"].float() - s["mean"][:, None]) * rstd
    g = dy * s["w"]
    dx = rstd * (g - g.mean(1, keepdim=True) - unit * (g * unit).mean(1, keepdim=True))
    return [dx.to(s["x"].dtype), (dy * unit).sum(0), dy.sum(0)]


def run(state):
    case = state["case"]
    if own:
        F = _extension()
        if case["op"] == "attention":
            return F.mha_packed(state["q"], state["k"], state["v"], state["offsets"], case["causal"])
        if case["op"] == "linear":
            return F.linear_residual(state["x"], state["w"], state["bias"], state["residual"], case["act"], TYPES[case["out"]])
        if case["op"] == "norm":
            return F.layer_norm(state["x"], state["w"], state["b"], EPS, True)
        return F.layer_norm_backward(state["dy"], state["x"], state["w"], state["mean"], state["rstd"])
    plain = {"attention": _attention_plain, "linear": _linear_plain, "norm": _norm_plain, "norm_gradient": _norm_gradient_plain}
    return plain[case["op"]](state)


def work(case):
    if case["op"] == "attention":
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in _lengths(case))
        rows = 2 * case["heads"] + 2 * case["kv_heads"]
        return {"bytes": sum(_lengths(case)) * rows * case["dim"] * 2, "flops": 4 * pairs * case["heads"] * case["dim"]}
    if case["op"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": 2 * (M * K + N * K) + 4 * N + M * N * (BYTES[case["residual"]] + BYTES[case["out"]]), "flops": 2 * M * N * K}
    rows, width, b = case["rows"], case["width"], BYTES[case["dtype"]]
    if case["op"] == "norm":
        return {"bytes": 2 * rows * width * b + 8 * width + 8 * rows, "flops": 8 * rows * width}
    return {"bytes": 3 * rows * width * b + 12 * width + 8 * rows, "flops": 14 * rows * width}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        q, k, v = (s[n].double() for n in "qkv")
        out, begin = torch.zeros_like(q), 0
        for n in _lengths(case):
            here = slice(begin, begin + n)
            for h in range(case["heads"]):
                j = h * case["kv_heads"] // case["heads"]
                a = (q[here, h] @ k[here, j].t()) / math.sqrt(case["dim"])
                if case["causal"]:
                    a = a.masked_fill(torch.ones(n, n, dtype=torch.bool, device=a.device).triu(1), -math.inf)
                out[here, h] = torch.exp(a - torch.logsumexp(a, 1, keepdim=True)) @ v[here, j]
            begin += n
        return out
    if case["op"] == "linear":
        y = torch.addmm(s["bias"].double(), s["x"].double(), s["w"].double().t())
        act = case["act"]
        if act == "gelu_tanh":
            y = y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y))
        elif act == "gelu":
            y = y * 0.5 * torch.special.erfc(-y / math.sqrt(2))
        elif act == "silu":
            y = y * torch.sigmoid(y)
        elif act == "relu":
            y = torch.where(y > 0, y, torch.zeros_like(y))
        return y if s["residual"] is None else s["residual"].double() + y
    x, w = s["x"].double(), s["w"].double()
    if case["op"] == "norm":
        var, mean = torch.var_mean(x, 1, correction=0)
        r = torch.rsqrt(var + EPS)
        return [torch.addcmul(s["b"].double(), (x - mean[:, None]) * r[:, None], w), mean, r]
    # the derivatives of sum(dy * y) with the mean and the reciprocal deviation as functions of x
    dy, r = s["dy"].double(), s["rstd"].double()
    unit = (x - s["mean"].double()[:, None]) * r[:, None]
    along = torch.einsum("ij,ij,j->i", dy, unit, w) / case["width"]
    level = torch.einsum("ij,j->i", dy, w) / case["width"]
    dx = (dy * w - level[:, None] - unit * along[:, None]) * r[:, None]
    return [dx, torch.einsum("ij,ij->j", dy, unit), dy.sum(0)]
