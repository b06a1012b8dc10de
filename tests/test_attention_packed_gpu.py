"""Attention over packed sequences against softmax(scale q k^T) v in 64 bits, sequence by sequence.

Tolerances.  The exponentials enter the second product as bf16, each off by half a step, 2^-8 of its value, and one of eight
comes from a cubic that is off by at most 8.5e-4.  Scores and sums are fp32: products of bf16 are exact, and a score of D terms
is off by at most D cut-off steps of 2^-23 of sum |q k| scale, which the exponential turns into a relative error.  The output
is rounded to bf16, half a step, 2^-8 of its value.  So, with P the exact weights,
|got - want| <= (2^-8 + 8.5e-4 + D 2^-23 max sum |q k| scale) sum_j P_j |v_j| + 2^-8 |want|."""
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu


def oracle(q, k, v, lengths, causal, scale):
    """(want, sum_j P_j |v_j|, the scores' error) of the rows of the sequences"""
    out, size = torch.zeros_like(q, dtype=torch.double), torch.zeros_like(q, dtype=torch.double)
    group, begin, worst = q.shape[1] // k.shape[1], 0, 0.0
    for n in lengths:
        if n:
            a, b, c = (t[begin:begin + n].double().transpose(0, 1) for t in (q, k, v))
            b, c = b.repeat_interleave(group, 0), c.repeat_interleave(group, 0)
            s = a @ b.transpose(1, 2) * scale
            worst = max(worst, (a.abs() @ b.abs().transpose(1, 2)).max().item() * scale)
            if causal:
                s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=s.device).triu(1), float("-inf"))
            p = s.softmax(-1)
            out[begin:begin + n] = (p @ c).transpose(0, 1)
            size[begin:begin + n] = (p @ c.abs()).transpose(0, 1)
        begin += n
    return out, size, q.shape[2] * 2.0 ** -23 * worst


def make(T, heads, kv_heads, D, seed=0, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    qkv = torch.randn(T, heads + 2 * kv_heads, D, device="cuda", generator=g).mul_(spread).bfloat16()
    return qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]


def offsets_of(lengths):
    o = [0]
    for n in lengths:
        o.append(o[-1] + n)
    return torch.tensor(o, dtype=torch.int32, device="cuda")


def compare(got, q, k, v, lengths, causal, scale):
    T = sum(lengths)
    want, size, scores = oracle(q, k, v, lengths, causal, scale)
    tol = (2.0 ** -8 + 8.5e-4 + scores) * size[:T] + 2.0 ** -8 * want[:T].abs()
    off = (got[:T].double() - want[:T]).abs() - tol
    assert torch.isfinite(got[:T]).all()
    assert (off <= 0).all(), "off by %g" % off.max().item()


def check(sd3, lengths, heads, kv_heads, D, causal, scale=None, seed=0, spread=1.0, extra=0):
    T = sum(lengths)
    q, k, v = make(T + extra, heads, kv_heads, D, seed, spread)
    out = torch.full((T + extra, heads, D), 7.0, device="cuda", dtype=torch.bfloat16)
    got = sd3.attention_packed(q, k, v, offsets_of(lengths), causal, scale, out)
    torch.cuda.synchronize()
    sd3.assert_healthy()
    compare(got, q, k, v, lengths, causal, scale or D ** -0.5)
    assert (got[T:] == 7).all()  # rows behind the last sequence
    again = sd3.attention_packed(q, k, v, offsets_of(lengths), causal, scale)
    assert torch.equal(again[:T], got[:T])


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lengths", [[1], [2], [77], [127], [128], [129], [255], [256], [257], [400], [1, 1, 1], [0, 5, 0, 0, 130, 0],
                                     [77, 77], [300, 1, 64, 129, 2, 511], [1000], [128, 256, 384]])
def test_lengths(sd3, lengths, D, causal):
    check(sd3, lengths, 4, 2, D, causal, seed=sum(lengths))


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (6, 2), (8, 1), (5, 5), (32, 8)])
@pytest.mark.parametrize("D", [64, 128])
def test_heads(sd3, heads, kv_heads, D):
    check(sd3, [40, 200, 3], heads, kv_heads, D, True, seed=heads)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_long(sd3, D, causal):
    check(sd3, [3000, 5, 1234], 2, 1, D, causal, seed=1)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("extra", [1, 33, 65, 97, 128])
def test_query_tiles_with_few_rows_and_many_keys(sd3, extra, D, causal):
    """Warps without rows, or whose rows see nothing of a key tile, run ahead of the others."""
    for k in (3, 12):
        check(sd3, [128 * k + extra] * 3, 9, 9, D, causal, seed=extra)


@pytest.mark.parametrize("count", [31, 32, 33, 255, 256, 257, 700])
def test_many_sequences(sd3, count):
    g = torch.Generator().manual_seed(count)
    lengths = torch.randint(0, 20, (count,), generator=g).tolist()
    lengths[count // 2] = 300
    check(sd3, lengths, 2, 2, 64, True, seed=count)


@pytest.mark.parametrize("D", [64, 128])
def test_rows_behind_the_last_sequence(sd3, D):
    check(sd3, [50, 130], 2, 2, D, True, extra=200)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths", [[1], [127], [129], [1, 1, 1], [0, 5, 0, 0, 130, 0], [300, 1, 64, 129, 2, 511], [1000]])
@pytest.mark.parametrize("heads,kv_heads,D", [(4, 2, 64), (3, 3, 128), (4, 2, 128), (32, 8, 128)])
def test_short_sequences_in_a_long_buffer(sd3, heads, kv_heads, D, lengths, causal):
    # the variants are chosen by the rows there are, not by the sequences' (the host does not see the offsets)
    check(sd3, lengths, heads, kv_heads, D, causal, seed=sum(lengths), extra=2048 * len(lengths))


@pytest.mark.parametrize("spread,scale", [(8.0, None), (0.01, None), (1.0, 3.0), (3.0, 1e-6)])
@pytest.mark.parametrize("D", [64, 128])
def test_scores_of_all_sizes(sd3, spread, scale, D):
    """Peaked softmaxes (scores in the thousands), flat ones, and running maxima that move."""
    check(sd3, [700, 60], 2, 1, D, True, scale, seed=3, spread=spread)


@pytest.mark.parametrize("D", [64, 128])
def test_a_maximum_that_rises_with_every_key(sd3, D):
    n = 520
    q = torch.ones(n, 1, D, device="cuda", dtype=torch.bfloat16)
    k = (torch.arange(n, device="cuda").float() / 8)[:, None, None].expand(n, 1, D).contiguous().bfloat16()
    v = torch.randn(n, 1, D, device="cuda").bfloat16()
    for causal in (False, True):
        got = sd3.attention_packed(q, k, v, offsets_of([n]), causal)
        compare(got, q, k, v, [n], causal, D ** -0.5)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_other_sequences_reach_nothing(sd3, D, causal):
    """Infinities and NaN in the neighbours' rows and behind the last one change no bit."""
    lengths = [70, 200, 33]
    q, k, v = (t.contiguous() for t in make(sum(lengths) + 40, 2, 1, D, seed=5))
    clean = sd3.attention_packed(q, k, v, offsets_of(lengths), causal)
    for bad in (float("inf"), float("nan"), float("-inf")):
        for t in (q, k, v):
            t[:70] = bad
            t[270:] = bad
        got = sd3.attention_packed(q, k, v, offsets_of(lengths), causal)
        assert torch.equal(got[70:270], clean[70:270])


def test_later_keys_reach_nothing(sd3):
    """A causal row depends on no bit of the rows after it."""
    for D in (64, 128):
        q, k, v = (t.contiguous() for t in make(300, 2, 2, D, seed=6))
        first = sd3.attention_packed(q, k, v, offsets_of([300]), True)
        for t in (q, k, v):
            t[150:] = torch.randn_like(t[150:]) * 50
        got = sd3.attention_packed(q, k, v, offsets_of([300]), True)
        assert torch.equal(got[:150], first[:150])
        k[150:] = float("nan")
        assert torch.equal(sd3.attention_packed(q, k, v, offsets_of([300]), True)[:150], first[:150])


@pytest.mark.parametrize("whole", [False, True])
@pytest.mark.parametrize("at", [0, 1, 63, 64, 127, 128, 200, 298])
@pytest.mark.parametrize("heads,kv_heads,D,extra", [(2, 1, 64, 0), (3, 3, 128, 0), (4, 2, 128, 3000)])
def test_values_of_later_keys_that_are_no_numbers(sd3, heads, kv_heads, D, extra, at, whole):
    lengths = [90, 300]  # extra: rows enough for two heads a CTA
    q, k, v = (t.contiguous() for t in make(390 + extra, heads, kv_heads, D, seed=at))
    want, size, scores = oracle(q, k, v, lengths, True, D ** -0.5)
    bad = v.clone()
    bad[90 + at, :, 3:(D if whole else 4)] = float("nan")
    bad[90 + at + 1, :, 1] = float("-inf")
    got = sd3.attention_packed(q, k, bad, offsets_of(lengths), True)[:390].double()
    torch.cuda.synchronize()
    sd3.assert_healthy()
    nan, inf = torch.zeros_like(got, dtype=torch.bool), torch.zeros_like(got, dtype=torch.bool)
    nan[90 + at:, :, 3:(D if whole else 4)] = True
    inf[90 + at + 1:, :, 1] = True
    assert torch.isnan(got[nan]).all() and (got[inf] == float("-inf")).all()
    ok = ~(nan | inf)
    off = (got - want[:390]).abs() - (2.0 ** -8 + 8.5e-4 + scores) * size[:390] - 2.0 ** -8 * want[:390].abs()
    assert torch.isfinite(got[ok]).all() and (off[ok] <= 0).all()


def test_separate_tensors_and_strides(sd3):
    q, k, v = (t.contiguous() for t in make(200, 4, 2, 64, seed=7))
    want = sd3.attention_packed(q, k, v, offsets_of([200]), True)
    wide = torch.full((200, 6, 64), float("nan"), device="cuda", dtype=torch.bfloat16)
    wide[:, 1:5] = q
    out = torch.zeros(200, 8, 64, device="cuda", dtype=torch.bfloat16)
    got = sd3.attention_packed(wide[:, 1:5], k, v, offsets_of([200]), True, out=out[:, 2:6])
    assert torch.equal(got, want) and (out[:, :2] == 0).all() and (out[:, 6:] == 0).all()


def test_offsets_that_are_no_offsets(sd3):
    """Row numbers outside the tensor are taken as the nearest row, descending ones as empty sequences."""
    q, k, v = make(200, 2, 2, 64, seed=8)
    want = sd3.attention_packed(q, k, v, offsets_of([200]), True)
    bad = torch.tensor([-5, 1 << 30], dtype=torch.int32, device="cuda")
    assert torch.equal(sd3.attention_packed(q, k, v, bad, True), want)
    out = torch.full_like(want, 3.0)
    sd3.attention_packed(q, k, v, torch.tensor([150, 100, 50, -7], dtype=torch.int32, device="cuda"), True, out=out)
    sd3.assert_healthy()
    assert (out == 3).all()


def test_nothing_to_do(sd3):
    q, k, v = make(10, 2, 2, 64)
    out = torch.full((10, 2, 64), 3.0, device="cuda", dtype=torch.bfloat16)
    sd3.attention_packed(q, k, v, offsets_of([]), True, out=out)
    sd3.attention_packed(q, k, v, offsets_of([0, 0]), True, out=out)
    torch.cuda.synchronize()
    assert (out == 3).all()
    assert sd3.attention_packed(q[:0], k[:0], v[:0], offsets_of([0]), True).shape == (0, 2, 64)


def test_captured_with_offsets_that_change(sd3):
    q, k, v = make(400, 4, 2, 128, seed=9)
    offsets = offsets_of([100, 300])
    out = torch.empty(400, 4, 128, device="cuda", dtype=torch.bfloat16)
    sd3.attention_packed(q, k, v, offsets, True, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sd3.attention_packed(q, k, v, offsets, True, out=out)
    for lengths in ([100, 300], [399, 1], [0, 400], [257, 143]):
        offsets.copy_(offsets_of(lengths))
        graph.replay()
        compare(out, q, k, v, lengths, True, 128 ** -0.5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = sd3.attention_packed(q, k, v, offsets, True)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, out)


def test_extension(sd3):
    sys.path.insert(0, os.path.dirname(sd3.LIB_PATH))
    import custom_modules as F
    q, k, v = make(300, 6, 3, 64, seed=10)
    o = offsets_of([120, 180])
    want = sd3.attention_packed(q, k, v, o, True)
    assert torch.equal(F.mha_packed(q, k, v, o, True), want)
    assert torch.equal(F.mha_packed(q, k, v, o, causal=True, scale=0.125), want)
    turned = q.transpose(0, 1).contiguous().transpose(0, 1)  # another memory order
    assert torch.equal(F.mha_packed(turned, k, v, o, True), want)
    out = torch.empty_like(want)
    assert F.mha_packed(q, k, v, o, True, None, out) is out and torch.equal(out, want)
    assert torch.equal(F.mha_packed(q, k, v, o), sd3.attention_packed(q, k, v, o))
    for bad in (dict(q=q.float()), dict(k=k[:100]), dict(k=k[:, :2], v=v[:, :2], q=q[:, :5]), dict(offsets=o.long()), dict(offsets=o.cpu()),
                dict(q=q[:, :, :32], k=k[:, :, :32], v=v[:, :, :32]), dict(scale=-1.0), dict(out=out[:, :3]), dict(q=q.cpu()),
                dict(out=out.transpose(0, 1).contiguous().transpose(0, 1))):
        with pytest.raises(RuntimeError):
            F.mha_packed(**dict(dict(q=q, k=k, v=v, offsets=o), **bad))
