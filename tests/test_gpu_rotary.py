"""rotate (norms of heads and rotary positions) vs 64 bits.

Bound on an element: its own rounding, half a step (finfo.eps / 2 of it), and for the fp32 work 2^-20 of
the two numbers that it is made of: the norm's factor is off by some 2^-22 (a sum of D <= 256 squares in
a tree of fp32 sums, a root and a division), the angle by 2 pi 2^-26 in fp32 turns, sine and cosine by two
steps, three products and a sum by a half each.
"""

import math

import pytest
import torch

from lsa_rocm_lab.port import pipeline

pytestmark = pytest.mark.gpu
DEV = "cuda"


def want(x, pos, freq, weight, eps, interleaved, magnitude=1.0):
    """The row's numbers in fp64 and what its elements are made of."""
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * weight.double()
    n = 0 if freq is None else freq.numel()
    out, made = y.clone(), y.abs()
    if n:
        t = pos.double()[..., None, None] * freq.double()
        a, b = ((slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n)))
        out[..., a] = magnitude * (y[..., a] * t.cos() - y[..., b] * t.sin())
        out[..., b] = magnitude * (y[..., a] * t.sin() + y[..., b] * t.cos())
        made = made.clone()
        made[..., a] = made[..., b] = magnitude * (y[..., a].abs() + y[..., b].abs())
    return out, made


def check(got, ref, made, dtype):
    half = torch.finfo(dtype).eps / 2
    off = (got.double().cpu() - ref).abs()
    bound = half * ref.abs() + 2.0 ** -20 * made + torch.finfo(dtype).tiny
    assert (off <= bound).all(), f"off by {(off / bound).max():.2f} of the bound"


CASES = [
    # dtype, B, T, Hq, Hkv, D, pairs, interleaved, norms, view
    (torch.float32, 1, 1, 1, 1, 32, 16, False, "qk", False),
    (torch.float32, 2, 3, 4, 2, 64, 32, True, "", True),
    (torch.float32, 1, 5, 6, 3, 128, 10, False, "q", False),
    (torch.float32, 3, 7, 2, 1, 256, 128, True, "k", False),
    (torch.bfloat16, 1, 1, 32, 8, 128, 64, False, "qk", True),
    (torch.bfloat16, 2, 613, 5, 5, 128, 64, False, "qk", True),
    (torch.bfloat16, 1, 1025, 3, 1, 64, 16, True, "qk", False),
    (torch.bfloat16, 4, 300, 8, 2, 256, 32, False, "", True),
    (torch.bfloat16, 1, 2000, 8, 1, 32, 1, False, "qk", False),
    (torch.float16, 3, 1, 24, 8, 128, 48, False, "q", False),
    (torch.float16, 1, 1500, 8, 2, 128, 27, False, "qk", True),
    (torch.float16, 2, 9, 71, 1, 64, 31, True, "qk", True),
    (torch.float16, 1, 1200, 2, 2, 256, 0, False, "qk", False),
]


def make(dtype, B, T, Hq, Hkv, D, pairs, interleaved, norms, view, seed=0):
    g = torch.Generator().manual_seed(seed)
    rows = torch.randn(B, T, Hq + 2 * Hkv, D, generator=g).to(dtype)
    q, k = rows[:, :, :Hq], rows[:, :, Hq:Hq + Hkv]
    freq = (10000.0 ** (-torch.arange(pairs, dtype=torch.float64) / max(pairs, 1))) if pairs else None
    pos = torch.randint(0, 1 << 20, (B, T), generator=g)
    w = [torch.rand(D, generator=g).add(0.5).to(dtype) if n in norms else None for n in "qk"]
    return rows, q, k, freq, pos, w


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_rotate(case):
    dtype, B, T, Hq, Hkv, D, pairs, interleaved, norms, view = case
    rows, q, k, freq, pos, (wq, wk) = make(*case)
    dev = rows.to(DEV)
    qd, kd = (dev[:, :, :Hq], dev[:, :, Hq:Hq + Hkv]) if view else (q.to(DEV).contiguous(), k.to(DEV).contiguous())
    for kind in (torch.float32, torch.float64):
        f = None if freq is None else freq.to(kind)
        fd = None if f is None else f.to(DEV)
        at = pos.to(DEV).to(torch.int32 if kind == torch.float32 else torch.int64) if pairs else None
        got = pipeline.rotate(qd, kd, at, fd, *(None if w is None else w.to(DEV) for w in (wq, wk)), interleaved=interleaved,
                              eps=1e-5, magnitude=1.25 if kind == torch.float64 else 1.0)
        for x, w, y in ((q, wq, got[0]), (k, wk, got[1])):
            assert y.is_contiguous() and y.dtype == dtype
            check(y, *want(x, pos, f, w, 1e-5, interleaved, 1.25 if kind == torch.float64 else 1.0), dtype)


def test_far_and_negative_positions_and_one_row_of_them():
    """Positions past 2^31, negative ones, [T] for every batch row, and fp32 weights for bf16 rows."""
    g = torch.Generator().manual_seed(1)
    q = torch.randn(2, 4, 3, 128, generator=g).to(torch.bfloat16)
    freq = pipeline.rotary_frequencies(128, dtype=torch.float64)
    pos = torch.tensor([-5, 0, (1 << 31) + 12345, (1 << 33) + 7])
    w = torch.rand(128, generator=g) + 0.5
    got, none = pipeline.rotate(q.to(DEV), None, pos.to(DEV), freq.to(DEV), q_weight=w.to(DEV))
    assert none is None
    ref, made = want(q, pos.expand(2, 4), freq, w, 1e-6, False)
    half = torch.finfo(torch.bfloat16).eps / 2  # fp64 products of such positions are off by 2^33 2^-53 turns: nothing
    assert ((got.double().cpu() - ref).abs() <= half * ref.abs() + 2.0 ** -20 * made).all()


def test_rows_that_are_not_aligned_or_not_contiguous():
    g = torch.Generator().manual_seed(2)
    flat = torch.randn(2 * 5 * 4 * 64 + 3, generator=g).to(torch.float16)
    q = flat[3:].view(2, 5, 4, 64)  # 6 bytes off
    k = torch.randn(2, 5, 64, 2, generator=g).to(torch.float16).transpose(2, 3)
    freq, pos = pipeline.rotary_frequencies(64), torch.arange(5, dtype=torch.int32)
    fd = flat.to(DEV)
    got = pipeline.rotate(fd[3:].view(2, 5, 4, 64), k.to(DEV), pos.to(DEV), freq.to(DEV))
    for x, y in zip((q, k), got):
        check(y, *want(x, pos.expand(2, 5), freq, None, 0.0, False), torch.float16)


def test_infinities_and_nan_stay_in_their_pairs():
    q = torch.ones(1, 1, 1, 64, dtype=torch.float32)
    q[..., 3], q[..., 60], q[..., 62] = math.inf, math.nan, -math.inf
    freq = pipeline.rotary_frequencies(32).to(DEV)  # dims 0..31, pairs (j, j + 16)
    got = pipeline.rotate(q.to(DEV), None, torch.tensor([2], dtype=torch.int32, device=DEV), freq)[0].cpu().view(-1)
    odd = ~torch.isfinite(got)
    assert odd.nonzero().flatten().tolist() == [3, 19, 60, 62]
    assert got[62] == -math.inf and got[60].isnan()


def test_nothing_to_rotate():
    q = torch.empty(0, 3, 4, 64, device=DEV)
    assert pipeline.rotate(q, None, None, None)[0].shape == q.shape
    q = torch.randn(1, 2, 4, 64, device=DEV)
    assert torch.equal(pipeline.rotate(q, q[:, :, :2], None, None)[1], q[:, :, :2])  # no norm, no rotation


def test_in_a_graph_and_on_another_stream():
    case = (torch.bfloat16, 2, 40, 8, 2, 128, 64, False, "qk", False)
    _, q, k, freq, pos, (wq, wk) = make(*case)
    q, k, freq, pos, wq, wk = (x.to(DEV) for x in (q.contiguous(), k.contiguous(), freq.float(), pos.int(), wq, wk))
    eager = pipeline.rotate(q, k, pos, freq, wq, wk)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        other = pipeline.rotate(q, k, pos, freq, wq, wk)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            held = pipeline.rotate(q, k, pos, freq, wq, wk)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    for i in range(3):
        q.mul_(-1.0)
        graph.replay()
        again = pipeline.rotate(q, k, pos, freq, wq, wk)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, again))
