"""key_mass, evict and evict_slots vs 64 bits, and a cache through all of it.

Bound on a mass: its share of the fp32 scores' error (2^-13 of a weight, as in the prefix tests),
2^-24 a sum step, and 2^-45 a weight where many rows add up in integers.
"""

import math

import numpy as np
import pytest
import torch

from lsa_rocm_lab.port import pipeline
from lsa_rocm_lab.port import eviction

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(dtype, B, Tq, Hq, Hkv, D, Tk, W, per_head=False, pool=False, seed=0):
    g = torch.Generator().manual_seed(seed)
    rng = np.random.default_rng(seed)
    q = torch.randn(B, Tq, Hq, D, generator=g).to(dtype)
    k = torch.randn(1 if pool else B, Tk, Hkv, D, generator=g).to(dtype)
    lead = (B, Tq, Hkv) if per_head else (B, Tq)
    n = int(np.prod(lead))
    ids = rng.integers(0, Tk, (n, W)).astype(np.int32)  # some twice
    ids[:, 2::7] = -1
    ids[::5, 0] = Tk + 2
    lens = rng.integers(0, W + 1, n).astype(np.int32)
    lens[::4] = 0
    return q, k, torch.from_numpy(ids.reshape(*lead, W)), torch.from_numpy(lens.reshape(lead))


def want(q, k, ids, lens, scale=None, lse=None):
    B, Tq, Hq, D = q.shape
    C, Tk, Hkv = k.shape[:3]
    G = Hq // Hkv
    scale = D ** -0.5 if scale is None else scale
    mass = torch.zeros(C, Hkv, Tk, dtype=torch.float64)
    for b in range(B):
        for t in range(Tq):
            for g in range(Hkv):
                per = ids.dim() == 4
                at = (ids[b, t, g] if per else ids[b, t])[: int(lens[b, t, g] if per else lens[b, t])].long()
                at = at[(at >= 0) & (at < Tk)]
                if not len(at):
                    continue
                c = b if C == B else 0
                for h in range(g * G, (g + 1) * G):
                    s = scale * (k[c, at, g].double() @ q[b, t, h].double())
                    z = torch.logsumexp(s, 0) if lse is None else lse[b, t, h].double()
                    w = torch.exp(s - z)
                    mass[c, g].index_add_(0, at, w if torch.isfinite(z) else torch.zeros_like(w))
    return mass


def close(got, ref, rows, group, start=0.0):
    off = (got.double().cpu() - ref).abs()
    bound = (2.0 ** -13 + 2.0 ** -23) * ref + 2.0 ** -24 * np.abs(start) + rows * group * 2.0 ** -44
    assert (off <= bound).all(), f"off by {(off / bound).max():.2f} of the bound"


MASS = [
    # dtype, B, Tq, Hq, Hkv, D, Tk, W, per_head, pool
    (torch.float32, 1, 1, 8, 2, 64, 100, 33, True, False),
    (torch.float32, 2, 3, 4, 4, 32, 300, 65, False, False),
    (torch.float32, 2, 1, 8, 1, 128, 70, 40, False, True),
    (torch.float32, 1, 2, 2, 1, 256, 70, 40, False, False),
    (torch.bfloat16, 1, 1, 32, 8, 128, 4000, 2500, True, False),
    (torch.bfloat16, 3, 1, 8, 8, 128, 50, 1, False, False),
    (torch.bfloat16, 5, 1, 4, 2, 128, 600, 257, True, True),
    (torch.bfloat16, 1, 17, 8, 1, 64, 900, 300, False, False),
    (torch.bfloat16, 2, 9, 16, 2, 256, 100, 64, True, False),
    (torch.bfloat16, 4, 1, 8, 2, 32, 1000, 511, False, False),
    (torch.float16, 2, 33, 32, 8, 128, 2000, 400, False, False),
    (torch.float16, 1, 1, 1, 1, 64, 1, 1, False, False),
    (torch.float16, 7, 2, 2, 2, 64, 100000, 20, True, False),
]


@pytest.mark.parametrize("case", MASS, ids=lambda c: "-".join(map(str, c)).replace("torch.", ""))
def test_key_mass(case):
    q, k, ids, lens = make(*case)
    args = [x.to(DEV) for x in (q, k, ids, lens)]
    print("key_mass", case, flush=True)
    got = pipeline.key_mass(*args)
    ref = want(q, k, ids, lens)
    rows, group = case[1] * case[2], case[3] // case[4]
    close(got, ref, rows, group)
    for _ in range(2):  # the same bits every time
        assert torch.equal(pipeline.key_mass(*args), got)
    # into weights that are there, a view of a longer buffer
    C, Hkv, Tk = got.shape
    buf = torch.full((C, Hkv, Tk + 5), 0.25, device=DEV)
    mass = buf[:, :, :Tk]
    assert pipeline.key_mass(*args, mass=mass) is mass
    close(mass, ref + 0.25, rows, group, 0.25)
    assert (buf[:, :, Tk:] == 0.25).all()


@pytest.mark.parametrize("dtype,Tq", [(torch.bfloat16, 1), (torch.bfloat16, 5), (torch.float32, 1)])
def test_key_mass_of_a_wider_softmax(dtype, Tq):
    q, k, ids, lens = make(dtype, 3, Tq, 8, 2, 64, 200, 80, seed=2)
    kp, vp = (torch.randn(1, 150, 2, 64).to(dtype).to(DEV) for _ in range(2))
    args = [x.to(DEV) for x in (q, k, ids, lens)]
    _, lse = pipeline.prefix_read(args[0], kp, vp, args[1], torch.randn_like(args[1]), args[2], args[3], return_lse=True)
    lse[0, 0, 3] = -math.inf
    lse[1, 0, 2] = math.nan
    lse[2, 0, 1] = math.inf
    ref = want(q, k, ids, lens, lse=lse.cpu())
    close(pipeline.key_mass(*args, lse=lse), ref, 3 * Tq, 4)
    assert 0 < float(ref.sum()) < 0.9 * 3 * Tq * 8


def test_rows_whose_sum_is_not_a_number_add_nothing():
    q, k, ids, lens = make(torch.bfloat16, 2, 3, 8, 2, 128, 60, 30, seed=4)
    lens.fill_(30)
    q[0, 1, 5] = math.nan
    k[1, :, 1] = math.inf
    got = pipeline.key_mass(*[x.to(DEV) for x in (q, k, ids, lens)])
    q2, k2 = q.clone(), k.clone()
    ref = want(q2, k2, ids, lens)
    assert torch.isfinite(got).all() and (got[1, 1] == 0).all()
    close(got, ref, 6, 4)


def test_key_mass_in_slabs_of_rows(monkeypatch):
    """More rows than the scores' buffer holds: slabs, the same weights (another order of fp32 sums)."""
    for per_head, pool in ((False, False), (True, True)):
        q, k, ids, lens = make(torch.bfloat16, 2, 23, 8, 2, 64, 300, 70, per_head, pool, seed=6)
        args = [x.to(DEV) for x in (q, k, ids, lens)]
        lse = torch.full((2, 23, 8), 5.0, device=DEV)
        lse[:, 7] = 6.0
        whole, wide = pipeline.key_mass(*args), pipeline.key_mass(*args, lse=lse)
        monkeypatch.setattr(eviction, "_SLAB_BYTES", 4 * 2 * 8 * 70 * 5)
        close(pipeline.key_mass(*args), whole.double().cpu(), 46, 4)
        close(pipeline.key_mass(*args, lse=lse), wide.double().cpu(), 46, 4)
        monkeypatch.undo()


@pytest.mark.parametrize("dtype,Hq,Hkv,D", [(torch.bfloat16, 4, 1, 64), (torch.float16, 8, 1, 128), (torch.float32, 8, 2, 64),
                                            (torch.bfloat16, 2, 2, 32)])
@pytest.mark.parametrize("Tq", [1, 3])
def test_key_mass_of_long_lists(dtype, Hq, Hkv, D, Tq):
    """Lists of many spans: their sums join, and one workgroup adds slots in several steps."""
    q, k, ids, lens = make(dtype, 1, Tq, Hq, Hkv, D, 9000, 7777, seed=43)
    lens[:] = torch.tensor([7777, 3100, 1025])[:Tq]
    args = [x.to(DEV) for x in (q, k, ids, lens)]
    got = pipeline.key_mass(*args)
    close(got, want(q, k, ids, lens), Tq, Hq // Hkv)
    assert torch.equal(pipeline.key_mass(*args), got)


def test_key_mass_of_a_key_that_a_million_softmaxes_list():
    """More of them than a 64-bit sum of 2^-44 holds: every one counts (integers, exact in fp32)."""
    n = 131080
    q = torch.zeros(1, n, 8, 32, dtype=torch.bfloat16, device=DEV)
    k = torch.zeros(1, 5, 1, 32, dtype=torch.bfloat16, device=DEV)
    ids = torch.full((1, n, 1), 3, dtype=torch.int32, device=DEV)
    got = pipeline.key_mass(q, k, ids, torch.ones(1, n, dtype=torch.int32, device=DEV))
    assert got.flatten().tolist() == [0.0, 0.0, 0.0, 8.0 * n, 0.0]


@pytest.mark.parametrize("Tq", [1, 6])
def test_key_mass_in_a_graph(Tq):
    q, k, ids, lens = make(torch.bfloat16, 3, Tq, 8, 2, 128, 500, 200, seed=8)
    t = [x.to(DEV) for x in (q, k, ids, lens)]
    mass = torch.zeros(3, 2, 500, device=DEV)
    once = pipeline.key_mass(*t)
    g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(g, stream=side):
        fresh = pipeline.key_mass(*t)
        pipeline.key_mass(*t, mass=mass)
    torch.cuda.synchronize()
    mass.zero_()
    for n in range(1, 5):
        g.replay()
        eager = pipeline.key_mass(*t)
        torch.cuda.synchronize()
        assert torch.equal(fresh, once) and torch.equal(eager, once)
        close(mass, n * once.double().cpu(), n * Tq, 4, n * 4.0)


# ------------------------------------------------------------------------------- eviction


def keep(seen, n, budget, window, sink):
    """Positions kept, ascending: by sorted tuples."""
    if n <= budget:
        return list(range(n))
    must = [i for i in range(n) if i < sink or i >= n - window]
    rest = [i for i in range(n) if sink <= i < n - window]
    rest.sort(key=lambda i: (math.isnan(seen[i]), 0.0 if math.isnan(seen[i]) else -float(seen[i]), i))
    return sorted(must + rest[: budget - len(must)])


def odd_masses(B, Hkv, T, seed):
    """Ties, zeros of both signs, denormals, negatives, infinities and NaN among ordinary masses."""
    rng = np.random.default_rng(seed)
    m = np.exp(2 * rng.standard_normal((B, Hkv, T))).astype(np.float32)
    kind = rng.integers(0, 14, (B, Hkv, T))
    for i, x in enumerate((0.0, -0.0, 1e-42, -1.5, math.inf, -math.inf, math.nan, 0.5, 0.5)):
        m[kind == i] = x
    return m


EVICT = [
    # B, T, Hkv, D, dtype, budget, window, sink
    (1, 1, 1, 64, torch.bfloat16, 1, 0, 0),
    (2, 100, 2, 64, torch.float32, 30, 10, 4),
    (3, 1000, 4, 128, torch.bfloat16, 999, 100, 4),
    (2, 1025, 3, 128, torch.float16, 1, 0, 0),
    (2, 1024, 2, 32, torch.float32, 1024, 5, 5),
    (4, 3000, 2, 128, torch.bfloat16, 700, 700, 0),
    (2, 5000, 8, 96, torch.bfloat16, 1234, 64, 64),
    (1, 40000, 2, 64, torch.float16, 20000, 512, 4),
    (2, 32769, 2, 32, torch.bfloat16, 32768, 1, 0),
    (2, 100001, 3, 32, torch.bfloat16, 33000, 32800, 70),
    (3, 70000, 1, 32, torch.float16, 40000, 0, 33000),
]


@pytest.mark.parametrize("case", EVICT, ids=lambda c: "-".join(map(str, c)).replace("torch.", ""))
@pytest.mark.parametrize("shared", [False, True])
def test_evict(case, shared):
    B, T, Hkv, D, dtype, budget, window, sink = case
    m = odd_masses(B, Hkv, T, seed=T + budget)
    rng = np.random.default_rng(T)
    lens = rng.integers(0, T + 1, B)
    lens[0] = T
    g = torch.Generator().manual_seed(T)
    k, v = (torch.randn(B, T, Hkv, D, generator=g).to(dtype) for _ in range(2))
    k[0, T // 2] = math.nan  # bits move as they are
    print("evict", case, shared, lens.tolist(), flush=True)
    got = pipeline.evict(k.to(DEV), v.to(DEV), torch.from_numpy(m).to(DEV), budget, torch.from_numpy(lens).to(DEV),
                         window, sink, shared)
    k2, v2, m2, kept, n2 = [x.cpu() for x in got]
    out = (torch.full((B, budget + 3, Hkv, D), 7.0, dtype=dtype, device=DEV),
           torch.full((B, budget + 3, Hkv, D), 8.0, dtype=dtype, device=DEV),
           torch.full((B, Hkv, budget + 2), 9.0, device=DEV))
    again = pipeline.evict(k.to(DEV), v.to(DEV), torch.from_numpy(m).to(DEV), budget, torch.from_numpy(lens).to(DEV),
                           window, sink, shared, out)
    assert again[0] is out[0] and torch.equal(again[3].cpu(), kept)
    bits = {2: torch.int16, 4: torch.int32}[k.element_size()]
    for b in range(B):
        n = int(lens[b])
        assert int(n2[b]) == min(n, budget)
        for h in range(Hkv):
            if shared:
                with np.errstate(invalid="ignore"):
                    seen = np.zeros(T)
                    for x in range(Hkv):
                        seen = seen + m[b, x].astype(np.float64)
                    seen = seen.astype(np.float32)
            else:
                seen = m[b, h]
            at = keep(seen, n, budget, window, sink)
            row = kept[b] if shared else kept[b, h]
            assert row.tolist() == at + [-1] * (budget - len(at))
            for new, old, fill, o in ((k2, k, 7.0, out[0].cpu()), (v2, v, 8.0, out[1].cpu())):
                assert torch.equal(new[b, : len(at), h].view(bits), old[b, at, h].view(bits))
                assert (new[b, len(at):, h] == 0).all()
                assert torch.equal(o[b, : len(at), h].view(bits), old[b, at, h].view(bits))
                assert (o[b, len(at):, h] == fill).all()
            assert np.array_equal(m2[b, h, : len(at)].numpy(), m[b, h, at], equal_nan=True)
            assert (m2[b, h, len(at):] == 0).all() and (out[2][b, h, len(at):] == 9.0).all()


@pytest.mark.parametrize("R,T,Hkv,budget,window,sink", [(1, 1, 1, 1, 0, 0), (3, 700, 2, 100, 20, 4), (2, 1024, 8, 1023, 0, 1),
                                                        (4, 5000, 3, 2000, 512, 4), (2, 33000, 2, 9000, 0, 0),
                                                        (3, 98304, 2, 50000, 512, 4), (2, 70001, 1, 1, 0, 0)])
def test_evict_slots(R, T, Hkv, budget, window, sink):
    rng = np.random.default_rng(T)
    pool = R * T + 50
    table = rng.permutation(pool)[: R * T].reshape(R, T).astype(np.int32)
    table[:, 7::31] = -1
    table[:, 9::37] = pool + 4
    m = odd_masses(1, Hkv, pool, seed=T)
    lens = rng.integers(0, T + 1, R)
    lens[0] = T
    print("evict_slots", R, T, Hkv, budget, lens.tolist(), flush=True)
    wide = torch.full((1, Hkv, pool + 3), math.nan, device=DEV)
    wide[:, :, :pool] = torch.from_numpy(m).to(DEV)
    new, n2, kept = [x.cpu().numpy() for x in pipeline.evict_slots(
        torch.from_numpy(table).to(DEV), wide[:, :, :pool], budget, torch.from_numpy(lens).to(DEV), window, sink)]
    for r in range(R):
        n = int(lens[r])
        ok = (table[r, :n] >= 0) & (table[r, :n] < pool)
        seen = np.zeros(n)
        with np.errstate(invalid="ignore"):
            for h in range(Hkv):
                seen = seen + m[0, h, np.where(ok, table[r, :n], 0)].astype(np.float64)
        seen = np.where(ok, seen.astype(np.float32), np.nan)
        at = keep(seen, n, budget, window, sink)
        assert n2[r] == len(at) and kept[r].tolist() == at + [-1] * (budget - len(at))
        assert np.array_equal(new[r], np.concatenate([table[r, at], np.delete(table[r, :n], at), table[r, n:]]))


@pytest.mark.parametrize("T", [3000, 70000])
@pytest.mark.parametrize("kind", ["equal", "nan", "zero and one"])
def test_evict_of_ties_alone(T, kind):
    """All masses the same, none a number, or two values: the lower positions of the heavier ones."""
    m = torch.zeros(2, 2, T)
    if kind == "nan":
        m += math.nan
    if kind == "zero and one":
        m[:, :, T // 2:] = 1.0
    k = torch.zeros(2, T, 2, 32, dtype=torch.bfloat16, device=DEV)
    budget = T // 3
    lens = torch.tensor([T, T - 7], dtype=torch.int32, device=DEV)
    for shared in (False, True):
        kept = pipeline.evict(k, k, m.to(DEV), budget, lens, window=5, sink=2, shared=shared)[3].cpu()
        for b, n in enumerate((T, T - 7)):
            at = keep(m[b, 0].tolist(), n, budget, 5, 2)
            assert (kept[b] if shared else kept[b, 1]).tolist() == at


@pytest.mark.parametrize("T", [4096, 8191, 10000, 16384, 20001, 32768, 33000, 65537])
@pytest.mark.parametrize("odd", [False, True])
def test_evict_of_masses_as_they_accumulate(T, odd):
    """A third exactly zero, the rest spread over decades; odd: one row's end holds a NaN and a negative one."""
    rng = np.random.default_rng(T)
    m = np.where(rng.random((2, 2, T)) < 0.33, 0.0, np.exp(3 * rng.standard_normal((2, 2, T)) - 5)).astype(np.float32)
    if odd:
        m[1, 0, T - 40], m[1, 0, T - 41] = math.nan, -1.0
    k = torch.zeros(2, T, 2, 32, dtype=torch.bfloat16, device=DEV)
    lens = torch.tensor([T, T - 9], dtype=torch.int32, device=DEV)
    print("evict", T, odd, flush=True)
    for budget in (T // 5, T - T // 4):  # the threshold is a weight, or zero
        kept, n2 = pipeline.evict(k, k, torch.from_numpy(m).to(DEV), budget, lens, window=33, sink=4)[3:]
        assert n2.tolist() == [budget] * 2
        for b, n in enumerate((T, T - 9)):
            for h in range(2):
                assert kept[b, h].tolist() == keep(m[b, h], n, budget, 33, 4)


def test_evict_of_views_and_in_a_graph():
    """A cache's first rows (a view), masses of a longer buffer, replayed with new masses."""
    B, T, Hkv, D, budget = 2, 600, 2, 64, 200
    g = torch.Generator().manual_seed(1)
    big = torch.randn(B, 800, Hkv, 2, D, generator=g).to(torch.bfloat16).to(DEV)
    k, v = big[:, :T, :, 0], big[:, :T, :, 1]
    buf = torch.rand(B, Hkv, 800, generator=g).to(DEV)
    mass = buf[:, :, :T]
    first = pipeline.evict(k, v, mass, budget, window=30, sink=4)
    dense = pipeline.evict(k.contiguous(), v.contiguous(), mass.contiguous(), budget, window=30, sink=4)
    for a, b in zip(first, dense):
        assert torch.equal(a, b)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        outs = pipeline.evict(k, v, mass, budget, window=30, sink=4, shared=True)
    for _ in range(3):
        buf.copy_(torch.rand_like(buf))
        graph.replay()
        ref = pipeline.evict(k, v, mass, budget, window=30, sink=4, shared=True)
        torch.cuda.synchronize()
        for a, b in zip(outs, ref):
            assert torch.equal(a, b)


def test_a_server_s_round():
    """Requests behind one prompt decode over it and their own caches, weigh their own keys by the
    whole softmax, give up most of them, and go on over what is left, dense and paged alike."""
    B, Hq, Hkv, D, Tp, T, budget = 3, 8, 2, 64, 300, 512, 128
    dt = torch.bfloat16
    g = torch.Generator().manual_seed(9)
    kp, vp = (torch.randn(1, Tp, Hkv, D, generator=g).to(dt).to(DEV) for _ in range(2))
    k, v = (torch.randn(B, T, Hkv, D, generator=g).to(dt).to(DEV) for _ in range(2))
    k[:, 100:110] *= 4.0  # keys worth keeping
    ids = torch.arange(T, dtype=torch.int32, device=DEV).expand(B, 1, T).contiguous()
    lens = torch.full((B, 1), T, dtype=torch.int32, device=DEV)
    mass = torch.zeros(B, Hkv, T, device=DEV)
    ref = torch.zeros(B, Hkv, T, dtype=torch.float64)
    for step in range(3):
        q = torch.randn(B, 1, Hq, D, generator=g).to(dt).to(DEV)
        out, lse = pipeline.prefix_read(q, kp, vp, k, v, ids, lens, return_lse=True)
        pipeline.key_mass(q, k, ids, lens, lse=lse, mass=mass)
        s = torch.einsum("bhgd,bthd->bhgt", q.double().cpu().view(B, Hkv, Hq // Hkv, D), k.double().cpu()) * D ** -0.5
        ref += torch.exp(s - lse.double().cpu().view(B, Hkv, -1, 1)).sum(2)
    close(mass, ref, 3, 4, 4.0)
    k2, v2, m2, kept, n2 = pipeline.evict(k, v, mass, budget, window=16, sink=4, shared=True)
    assert (n2 == budget).all() and bool((kept[:, :4] == torch.arange(4, device=DEV)).all())
    # the same through a slot table over one pool of all rows
    table = torch.arange(B * T, dtype=torch.int32, device=DEV).view(B, T)
    pooled = mass.permute(1, 0, 2).reshape(1, Hkv, B * T).contiguous()
    new, n3, kept3 = pipeline.evict_slots(table, pooled, budget, window=16, sink=4)
    assert torch.equal(kept3, kept) and torch.equal(n3, n2)
    q = torch.randn(B, 1, Hq, D, generator=g).to(dt).to(DEV)
    short = torch.arange(budget, dtype=torch.int32, device=DEV).expand(B, 1, budget).contiguous()
    n = n2.view(B, 1)
    a = pipeline.prefix_read(q, kp, vp, k2, v2, short, n)
    b = pipeline.prefix_read(q, kp, vp, k.view(1, B * T, Hkv, D), v.view(1, B * T, Hkv, D), new[:, None, :budget], n)
    assert torch.equal(a, b)
    # the smaller cache is indexed and decoded as any other
    buckets = pipeline.segment_buckets(k2[:1], 16, pool=4, max_size=64)
    config = pipeline.PortConfig(cluster_block_size=8, bucket_size=8, bucket_cap=64, top_p=16, top_k=budget, window_size=0,
                                 sink_size=0)
    dec, lists, lengths = pipeline.flat_decode(q[:1], k2[:1], v2[:1], torch.tensor([budget - 1], device=DEV,
                                                                                   dtype=torch.int32), buckets, config)
    assert (lengths == budget).all()
    whole = pipeline.lsa_read(q[:1], k2[:1], v2[:1], short[:1], n[:1], D ** -0.5)
    assert ((dec.float() - whole.float()).abs() <= 2.0 ** -8 * whole.float().abs() + 2.0 ** -11).all()


def test_offsets_past_32_bits():
    """Token rows 2^24 elements apart: 300 of them span 10 GB."""
    n, apart = 300, 1 << 24
    whole = torch.empty(n * apart, dtype=torch.bfloat16, device=DEV)
    for Tq in (1, 5):
        q, k, ids, lens = make(torch.bfloat16, 2, Tq, 8, 2, 64, n, 40, pool=True, seed=41)
        far = whole.as_strided((1, n, 2, 64), (n * apart, apart, 64, 1))
        far.copy_(k)
        mass = pipeline.key_mass(q.to(DEV), far, ids.to(DEV), lens.to(DEV))
        close(mass, want(q, k, ids, lens), 2 * Tq, 4)
    v = whole.as_strided((1, n, 2, 64), (n * apart, apart, 64, 1), 128)
    v.copy_(-k)
    k2, v2, m2, kept, length = pipeline.evict(far, v, mass, 120, window=9, sink=2)
    assert length.tolist() == [120]
    for h in range(2):
        at = kept[0, h].long().cpu()
        assert torch.equal(k2[0, :, h].cpu(), k[0, at, h]) and torch.equal(v2[0, :, h].cpu(), -k[0, at, h])
        assert torch.equal(m2[0, h].cpu(), mass[0, h].cpu()[at])
    assert kept[0, :, -1].tolist() == [n - 1] * 2


def test_threads_on_one_stream():
    """Calls of several threads share a stream's scratch and counters: each gets its own results."""
    import concurrent.futures

    jobs = []
    for seed in range(4):
        q, k, ids, lens = make(torch.bfloat16, 2, 1 + seed % 2 * 4, 8, 2, 64, 40000, 300, seed=50 + seed)
        args = [x.to(DEV) for x in (q, k, ids, lens)]
        v = args[1] * 2
        table = torch.randperm(40000, device=DEV, dtype=torch.int64).to(torch.int32)[None]

        def job(args=args, v=v, table=table):
            mass = pipeline.key_mass(*args)
            read = pipeline.prefix_read(args[0], args[1][:1, :700], v[:1, :700], args[1], v, *args[2:])
            return (mass, read, pipeline.evict(args[1], v, mass, 9000)[3],
                    pipeline.evict_slots(table, mass[:1], 9000)[0])

        jobs.append(job)
    alone = [job() for job in jobs]
    torch.cuda.synchronize()
    with concurrent.futures.ThreadPoolExecutor(4) as pool:
        for _ in range(10):
            for job, got in [(i, f.result()) for i, f in enumerate([pool.submit(j) for j in jobs])]:
                assert all(torch.equal(x, y) for x, y in zip(got, alone[job]))
