"""prefix_read (attention over shared prefixes and own lists in one softmax) vs 64 bits.

Bound on an output: its own rounding, half a step (finfo.eps / 2 of it); the weights' rounding to
16 bits on the matrix cores, half a step of each weight, so of at most the largest |v|; and 2^-13
of the largest |v| for the fp32 scores: D <= 256 products of |q k| scale <= 8 or so in all here, each
sum step off by 2^-24, is under 2^-14 of a score and moves a weight's share by twice that. The
logarithm of sums moves by what a score does: 2^-13.
"""

import math

import numpy as np
import pytest
import torch

from lsa_rocm_lab.port import pipeline, shared_prefix

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(dtype, B, Tq, P, Tp, Hq, Hkv, D, Tk, W, per_head=False, paged=0, seed=0):
    """CPU tensors of a case: prefixes (or one pool with slots), own caches, lists with -1, repeated
    and out-of-range ids, every third list empty; the last prefix row of P > 1 names no prefix."""
    g = torch.Generator().manual_seed(seed)
    rng = np.random.default_rng(seed)
    c = dict(q=torch.randn(B, Tq, Hq, D, generator=g).to(dtype), slots=None)
    if paged:
        pages = P * -(-Tp // paged)
        rows = (pages + 3) * paged
        where = rng.permutation(pages + 3)[:pages, None] * paged + np.arange(paged)
        c["slots"] = torch.from_numpy(where.reshape(P, -1)[:, :Tp].astype(np.int32)).contiguous()
        c["slots"][:, 3::29] = -1
        c["slots"][:, 5::31] = rows + 7
        shape = (1, rows, Hkv, D)
    else:
        shape = (P, Tp, Hkv, D)
    c["kp"], c["vp"] = (torch.randn(*shape, generator=g).to(dtype) for _ in range(2))
    c["k"], c["v"] = (torch.randn(B, Tk, Hkv, D, generator=g).to(dtype) for _ in range(2))
    lead = (B, Tq, Hkv) if per_head else (B, Tq)
    n = int(np.prod(lead))
    ids = rng.integers(0, max(Tk, 1), (n, W)).astype(np.int32)
    ids[:, 2::7] = -1
    if W:
        ids[::5, 0] = Tk + 2
    lens = rng.integers(0, W + 1, n).astype(np.int32)
    lens[::3] = 0
    c["ids"], c["lens"] = torch.from_numpy(ids.reshape(*lead, W)), torch.from_numpy(lens.reshape(lead))
    c["plen"] = torch.from_numpy(rng.integers(0, Tp + 1, P).astype(np.int32)) if P > 1 else None
    c["prow"] = torch.from_numpy((np.arange(B) % (P + 1)).astype(np.int32)) if P > 1 else None  # P: none
    return c


def want(c, scale=None):
    """out [B, Tq, Hq, D] and lse in fp64, on the CPU."""
    q = c["q"].double()
    B, Tq, Hq, D = q.shape
    Hkv = c["kp"].shape[2]
    G = Hq // Hkv
    scale = D ** -0.5 if scale is None else scale
    P = c["slots"].shape[0] if c["slots"] is not None else c["kp"].shape[0]
    out, lse = torch.zeros(B, Tq, Hq, D, dtype=torch.float64), torch.full((B, Tq, Hq), -math.inf, dtype=torch.float64)
    for b in range(B):
        p = 0 if c["prow"] is None else int(c["prow"][b])
        for t in range(Tq):
            for g in range(Hkv):
                ks, vs = [], []
                if 0 <= p < P:
                    Tp = c["slots"].shape[1] if c["slots"] is not None else c["kp"].shape[1]
                    n = Tp if c["plen"] is None else max(0, min(Tp, int(c["plen"][p])))
                    if c["slots"] is not None:
                        at = c["slots"][p, :n].long()
                        at = at[(at >= 0) & (at < c["kp"].shape[1])]
                        ks.append(c["kp"][0, at, g]), vs.append(c["vp"][0, at, g])
                    else:
                        ks.append(c["kp"][p, :n, g]), vs.append(c["vp"][p, :n, g])
                if c.get("k") is not None:
                    per = c["ids"].dim() == 4
                    ids = (c["ids"][b, t, g] if per else c["ids"][b, t])[: int(c["lens"][b, t, g] if per else c["lens"][b, t])]
                    ids = ids.long()
                    ids = ids[(ids >= 0) & (ids < c["k"].shape[1])]
                    bb = b if c["k"].shape[0] == B else 0
                    ks.append(c["k"][bb, ids, g]), vs.append(c["v"][bb, ids, g])
                kk, vv = torch.cat(ks).double(), torch.cat(vs).double()
                if not len(kk):
                    continue
                for h in range(g * G, (g + 1) * G):
                    s = scale * (kk @ q[b, t, h])
                    lse[b, t, h] = torch.logsumexp(s, 0)
                    out[b, t, h] = torch.softmax(s, 0) @ vv
    return out, lse


def dev(x):
    return None if x is None else x.to(DEV)


def call(c, scale=None, **kw):
    own = [dev(c[n]) for n in ("k", "v", "ids", "lens")] if c.get("k") is not None else []
    print("prefix", {n: tuple(x.shape) for n, x in c.items() if torch.is_tensor(x)}, c["q"].dtype, flush=True)
    return pipeline.prefix_read(dev(c["q"]), dev(c["kp"]), dev(c["vp"]), *own, scale=scale, prefix_lengths=dev(c["plen"]),
                                prefix_rows=dev(c["prow"]), prefix_slots=dev(c["slots"]), return_lse=True, **kw)


def compare(got, exact, c):
    out, lse = got[0].double().cpu(), got[1].double().cpu()
    ref, rlse = exact
    half = torch.finfo(c["q"].dtype).eps / 2
    vals = [c[n].double().abs()[torch.isfinite(c[n])] for n in ("vp", "v") if c.get(n) is not None]
    vmax = max((float(x.max()) for x in vals if x.numel()), default=0.0)
    weights = half if c["q"].dtype != torch.float32 else 0.0
    bound = half * ref.abs() + (weights + 2.0 ** -13) * vmax
    off = (out - ref).abs()
    assert (off <= bound).all(), f"off by {(off / bound).max():.2f} of the bound"
    none = torch.isinf(rlse)
    assert torch.equal(torch.isinf(lse) & (lse < 0), none)
    d = (lse - rlse)[~none].abs()
    assert d.numel() == 0 or float(d.max()) <= 2.0 ** -13
    assert (out[none] == 0).all()


CASES = [
    # dtype, B, Tq, P, Tp, Hq, Hkv, D, Tk, W, per_head, paged
    (torch.float32, 2, 1, 1, 130, 8, 2, 64, 40, 17, False, 0),
    (torch.float32, 3, 2, 2, 65, 4, 4, 32, 40, 17, True, 16),
    (torch.float32, 1, 1, 1, 1, 8, 1, 128, 1, 1, False, 0),
    (torch.float32, 5, 1, 3, 200, 4, 2, 256, 40, 33, True, 0),
    (torch.bfloat16, 1, 1, 1, 64, 4, 1, 128, 64, 64, False, 0),
    (torch.bfloat16, 1, 1, 1, 63, 1, 1, 128, 9, 5, False, 0),
    (torch.bfloat16, 7, 1, 1, 257, 32, 8, 128, 100, 65, True, 0),
    (torch.bfloat16, 40, 1, 1, 1000, 8, 2, 128, 100, 65, False, 0),
    (torch.bfloat16, 33, 3, 3, 500, 16, 2, 128, 50, 20, False, 16),
    (torch.bfloat16, 6, 4, 2, 333, 8, 8, 64, 50, 20, True, 0),
    (torch.bfloat16, 150, 1, 1, 321, 4, 2, 64, 30, 8, False, 0),
    (torch.bfloat16, 4, 1, 1, 300, 8, 2, 256, 30, 8, False, 0),
    (torch.bfloat16, 4, 1, 1, 300, 8, 2, 32, 30, 8, False, 16),
    (torch.float16, 2, 1, 1, 4097, 32, 8, 128, 600, 520, True, 0),
    (torch.float16, 9, 2, 4, 129, 8, 1, 128, 50, 20, False, 1),
    (torch.float16, 17, 1, 1, 96, 2, 2, 64, 50, 20, False, 16),
    (torch.float16, 64, 4, 1, 640, 8, 1, 64, 50, 20, False, 0),
    (torch.float16, 1, 1, 1, 9000, 1, 1, 64, 5, 2, False, 0),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)).replace("torch.", ""))
def test_against_64_bits(case):
    c = make(*case)
    compare(call(c), want(c), c)


@pytest.mark.parametrize("dtype,D", [(torch.float32, 64), (torch.bfloat16, 128), (torch.float16, 64)])
def test_no_own_part_and_no_prefix(dtype, D):
    c = make(dtype, 5, 1, 1, 70, 4, 2, D, 20, 9)
    c["k"] = None
    compare(call(c), want(c), c)
    c = make(dtype, 5, 1, 1, 70, 4, 2, D, 20, 9)
    c["plen"] = torch.zeros(1, dtype=torch.int32)
    compare(call(c), want(c), c)
    c["kp"], c["vp"], c["plen"] = c["kp"][:, :0], c["vp"][:, :0], None
    compare(call(c), want(c), c)
    c["prow"] = torch.tensor([-1, 0, 5, -(2 ** 31), 2 ** 31 - 1], dtype=torch.int32)
    compare(call(c), want(c), c)


@pytest.mark.parametrize("dtype,D,paged", [(torch.float32, 64, 0), (torch.bfloat16, 128, 0), (torch.bfloat16, 128, 16),
                                           (torch.float16, 64, 16), (torch.float16, 128, 0)])
def test_what_is_masked_may_hold_anything(dtype, D, paged):
    """Keys past a prefix's length, unlisted keys and the pool's other rows: NaN and infinities."""
    c = make(dtype, 8, 2, 2, 150, 8, 2, D, 60, 20, paged=paged, seed=3)
    c["plen"] = torch.tensor([37, 100], dtype=torch.int32)
    keep_p = torch.zeros(c["kp"].shape[:2], dtype=torch.bool)
    if paged:
        for p, n in enumerate((37, 100)):
            at = c["slots"][p, :n].long()
            keep_p[0, at[(at >= 0) & (at < keep_p.shape[1])]] = True
    else:
        keep_p[0, :37] = keep_p[1, :100] = True
    keep = torch.zeros(c["k"].shape[:2], dtype=torch.bool)
    for b in range(8):
        for t in range(2):
            at = c["ids"][b, t, : int(c["lens"][b, t])].long()
            keep[b, at[(at >= 0) & (at < 60)]] = True
    exact = want(c)
    for i, x in enumerate((math.nan, math.inf, -math.inf)):
        for n, k in (("kp", keep_p), ("vp", keep_p), ("k", keep), ("v", keep)):
            at = torch.nonzero(~k)[i::3]
            c[n][at[:, 0], at[:, 1]] = x
    # row 0 of a cache stands in for masked loads: keep it odd where nothing lists it
    compare(call(c), exact, c)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_one_large_and_many_small_weights(dtype):
    """16k keys of weight 2^-20 beside one of 1: the many hold 2^-6 of the sum."""
    D, n = 64, 16384
    c = make(dtype, 2, 1, 1, n, 2, 1, D, 4, 2)
    c["q"].zero_()
    c["q"][..., 0] = 16.0
    c["kp"].zero_()
    c["kp"][0, n // 3, 0, 0] = 20.0 * math.log(2.0) / 16.0
    c["vp"].fill_(1.0)
    c["vp"][0, n // 3] = 0.0
    c["k"] = None
    compare(call(c, scale=1.0), want(c, scale=1.0), c)


@pytest.mark.parametrize("dtype,B", [(torch.bfloat16, 3), (torch.bfloat16, 150), (torch.float16, 30), (torch.float16, 150)])
def test_a_key_that_fills_its_row_returns_its_value(dtype, B):
    """One score far above the rest: the output is that key's value, bit for bit."""
    g = torch.Generator().manual_seed(2)
    q = torch.randn(B, 1, 2, 128, generator=g)
    q = (q / q.norm(dim=-1, keepdim=True)).to(dtype)
    kp, vp = (torch.randn(1, 300, 1, 128, generator=g).to(dtype) for _ in range(2))
    kp[0, 7::11] = 0
    at = torch.randint(0, 300, (B,), generator=g)
    kp[0, at, 0] = q[:, 0, 0]
    out = pipeline.prefix_read(q[:, :, :1].to(DEV), kp.to(DEV), vp.to(DEV), scale=1000.0).cpu()
    s = 1000.0 * q[:, 0, :1].double() @ kp[0, :, 0].double().T
    gap = s.topk(2, -1).values  # where no other key has 2^-60 of the weight
    sure = (gap[:, 0, 0] - gap[:, 0, 1] > 42.0).nonzero()[:, 0]
    assert len(sure) > B // 2
    assert torch.equal(out[sure, 0, 0], vp[0, s[sure, 0].argmax(-1), 0])


@pytest.mark.parametrize("dtype,D", [(torch.float32, 64), (torch.bfloat16, 128), (torch.float16, 128)])
def test_views_strides_and_a_shared_pool(dtype, D):
    """Caches as views of wider buffers, K and V halves of one, the own cache a pool of every row."""
    c = make(dtype, 6, 1, 1, 200, 8, 2, D, 90, 30, seed=5)
    c["k"], c["v"] = c["k"][:1], c["v"][:1]
    exact = want(c)
    both = torch.full((1, 210, 2, 3, 2 * D), math.nan, dtype=dtype, device=DEV)  # token, K | V, heads
    kp, vp = both[:, 4:204, 0, 1:, :D], both[:, 4:204, 1, 1:, :D]
    kp.copy_(c["kp"]), vp.copy_(c["vp"])
    got = pipeline.prefix_read(dev(c["q"]), kp, vp, dev(c["k"]), dev(c["v"]), dev(c["ids"]), dev(c["lens"]),
                               return_lse=True)
    compare(got, exact, c)
    # K and V of different strides are made dense
    got = pipeline.prefix_read(dev(c["q"]), kp, dev(c["vp"]), dev(c["k"]), dev(c["v"]), dev(c["ids"]).long(),
                               dev(c["lens"]).long(), return_lse=True)
    compare(got, exact, c)


def test_as_the_read_over_a_joined_list():
    """The prefix laid in front of each own cache and listed whole: lsa_read's result."""
    c = make(torch.bfloat16, 4, 1, 1, 96, 8, 2, 128, 64, 24, seed=7)
    B, W = 4, 24
    k = torch.cat([c["kp"].expand(B, -1, -1, -1), c["k"]], 1).to(DEV)
    v = torch.cat([c["vp"].expand(B, -1, -1, -1), c["v"]], 1).to(DEV)
    own = torch.where((c["ids"] >= 0) & (c["ids"] < 64) & (torch.arange(W) < c["lens"][..., None]), c["ids"] + 96, -1)
    ids = torch.cat([torch.arange(96, dtype=torch.int32).expand(B, 1, 96), own], -1).to(DEV)
    lens = torch.full((B, 1), 96 + W, dtype=torch.int32, device=DEV)
    ref = pipeline.lsa_read(c["q"].to(DEV), k, v, ids, lens, 128 ** -0.5)
    out, _ = call(c)
    # each side rounds its output (half a step) and this one its weights
    bound = 2.0 ** -8 * ref.float().abs() + (2.0 ** -9 + 2.0 ** -12) * 5.0
    assert ((out.float() - ref.float()).abs() <= bound).all()


@pytest.mark.parametrize("dtype,D", [(torch.float32, 64), (torch.bfloat16, 128)])
def test_repeats_other_streams_and_graphs(dtype, D):
    c = make(dtype, 9, 2, 1, 700, 8, 2, D, 300, 280, seed=11)
    first = call(c)
    t = {n: dev(c[n]) for n in ("q", "kp", "vp", "k", "v", "ids", "lens")}

    def step():
        return pipeline.prefix_read(t["q"], t["kp"], t["vp"], t["k"], t["v"], t["ids"], t["lens"], return_lse=True)

    for _ in range(3):
        again = step()
        assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    side.synchronize()
    assert torch.equal(other[0], first[0])
    graphs, outs = [], []
    for _ in range(2):  # two graphs of one stream, replayed on two
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(step())
        graphs.append(g)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        for o in outs:
            o[0].fill_(7.0)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o in outs:
            assert torch.equal(o[0], first[0]) and torch.equal(o[1], first[1])
    t["q"].copy_(torch.randn_like(t["q"]))  # new inputs in place
    now = step()
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0][0], now[0]) and not torch.equal(now[0], first[0])


def test_a_row_does_not_depend_on_its_neighbours_prefix():
    """Rows of several prefixes: each as it reads alone (within the rounding of another split)."""
    c = make(torch.bfloat16, 12, 1, 3, 400, 8, 2, 128, 50, 20, seed=13)
    c["plen"] = torch.tensor([400, 17, 230], dtype=torch.int32)
    c["prow"] = torch.tensor([2, 0, 1, 1, 2, 0, -1, 2, 0, 0, 1, 7], dtype=torch.int32)
    compare(call(c), want(c), c)


@pytest.mark.parametrize("dtype,B,Tq,P,Hq,paged", [
    (torch.bfloat16, 5, 1, 1500, 8, 0),   # more prefixes than rows, some past the first thousand
    (torch.bfloat16, 600, 1, 9, 8, 16),   # several blocks a prefix
    (torch.float16, 70, 3, 40, 4, 0),
    (torch.float32, 20, 1, 1100, 4, 0),
])
def test_many_prefixes(dtype, B, Tq, P, Hq, paged):
    """Rows spread unevenly over prefixes, some of which none reads."""
    c = make(dtype, B, Tq, P, 40, Hq, 2, 64, 30, 6, paged=paged, seed=17)
    rng = np.random.default_rng(18)
    c["prow"] = torch.from_numpy((P * rng.random(B) ** 3).astype(np.int32))
    c["prow"][:4] = torch.tensor([P - 1, -1, P, P - 1], dtype=torch.int32)
    compare(call(c), want(c), c)


@pytest.mark.parametrize("dtype,B,Tq,paged", [(torch.bfloat16, 7, 1, 0), (torch.float16, 4, 40, 16), (torch.float32, 6, 2, 0)])
def test_a_prefix_a_row(dtype, B, Tq, paged):
    """Without prefix_rows row b reads prefix b; also from a graph that a first call is captured into."""
    c = make(dtype, B, Tq, B, 130, 8, 2, 64, 30, 6, paged=paged, seed=19)
    c["prow"] = torch.arange(B, dtype=torch.int32)
    exact = want(c)
    c["prow"] = None
    t = {n: dev(c[n]) for n in ("q", "kp", "vp", "k", "v", "ids", "lens", "plen", "slots")}
    print("a prefix a row", dtype, B, Tq, paged, flush=True)

    def step():
        return pipeline.prefix_read(t["q"], t["kp"], t["vp"], t["k"], t["v"], t["ids"], t["lens"], return_lse=True,
                                    prefix_lengths=t["plen"], prefix_slots=t["slots"])

    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    compare(step(), exact, c)
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        compare(out, exact, c)


@pytest.mark.parametrize("dtype,D", [(torch.float32, 64), (torch.bfloat16, 128), (torch.float16, 32)])
@pytest.mark.parametrize("scale", [0.0, -0.2])
def test_scales_that_are_not_positive(dtype, D, scale):
    c = make(dtype, 5, 2, 1, 150, 8, 2, D, 40, 9, seed=23)
    compare(call(c, scale=scale), want(c, scale=scale), c)


@pytest.mark.parametrize("B", [2, 80])
@pytest.mark.parametrize("paged", [False, True])
def test_offsets_past_32_bits(B, paged):
    """Token rows 2^24 elements apart: 300 of them span 10 GB."""
    n, apart = 300, 1 << 24
    c = make(torch.bfloat16, B, 1, 1, n, 4, 1, 64, n, 40, seed=29)
    c["k"], c["v"] = c["k"][:1], c["v"][:1]
    whole = torch.empty(n * apart, dtype=torch.bfloat16, device=DEV)
    views = []
    for i, x in enumerate((c["kp"], c["vp"], c["k"], c["v"])):
        views.append(whole.as_strided((1, n, 1, 64), (n * apart, apart, 64, 1), 64 * i))
        views[-1].copy_(x)
    if paged:
        c["slots"] = torch.from_numpy(np.random.default_rng(1).permutation(n).astype(np.int32))[None]
    got = pipeline.prefix_read(dev(c["q"]), views[0], views[1], views[2], views[3], dev(c["ids"]), dev(c["lens"]),
                               prefix_slots=dev(c["slots"]), return_lse=True)
    compare(got, want(c), c)


def test_a_chunk_of_a_prompt():
    """Query rows by the thousand (a few checked): many column blocks."""
    c = make(torch.bfloat16, 1, 2500, 1, 500, 8, 2, 128, 30, 6, seed=31)
    got = call(c)
    rows = [0, 1, 77, 1023, 1024, 2047, 2499]
    few = dict(c, q=c["q"][:, rows], ids=c["ids"][:, rows], lens=c["lens"][:, rows])
    compare((got[0][:, rows], got[1][:, rows]), want(few), few)


@pytest.mark.parametrize("B,Tq,P,per_head,pool,own", [(5, 3, 1, False, False, True), (6, 1, 6, True, False, True),
                                                      (4, 2, 3, True, True, True), (5, 1, 5, False, False, False)])
def test_in_slabs_of_rows(monkeypatch, B, Tq, P, per_head, pool, own):
    c = make(torch.bfloat16, B, Tq, P, 90, 8, 2, 64, 30, 9, per_head, seed=37)
    if pool:
        c["k"], c["v"] = c["k"][:1], c["v"][:1]
    if not own:
        c["k"] = None
    if P == B:
        c["prow"] = torch.arange(B, dtype=torch.int32)
    exact = want(c)
    if P == B:
        c["prow"] = None
    monkeypatch.setattr(shared_prefix, "_SLAB_BYTES", 1)
    compare(call(c), exact, c)
