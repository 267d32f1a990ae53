"""The 8-bit cache (byte_append, byte_values, byte_read) vs 64 bits.

What a code may be off by: half a step of it, which is the scale for int8 and, for e4m3, 2^-3 of its
power of two times the scale (at least 2^-9 of it); a value that the fp32 norm and rotation move by 2^-20 of
what it is made of moves by 2^-20 448 steps at most, 2^-11, before it is rounded: the bound is 0.5 + 2^-9 steps.
A scale is off by as much as its largest value: 2^-20. byte_read's bound: half a step of the output, 2^-13 of the
largest |v| for fp32 scores (D <= 256 products of |q k| scale <= 8 or so in all, each sum off by 2^-24: 2^-14 of a
score, twice that of a weight), and 2^-16 of it for weights in two bf16 parts.
"""

import math

import numpy as np
import pytest
import torch

from lsa_rocm_lab.port import byte_cache as module
from lsa_rocm_lab.port import pipeline
from test_gpu_rotary import want as turned

pytestmark = pytest.mark.gpu
DEV = "cuda"
MOST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
BOTH = [torch.int8, torch.float8_e4m3fn]


def numbers(codes):
    return codes.cpu().float().double()


def steps(y, scale, dtype):
    """The step of the code of y."""
    if dtype == torch.int8:
        return scale.expand_as(y)
    _, e = torch.frexp((y / scale).abs())
    return torch.exp2((e - 4).clamp(-9, 5).double()) * scale


def paged(batch, tokens, page, gen, spare=3):
    """Slot table [batch, tokens] over pages of a pool, and the pool's rows."""
    per = -(-tokens // page)
    where = torch.randperm(batch * per + spare, generator=gen)[: batch * per].view(batch, per, 1) * page
    return (where + torch.arange(page)).reshape(batch, -1)[:, :tokens].to(torch.int32).contiguous(), (batch * per + spare) * page


APPENDS = [
    # dtype, code, block, page, B, T, Hq, Hkv, D, pairs, interleaved, norm, cache, ragged
    (torch.bfloat16, torch.int8, 64, 0, 1, 1, 32, 8, 128, 64, False, True, 200, False),
    (torch.bfloat16, torch.float8_e4m3fn, 64, 64, 7, 1, 8, 2, 128, 64, False, True, 200, False),
    (torch.bfloat16, torch.int8, 16, 16, 5, 70, 8, 2, 128, 64, True, True, 333, True),
    (torch.float16, torch.float8_e4m3fn, 1, 0, 3, 65, 4, 4, 64, 16, False, False, 100, True),
    (torch.float16, torch.int8, 1, 1, 2, 3, 4, 1, 32, 16, False, True, 9, False),
    (torch.float32, torch.int8, 32, 0, 2, 129, 6, 2, 256, 100, False, True, 257, True),
    (torch.float32, torch.float8_e4m3fn, 8, 16, 4, 1, 2, 2, 64, 0, False, False, 50, False),
    (torch.bfloat16, torch.int8, 2, 32, 1, 1000, 8, 8, 128, 5, False, True, 1003, False),
    (torch.float16, torch.float8_e4m3fn, 4, 64, 9, 31, 3, 1, 256, 128, True, True, 64, True),
    (torch.bfloat16, torch.float8_e4m3fn, 64, 0, 2, 2000, 0, 2, 64, 32, False, False, 2100, False),
]


def setup(case, seed=0, grow=1.0):
    dtype, code, block, page, B, T, Hq, Hkv, D, pairs, interleaved, norm, cache, ragged = case
    g = torch.Generator().manual_seed(seed)
    table, rows = paged(B, cache, page, g) if page else (None, cache)
    held = pipeline.byte_cache(1 if page else B, rows, Hkv, D, block, code, DEV)
    raw = torch.randint(0, 256, (2, *held.k.shape), generator=g).to(torch.uint8)
    raw[(raw & 127) == 127] = 0x31  # e4m3's NaN has a test of its own
    raw[raw == 128] = 0x31          # -128 is no code
    held.k.copy_(raw[0].view(code)), held.v.copy_(raw[1].view(code))
    held.scales.copy_(0.01 + 0.01 * torch.rand(held.scales.shape, generator=g) if code == torch.int8 else
                      0.003 + 0.003 * torch.rand(held.scales.shape, generator=g))
    wide = torch.randn(B, T, Hq + 2 * Hkv, D, generator=g).mul(grow).to(dtype)
    starts = torch.randint(0, cache - T + 1, (B,), generator=g).to(torch.int32)
    lens = torch.randint(0, T + 1, (B,), generator=g).to(torch.int32) if ragged else None
    if ragged:
        lens[0] = 0
    freq = pipeline.rotary_frequencies(2 * pairs) if pairs else None
    w = torch.rand(2, D, generator=g).add(0.5).to(dtype)
    return dict(held=held, table=table, wide=wide, q=wide[:, :, :Hq], k=wide[:, :, Hq:Hq + Hkv], v=wide[:, :, Hq + Hkv:],
                starts=starts, lens=lens, freq=freq, wq=w[0] if norm else None, wk=w[1] if norm else None)


def dev(x):
    return None if x is None else x.to(DEV)


def append(s, case, **over):
    Hq, Hkv = case[6], case[7]
    wide = s["wide"].to(DEV)
    args = dict(lengths=dev(s["lens"]), slot_table=dev(s["table"]), q=wide[:, :, :Hq] if Hq else None,
                frequencies=dev(s["freq"]), q_weight=dev(s["wq"]), k_weight=dev(s["wk"]), interleaved=case[10])
    args.update(over)
    return pipeline.byte_append(s["held"], wide[:, :, Hq:Hq + Hkv], wide[:, :, Hq + Hkv:], dev(s["starts"]), **args)


def check_append(s, case, before, q):
    dtype, code, block, page, B, T, Hq, Hkv, D, pairs, interleaved, norm, cache, ragged = case
    held = s["held"]
    kc, vc, sc = numbers(held.k), numbers(held.v), held.scales.cpu().double()
    old_k, old_v, old_s = before
    free = torch.ones(kc.shape[:2], dtype=torch.bool)   # rows that no append may change
    free_s = torch.ones(sc.shape[:2], dtype=torch.bool)
    half = torch.finfo(dtype).eps / 2
    for b in range(B):
        n, first = T if s["lens"] is None else int(s["lens"][b]), int(s["starts"][b])
        pos = first + torch.arange(T)
        if q is not None:
            ref, made = turned(s["q"][b], pos, s["freq"], s["wq"], 1e-6, interleaved)
            off = (q[b].double().cpu() - ref).abs()
            assert (off[:n] <= half * ref[:n].abs() + 2.0 ** -20 * made[:n] + torch.finfo(dtype).tiny).all()
            assert (q[b, n:] == 0).all()
        ref, _ = turned(s["k"][b], pos, s["freq"], s["wk"], 1e-6, interleaved)
        at = first
        while at < first + n:
            lead, last = at // block * block, min(at // block * block + block, first + n)
            row = s["table"][b, lead].item() if page else lead
            c, place = (0, row // block) if page else (b, lead // block)
            free[c, row:row + last - lead] = False
            free_s[c, place] = False
            for i, (codes, old, x) in enumerate(((kc, old_k, ref), (vc, old_v, s["v"][b].double()))):
                x = x[at - first:last - first]
                scale = x.abs().amax((0, 2)) / MOST[code]
                if at > lead:
                    scale = torch.maximum(scale, old_s[c, place, :, i])
                got = sc[c, place, :, i]
                assert ((got - scale).abs() <= 2.0 ** -20 * scale).all()
                have = codes[c, row + at - lead:row + last - lead] * got[:, None]
                lim = (0.5 + 2.0 ** -9) * steps(x, got[None, :, None], code)
                assert ((have - x).abs() <= lim + 2.0 ** -20 * scale[:, None] * MOST[code]).all()
                was = old[c, row:row + at - lead]
                now = codes[c, row:row + at - lead]
                same = got == old_s[c, place, :, i]
                assert torch.equal(now[:, same], was[:, same])
                y = was * old_s[c, place, :, i, None]
                assert ((now * got[:, None] - y).abs() <= (0.5 + 2.0 ** -9) * steps(y, got[None, :, None], code)).all()
            at = last
    assert torch.equal(kc[free], old_k[free]) and torch.equal(vc[free], old_v[free]) and torch.equal(sc[free_s], old_s[free_s])


@pytest.mark.parametrize("grow", [1.0, 8.0])
@pytest.mark.parametrize("case", APPENDS, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_append(case, grow):
    """Into blocks that hold earlier tokens; with grow 8 their scales grow."""
    s = setup(case, grow=grow)
    print(case, grow, flush=True)
    held = s["held"]
    before = numbers(held.k), numbers(held.v), held.scales.cpu().double()
    q = append(s, case)
    check_append(s, case, before, q)


def test_append_drops_what_is_outside_and_takes_a_row_back():
    code, block = torch.int8, 16
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(3, 40, 2, 64, generator=g) for _ in range(2))
    held = pipeline.byte_cache(3, 50, 2, 64, block, code, DEV)
    starts = torch.tensor([30, -7, 1 << 30], dtype=torch.int32)
    pipeline.byte_append(held, k.to(DEV), v.to(DEV), starts.to(DEV))
    got = pipeline.byte_values(held, dtype=torch.float32)[0].cpu()
    lim = held.scales.cpu()[..., 0].repeat_interleave(block, 1)[:, :50, :, None] * (0.5 + 2.0 ** -9)
    want = torch.zeros(3, 50, 2, 64)
    want[0, 30:] = k[0, :20]
    want[1, :33] = k[1, 7:]
    assert ((got - want).abs() <= lim).all() and (got[2] == 0).all() and (got[0, :30] == 0).all()
    # row 0 again, from position 33 on, in smaller numbers: its block forgets the larger ones
    pipeline.byte_append(held, 1e-3 * k[:1, :4].to(DEV).expand(3, -1, -1, -1), 1e-3 * v[:, :4].to(DEV),
                         torch.tensor([33, 0, 0], dtype=torch.int32, device=DEV), torch.tensor([4, 0, 0], device=DEV))
    again = pipeline.byte_values(held, dtype=torch.float32)[0].cpu()
    assert ((again[0, 33:37] - 1e-3 * k[0, :4]).abs() <= (0.5 + 2.0 ** -9) * held.scales.cpu()[0, 2, :, 0, None]).all()
    assert torch.equal(again[0, 30:32], got[0, 30:32]) and torch.equal(again[1], got[1])


def test_dropped_tokens_have_no_part_in_a_scale():
    """Past a dense cache's end, past a table's width, past a pool's end: inside a block that is written to."""
    k = torch.ones(1, 16, 1, 64, device=DEV)
    k[:, 4:] = 100.0
    zero = torch.zeros(1, dtype=torch.int32, device=DEV)
    dense = pipeline.byte_cache(1, 20, 1, 64, 16, torch.int8, DEV)
    pipeline.byte_append(dense, k, k, zero + 16)
    pool = pipeline.byte_cache(1, 20, 1, 64, 16, torch.int8, DEV)
    pipeline.byte_append(pool, k, k, zero, slot_table=torch.arange(16, 32, dtype=torch.int32, device=DEV)[None])
    table = pipeline.byte_cache(1, 32, 1, 64, 16, torch.int8, DEV)
    pipeline.byte_append(table, k, k, zero + 16, slot_table=torch.arange(20, dtype=torch.int32, device=DEV)[None])
    for cache in (dense, pool, table):
        got = pipeline.byte_values(cache, dtype=torch.float32)[0][0, :, 0]
        assert (got[16:20] == 1).all() and (got[:16] == 0).all() and (got[20:] == 0).all()
        assert abs(float(cache.scales[0, 1, 0, 0]) - 1 / 127) <= 2.0 ** -20 / 127


def test_threads_on_one_stream():
    """Reads of two threads on one stream, of sizes that grow its scratch."""
    import threading

    held = cached(torch.float8_e4m3fn, 16, 1, 5000, 2, 64)
    g = torch.Generator().manual_seed(13)
    calls = []
    for n in range(2):
        q = torch.randn(1, 3 + n, 8, 64, generator=g).to(torch.bfloat16).to(DEV)
        ids = torch.randint(0, 5000, (1, 3 + n, 4000), generator=g).to(torch.int32).to(DEV)
        lens = torch.full((1, 3 + n), 4000 - n, dtype=torch.int32, device=DEV)
        calls.append((q, ids, lens, pipeline.byte_read(q, held, ids, lens)))
    torch.cuda.synchronize()
    bad = []

    def work(q, ids, lens, want):
        for _ in range(50):
            if not torch.equal(pipeline.byte_read(q, held, ids, lens), want):
                bad.append(1)

    threads = [threading.Thread(target=work, args=c) for c in calls]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


def test_append_with_bad_slots():
    """Blocks whose slot is missing, past the pool, negative or no multiple of the block are dropped; so are
    rows of a slot table that does not have them."""
    block, page = 16, 16
    held = pipeline.byte_cache(1, 64, 1, 64, block, torch.int8, DEV)
    table = torch.arange(96, dtype=torch.int32).view(1, 96).repeat(2, 1)
    table[0, 16:32] = -1
    table[0, 32:48] = 1 << 20
    table[0, 48:64] = torch.arange(16) + 8
    k = torch.ones(3, 96, 1, 64, device=DEV)
    pipeline.byte_append(held, k, k, torch.zeros(3, dtype=torch.int32, device=DEV), slot_table=table.to(DEV),
                         slot_rows=torch.tensor([0, 5, -1], dtype=torch.int32, device=DEV))
    got = pipeline.byte_values(held, dtype=torch.float32)[0].cpu().view(64, 64)
    assert (got[:16] == 1).all() and (got[16:] == 0).all()


@pytest.mark.parametrize("code", BOTH)
def test_append_of_nan_and_infinities(code):
    k = torch.ones(1, 3, 1, 64)
    k[0, 0, 0, :3] = torch.tensor([math.nan, math.inf, -math.inf])
    k[0, 1] = 0.0
    held = pipeline.byte_cache(1, 16, 1, 64, 1, code, DEV)
    pipeline.byte_append(held, k.to(DEV), torch.zeros_like(k).to(DEV), torch.zeros(1, dtype=torch.int32, device=DEV))
    got = pipeline.byte_values(held, dtype=torch.float32)[0].cpu()[0, :3, 0]
    assert (got[0, 3:] == 1).all() and (got[2] == 1).all() and (got[1] == 0).all()
    assert got[0, 0].isnan() if code == torch.float8_e4m3fn else got[0, 0] == 0
    assert got[0, 1] == 1 and got[0, 2] == -1  # the largest codes


def test_append_of_numbers_of_any_size():
    """Scales from the least one (2^-100) to the largest that fp32 holds."""
    for size in (1e-44, 1e-38, 1e-31, 1e-20, 1.0, 1e20, 3e38):
        k = torch.linspace(-1, 1, 64, dtype=torch.float64).mul(size).float().view(1, 1, 1, 64)
        held = pipeline.byte_cache(1, 1, 1, 64, 1, torch.int8, DEV)
        pipeline.byte_append(held, k.to(DEV), k.to(DEV), torch.zeros(1, dtype=torch.int32, device=DEV))
        got, scale = pipeline.byte_values(held, dtype=torch.float32)[0].cpu().view(-1), held.scales.cpu()[0, 0, 0, 0].double()
        top = k.abs().max().double()
        assert abs(scale - max(top / 127, 2.0 ** -100)) <= 2.0 ** -22 * scale
        assert ((got.double() - k.view(-1).double()).abs() <= (0.5 + 2.0 ** -20) * scale).all()


def cached(code, block, batch, rows, Hkv, D, seed=0, nan=False):
    """A cache of random codes and scales. nan: e4m3's NaN in row 3, NaN and infinite scales in the last block."""
    g = torch.Generator().manual_seed(seed)
    held = pipeline.byte_cache(batch, rows, Hkv, D, block, code, DEV)
    raw = torch.randint(0, 256, (2, *held.k.shape), generator=g).to(torch.uint8)
    raw[(raw & 127) == 127] = 0x31
    raw[raw == 128] = 0x31
    if code == torch.float8_e4m3fn:  # most of e4m3's random codes are tiny: the larger ones
        raw = (raw & 0x80) | 0x40 | (raw & 0x1F)
        if nan:
            raw[:, :, 3] = 0x7F
    held.k.copy_(raw[0].view(code)), held.v.copy_(raw[1].view(code))
    top = 2.0 / MOST[code] if code == torch.int8 else 0.25
    held.scales.copy_(top * (0.5 + torch.rand(held.scales.shape, generator=g)))
    if nan:
        held.scales[:, -1] = math.nan
        held.scales[:, -1, :, 1] = math.inf
    return held


READS = [
    # dtype, code, block, B, Tq, Hq, Hkv, D, rows, W, per_head, pool
    (torch.bfloat16, torch.int8, 64, 1, 1, 32, 8, 128, 4000, 700, True, False),
    (torch.bfloat16, torch.float8_e4m3fn, 16, 1, 1, 32, 8, 128, 4000, 1500, True, False),
    (torch.bfloat16, torch.float8_e4m3fn, 64, 5, 1, 8, 2, 128, 300, 129, False, False),
    (torch.bfloat16, torch.int8, 1, 3, 2, 4, 1, 64, 100, 33, False, True),
    (torch.bfloat16, torch.int8, 32, 2, 3, 6, 2, 256, 200, 400, True, True),
    (torch.bfloat16, torch.float8_e4m3fn, 8, 2, 1, 16, 1, 32, 90, 257, False, False),
    (torch.bfloat16, torch.int8, 64, 70, 5, 8, 8, 128, 200, 31, False, True),
    (torch.float16, torch.float8_e4m3fn, 16, 1, 4, 17, 1, 128, 500, 1000, False, False),
    (torch.float16, torch.int8, 2, 4, 1, 40, 2, 64, 64, 64, True, False),
    (torch.float16, torch.int8, 64, 1, 1, 64, 1, 256, 3000, 2500, False, False),
    (torch.float16, torch.float8_e4m3fn, 4, 600, 1, 4, 4, 32, 70, 65, True, True),
    (torch.float32, torch.int8, 16, 2, 1, 8, 2, 128, 400, 333, True, False),
    (torch.float32, torch.float8_e4m3fn, 64, 1, 1, 3, 1, 64, 20, 1, False, False),
    (torch.float32, torch.int8, 1, 3, 7, 5, 5, 32, 33, 50, False, True),
    (torch.float32, torch.float8_e4m3fn, 32, 1, 2, 8, 1, 256, 800, 640, False, False),
]


def lists(case, seed):
    """Lists with -1, repeated and out-of-range ids, rows 3 and the last block unlisted, every third list empty."""
    dtype, code, block, B, Tq, Hq, Hkv, D, rows, W, per_head, pool = case
    rng = np.random.default_rng(seed)
    lead = (B, Tq, Hkv) if per_head else (B, Tq)
    n = int(np.prod(lead))
    most = max((rows - 1) // block * block, 1)
    ids = rng.integers(0, most, (n, W)).astype(np.int32)
    ids[ids == 3] = 0
    ids[:, 2::7] = -1
    ids[::5, 0] = rows + 2
    ids[1::5, 0] = -(1 << 31)
    ids[2::5, 0] = (1 << 31) - 1
    lens = rng.integers(0, W + 1, n).astype(np.int32)
    lens[::3] = W
    if n > 1:
        lens[1::3] = 0
    return torch.from_numpy(ids.reshape(*lead, W)), torch.from_numpy(lens.reshape(lead))


def exact(q, held, ids, lens, scale):
    B, Tq, Hq, D = q.shape
    Hkv = held.k.shape[2]
    G = Hq // Hkv
    kc, vc, sc = numbers(held.k), numbers(held.v), held.scales.cpu().double()
    out = torch.zeros(q.shape, dtype=torch.float64)
    vmax = torch.zeros(B, Tq, Hq, 1, dtype=torch.float64)
    for b in range(B):
        c = b if kc.shape[0] == B else 0
        for t in range(Tq):
            for g in range(Hkv):
                at = (ids[b, t, g] if ids.dim() == 4 else ids[b, t])[: int(lens[b, t, g] if ids.dim() == 4 else lens[b, t])].long()
                at = at[(at >= 0) & (at < kc.shape[1])]
                if not len(at):
                    continue
                s = sc[c, at // held.block, g]
                k, v = kc[c, at, g] * s[:, :1], vc[c, at, g] * s[:, 1:]
                h = slice(g * G, (g + 1) * G)
                out[b, t, h] = torch.softmax(scale * (q[b, t, h].double() @ k.T), 1) @ v
                vmax[b, t, h] = v.abs().max()
    return out, vmax


def check_read(got, ref, vmax, dtype):
    half = torch.finfo(dtype).eps / 2
    bound = half * ref.abs() + (2.0 ** -13 + (2.0 ** -16 if dtype != torch.float32 else 0.0)) * vmax
    off = (got.double().cpu() - ref).abs()
    assert (off <= bound).all(), f"off by {(off / bound)[bound > 0].max():.2f} of the bound"


@pytest.mark.parametrize("case", READS, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_read(case):
    dtype, code, block, B, Tq, Hq, Hkv, D, rows, W, per_head, pool = case
    held = cached(code, block, 1 if pool else B, rows, Hkv, D, nan=rows > 2 * block)
    q = torch.randn(B, Tq, Hq, D, generator=torch.Generator().manual_seed(5)).to(dtype)
    ids, lens = lists(case, 7)
    print(case, flush=True)
    got = pipeline.byte_read(q.to(DEV), held, ids.to(DEV), lens.to(DEV))
    check_read(got, *exact(q, held, ids, lens, D ** -0.5), dtype)
    assert torch.equal(got, pipeline.byte_read(q.to(DEV), held, ids.to(DEV), lens.to(DEV)))


@pytest.mark.parametrize("code", BOTH)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_read_of_one_key_returns_its_value(dtype, code):
    """One key, or one that outweighs the others: its value, rounded once."""
    held = cached(code, 16, 1, 64, 2, 128)
    q = torch.randn(1, 3, 4, 128, generator=torch.Generator().manual_seed(5)).to(dtype).to(DEV)
    ids = torch.tensor([[[5], [-1], [63]]], dtype=torch.int32, device=DEV)
    got = pipeline.byte_read(q, held, ids, torch.ones(1, 3, dtype=torch.int32, device=DEV))
    v = pipeline.byte_values(held, dtype=torch.float32)[1]
    for t, row in ((0, 5), (2, 63)):
        want = v[0, row].repeat_interleave(2, 0)
        off = (got[0, t].float() - want).abs()
        assert (off <= (torch.finfo(dtype).eps / 2 + 2.0 ** -16) * want.abs()).all()
    assert (got[0, 1] == 0).all()


def test_read_scales_of_any_sign_and_large_scores():
    """A negative and a zero scale, and scores in the thousands."""
    held = cached(torch.int8, 16, 2, 100, 1, 64)
    g = torch.Generator().manual_seed(6)
    q = torch.randn(2, 1, 4, 64, generator=g).to(torch.bfloat16)
    ids = torch.randint(0, 100, (2, 1, 80), generator=g).to(torch.int32)
    lens = torch.tensor([[80], [41]], dtype=torch.int32)
    for scale in (-0.125, 0.0):
        check_read(pipeline.byte_read(q.to(DEV), held, ids.to(DEV), lens.to(DEV), scale=scale),
                   *exact(q, held, ids, lens, scale), torch.bfloat16)
    ref, vmax = exact(q, held, ids, lens, 100.0)
    got = pipeline.byte_read(q.to(DEV), held, ids.to(DEV), lens.to(DEV), scale=100.0).double().cpu()
    # scores to 2^13 and more in fp32: each is off by 2^-10 of itself at most, a weight by a factor e^8
    assert torch.isfinite(got).all() and (got.abs() <= vmax * (1 + 2.0 ** -7)).all()


def test_views_of_a_wider_cache():
    """K and V side by side in one buffer, a slice of its heads."""
    wide = torch.randint(0, 120, (2, 80, 2, 6, 64), dtype=torch.int8, generator=torch.Generator().manual_seed(1)).to(DEV)
    held = pipeline.ByteCache(wide[:, :, 0, 1:4], wide[:, :, 1, 1:4], torch.rand(2, 5, 3, 2, device=DEV) * 0.01, 16)
    q = torch.randn(2, 1, 6, 64, generator=torch.Generator().manual_seed(5)).to(torch.bfloat16)
    ids = torch.arange(80, dtype=torch.int32).flip(0).expand(2, 1, 80).contiguous()
    lens = torch.tensor([[80], [33]], dtype=torch.int32)
    check_read(pipeline.byte_read(q.to(DEV), held, ids.to(DEV), lens.to(DEV)), *exact(q, held, ids, lens, 64 ** -0.5),
               torch.bfloat16)
    kv = torch.randn(2, 7, 3, 64, device=DEV)
    rest = wide.clone()
    pipeline.byte_append(held, kv, kv, torch.tensor([3, 60], dtype=torch.int32, device=DEV))
    rest[:, :, :, 1:4] = wide[:, :, :, 1:4]
    assert torch.equal(rest, wide)  # its neighbours are left alone
    got = pipeline.byte_values(held, dtype=torch.float32)[1]
    lim = held.scales[..., 1].repeat_interleave(16, 1)[..., None] * (0.5 + 2.0 ** -9)
    for b, p in ((0, 3), (1, 60)):
        assert ((got[b, p:p + 7] - kv[b]).abs() <= lim[b, p:p + 7]).all()


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("code", BOTH)
@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_values(code, D, out):
    held = cached(code, 16, 3, 75, 2, D, seed=D)
    want = [numbers(c) * held.scales.cpu().double()[..., i].repeat_interleave(16, 1)[:, :75, :, None] for i, c in
            enumerate((held.k, held.v))]
    half = torch.finfo(out).eps / 2
    for got, ref in zip(pipeline.byte_values(held, dtype=out), want):
        assert ((got.double().cpu() - ref).abs() <= half * ref.abs() + torch.finfo(out).tiny).all()
    ids = torch.tensor([[74, 0, -1, 75, 5], [1, 1, 1, 1, 1], [9, 8, 7, 6, 5]], dtype=torch.int32)
    lens = torch.tensor([5, 0, 9], dtype=torch.int32)
    for got, ref in zip(pipeline.byte_values(held, ids.to(DEV), lens.to(DEV), out), want):
        assert got.shape == (3, 5, 2, D) and (got[1] == 0).all() and (got[0, 2:4] == 0).all()
        at = ref[torch.arange(3)[:, None], ids.long().clamp(0, 74)]
        off = (got.double().cpu() - at).abs() <= half * at.abs() + torch.finfo(out).tiny
        assert off[0, [0, 1, 4]].all() and off[2].all()


def test_offsets_past_32_bits():
    """A pool of 5 GB a side: rows a megabyte apart."""
    rows, step = 5000, 1 << 20
    k8, v8 = (torch.empty(rows * step, dtype=torch.int8, device=DEV).as_strided((1, rows, 1, 64), (0, step, 64, 1))
              for _ in range(2))
    held = pipeline.ByteCache(k8, v8, torch.zeros(1, -(-rows // 8), 1, 2, device=DEV), 8)
    g = torch.Generator().manual_seed(4)
    k, v = (torch.randn(1, rows, 1, 64, generator=g).to(torch.bfloat16) for _ in range(2))
    pipeline.byte_append(held, k.to(DEV), v.to(DEV), torch.zeros(1, dtype=torch.int32, device=DEV))
    got = pipeline.byte_values(held, dtype=torch.float32)
    for i, (x, y) in enumerate(((got[0], k), (got[1], v))):
        lim = held.scales[..., i].repeat_interleave(8, 1)[..., None].cpu() * (0.5 + 2.0 ** -9)
        assert ((x.cpu() - y.float()).abs() <= lim).all()
    q = torch.randn(1, 1, 2, 64, generator=g).to(torch.bfloat16)
    ids = torch.arange(rows, dtype=torch.int32).flip(0).view(1, 1, -1)
    lens = torch.tensor([[rows]], dtype=torch.int32)
    plain = pipeline.ByteCache(k8.contiguous(), v8.contiguous(), held.scales, 8)
    got = pipeline.byte_read(q.to(DEV), held, ids.to(DEV), lens.to(DEV))
    assert torch.equal(got, pipeline.byte_read(q.to(DEV), plain, ids.to(DEV), lens.to(DEV)))
    check_read(got, *exact(q, plain, ids, lens, 0.125), torch.bfloat16)


def test_graphs_and_streams():
    """Two graphs captured on one stream, replayed on two at once, and eager calls between them."""
    held = cached(torch.int8, 16, 2, 3000, 2, 128)
    g = torch.Generator().manual_seed(9)
    qs = [torch.randn(2, 1, 8, 128, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2)]
    ids = torch.randint(0, 3000, (2, 1, 2, 2000), generator=g).to(torch.int32).to(DEV)
    lens = torch.tensor([2000, 1, 0, 777], dtype=torch.int32, device=DEV).view(2, 1, 2)
    stream, graphs, outs = torch.cuda.Stream(), [], []
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for q in qs:
            pipeline.byte_read(q, held, ids, lens)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                outs.append(pipeline.byte_read(q, held, ids, lens))
            graphs.append(graph)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(4):
        for q in qs:
            q.mul_(0.9)
        torch.cuda.synchronize()
        for st, graph in zip(streams, graphs):
            with torch.cuda.stream(st):
                graph.replay()
        eager = [pipeline.byte_read(q, held, ids, lens) for q in qs]
        torch.cuda.synchronize()
        for q, o, e in zip(qs, outs, eager):
            want = exact(q.cpu(), held, ids.cpu(), lens.cpu(), 128 ** -0.5)
            check_read(o, *want, torch.bfloat16)
            check_read(e, *want, torch.bfloat16)


def test_append_and_read_in_a_graph():
    """A captured decode step whose starts grow in place, replayed; every replay as the eager step."""
    caches = [pipeline.byte_cache(2, 64, 2, 64, 16, torch.float8_e4m3fn, DEV) for _ in range(2)]
    g = torch.Generator().manual_seed(11)
    kv = torch.randn(2, 1, 2, 64, generator=g).to(torch.bfloat16).to(DEV)
    q = torch.randn(2, 1, 4, 64, generator=g).to(torch.bfloat16).to(DEV)
    freq, starts = pipeline.rotary_frequencies(64, device=DEV), torch.tensor([0, 5], dtype=torch.int32, device=DEV)
    ids = torch.arange(64, dtype=torch.int32, device=DEV).expand(2, 1, 64).contiguous()

    def step(cache):
        turned_q = pipeline.byte_append(cache, kv, kv, starts, q=q, frequencies=freq)
        return pipeline.byte_read(turned_q, cache, ids, (starts + 1)[:, None])

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(caches[0])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = step(caches[0])
    torch.cuda.synchronize()
    step(caches[1])
    for i in range(30):
        kv.mul_(1.1 if i % 2 else -0.95)
        starts.add_(1)
        graph.replay()
        eager = step(caches[1])
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        assert torch.equal(caches[0].k.view(torch.uint8), caches[1].k.view(torch.uint8))
        assert torch.equal(caches[0].scales, caches[1].scales)


def test_a_run_of_them():
    """A prompt into a paged 8-bit cache, an index over what it holds, decode steps that append, select and read."""
    B, T, Hq, Hkv, D, page, block = 2, 600, 8, 2, 64, 32, 16
    g = torch.Generator().manual_seed(12)
    table, rows = paged(B, 700, page, g)
    held = pipeline.byte_cache(1, rows, Hkv, D, block, torch.int8, DEV)
    wide = torch.randn(B, T, Hq + 2 * Hkv, D, generator=g).to(torch.bfloat16).to(DEV)
    freq, wk = pipeline.rotary_frequencies(D, device=DEV), torch.ones(D, device=DEV)
    slots = table.to(DEV)
    pipeline.byte_append(held, wide[:, :, Hq:Hq + Hkv], wide[:, :, Hq + Hkv:], torch.zeros(B, dtype=torch.int32, device=DEV),
                         slot_table=slots, frequencies=freq, k_weight=wk)
    keys, _ = pipeline.byte_values(held, slots[:, :T].contiguous())
    _, k_turned = pipeline.rotate(wide[:, :, :Hq], wide[:, :, Hq:Hq + Hkv], torch.arange(T, device=DEV), freq, k_weight=wk)
    # a key's norm is sqrt(D) and no element of it above 8, so its step is at most 8 / 127: 0.5 + the two bf16 roundings
    assert (keys.float() - k_turned.float()).abs().max() <= 0.5 * 8 / 127 + 2 * 8 * 2.0 ** -8
    buckets = pipeline.segment_buckets(keys, 16)
    config = pipeline.PortConfig(top_p=6, top_k=512, window_size=64, sink_size=4)
    for n in range(T, T + 3):
        new = torch.randn(B, 1, Hq + 2 * Hkv, D, generator=g).to(torch.bfloat16).to(DEV)
        starts = torch.full((B,), n, dtype=torch.int32, device=DEV)
        q = pipeline.byte_append(held, new[:, :, Hq:Hq + Hkv], new[:, :, Hq + Hkv:], starts, slot_table=slots, q=new[:, :, :Hq],
                                 frequencies=freq, k_weight=wk)
        ids, lens = pipeline.flat_select(pipeline.index_queries(q, Hkv)[:, 0], starts, buckets, config, slot_table=slots)
        got = pipeline.byte_read(q, held, ids[:, None], lens[:, None])
        assert int(lens.min()) >= 68
        check_read(got, *exact(q.cpu(), held, ids[:, None].cpu(), lens[:, None].cpu(), D ** -0.5), torch.bfloat16)
        k16, v16 = (x.view(1, rows, Hkv, D) for x in pipeline.byte_values(held, dtype=torch.bfloat16))
        near = pipeline.lsa_read(q, k16, v16, ids[:, None], lens[:, None], D ** -0.5)
        assert (near.float() - got.float()).abs().max() <= 2.0 ** -5 * float(v16.abs().max())


def test_empty_calls():
    held = pipeline.byte_cache(0, 16, 2, 64, 16, torch.int8, DEV)
    kv = torch.empty(0, 3, 2, 64, device=DEV)
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    pipeline.byte_append(held, kv, kv, none)
    assert pipeline.byte_values(held)[0].shape == (0, 16, 2, 64)
    assert pipeline.byte_read(kv, held, none.view(0, 3, 0), none.view(0, 3)).shape == kv.shape
    held = pipeline.byte_cache(1, 0, 2, 64, 16, torch.int8, DEV)  # a cache of no tokens
    kv = torch.ones(1, 3, 2, 64, device=DEV)
    pipeline.byte_append(held, kv, kv, torch.zeros(1, dtype=torch.int32, device=DEV))
    ids = torch.zeros(1, 3, 4, dtype=torch.int32, device=DEV)
    assert (pipeline.byte_read(kv, held, ids, torch.full((1, 3), 4, device=DEV)) == 0).all()
    held = cached(torch.int8, 16, 1, 16, 2, 64)
    assert (pipeline.byte_read(kv, held, ids[..., :0], torch.full((1, 3), 4, device=DEV)) == 0).all()
    assert module.ByteCache is pipeline.ByteCache
