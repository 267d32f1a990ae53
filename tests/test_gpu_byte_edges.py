"""Calls of rotate and of the 8-bit cache that are all edge, vs 64 bits or the ordinary call."""

import math

import pytest
import torch

from lsa_rocm_lab.port import byte_cache as module
from lsa_rocm_lab.port import pipeline

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotate_of_keys_alone(interleaved):
    """No query heads: the keys come out as they do beside some."""
    g = torch.Generator().manual_seed(1)
    q, k = (torch.randn(2, 5, n, 64, generator=g).to(torch.bfloat16).to(DEV) for n in (4, 2))
    w = torch.rand(2, 64, generator=g).add(0.5).to(DEV)
    rest = torch.arange(7, 12, device=DEV), pipeline.rotary_frequencies(64, device=DEV), w[0], w[1]
    want = pipeline.rotate(q, k, *rest, interleaved=interleaved)[1]
    none, got = pipeline.rotate(q[:, :, :0], k, *rest, interleaved=interleaved)
    assert none.shape == (2, 5, 0, 64) and torch.equal(got, want)


CODES = [torch.int8, torch.float8_e4m3fn]


def held(code, block, rows, seed=0, batch=1):
    """A cache whose rows hold numbers of N(0, 1), and those numbers as it holds them."""
    g = torch.Generator().manual_seed(seed)
    cache = pipeline.byte_cache(batch, rows, 2, 64, block, code, DEV)
    kv = torch.randn(2, batch, rows, 2, 64, generator=g).to(DEV)
    pipeline.byte_append(cache, kv[0], kv[1], torch.zeros(batch, dtype=torch.int32, device=DEV),
                         slot_table=None if batch > 1 else torch.arange(rows, dtype=torch.int32, device=DEV)[None])
    return cache, pipeline.byte_values(cache, dtype=torch.float32)


def slots(*pieces):
    return torch.cat([torch.arange(a, b) if b >= a else torch.arange(a, b, -1) for a, b in pieces]).to(torch.int32)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("block,table,start,n", [
    # the block's first slots are whole, its own first position's is not where the new token goes
    (16, slots((32, 40), (64, 96)), 8, 3),
    # aligned where the block begins, another row's in the middle: a new token there, one before it, one behind it
    (16, slots((16, 24), (90, 98)), 10, 2),
    (16, slots((16, 20), (90, 94), (24, 32)), 9, 5),
    (16, slots((16, 24), (90, 98)), 2, 3),
    # given-up rows at the end of an evicted table: half a block, the other half of it is kept elsewhere
    (32, slots((0, 32), (64, 80), (96, 112)), 32, 1),
    (64, slots((64, 128), (0, 32), (33, 65)), 64, 20),
    # whole slots, in the wrong order
    (8, slots((23, 15),), 0, 8),
    (2, slots((1, 3), (5, 3)), 0, 4),
])
def test_append_leaves_blocks_that_a_table_does_not_map_whole(code, block, table, start, n):
    """Slots permuted token by token, as an evicted table's are: where a block of positions is no block of the pool
    nothing is written, so no other key changes."""
    cache, before = held(code, block, 128, seed=block)
    k = 100.0 * torch.randn(1, n, 2, 64, generator=torch.Generator().manual_seed(2)).to(DEV)
    raw = [x.clone() for x in (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.scales)]
    pipeline.byte_append(cache, k, k, torch.tensor([start], dtype=torch.int32, device=DEV), slot_table=table[None].to(DEV))
    for x, y in zip((cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.scales), raw):
        assert torch.equal(x, y)


def test_append_writes_the_whole_blocks_of_such_a_table():
    """The blocks beside them are written, and a table that ends inside a block."""
    cache, before = held(torch.int8, 16, 96)
    table = slots((80, 96), (3, 19), (32, 48), (64, 70))  # whole, not, whole, whole as far as it goes
    k = torch.randn(1, 54, 2, 64, generator=torch.Generator().manual_seed(2)).to(DEV)
    pipeline.byte_append(cache, k, -k, torch.zeros(1, dtype=torch.int32, device=DEV), slot_table=table[None].to(DEV))
    got = pipeline.byte_values(cache, dtype=torch.float32)
    lim = (0.5 + 2.0 ** -9) * cache.scales.repeat_interleave(16, 1)
    rest = torch.ones(96, dtype=torch.bool, device=DEV)
    for at, row, m in ((0, 80, 16), (32, 32, 16), (48, 64, 6)):
        rest[row:row + 16] = False
        for i, x in enumerate((k, -k)):
            assert ((got[i][0, row:row + m] - x[0, at:at + m]).abs() <= lim[0, row:row + m, :, i, None]).all()
    assert all(torch.equal(x[0, rest], y[0, rest]) for x, y in zip(got, before))


def test_append_through_a_table_that_is_filled_token_by_token():
    """Entries behind the new tokens that name no row yet (negative, past the pool) are no matter."""
    got = []
    for rest in (None, -1, 64, (1 << 31) - 1, -(1 << 31)):
        cache = held(torch.int8, 16, 64)[0]
        table = slots((48, 64), (16, 32))
        k = torch.randn(1, 9, 2, 64, generator=torch.Generator().manual_seed(2)).to(DEV)
        for t in range(9):
            now = table.clone()
            if rest is not None:
                now[13 + t + 1:] = rest
            pipeline.byte_append(cache, k[:, t:t + 1], -k[:, t:t + 1], torch.tensor([13 + t], dtype=torch.int32, device=DEV),
                                 slot_table=now[None].to(DEV))
        got.append((cache.k, cache.v, cache.scales))
    values = pipeline.byte_values(cache, table[None].to(DEV), dtype=torch.float32)[0]
    assert ((values[0, 21] - k[0, 8]).abs() <= (0.5 + 2.0 ** -9) * cache.scales[0, 1, :, 0, None]).all()  # the last one
    assert all(torch.equal(x, y) for other in got[1:] for x, y in zip(other, got[0]))


def test_append_through_an_evicted_table_of_single_rows():
    """With a block a row any table serves: the new tokens land in the rows given up, the kept ones stay."""
    cache, before = held(torch.int8, 1, 64)
    mass = torch.rand(1, 2, 64, generator=torch.Generator().manual_seed(5)).to(DEV)
    table, lens, kept = pipeline.evict_slots(torch.arange(64, dtype=torch.int32, device=DEV)[None], mass, 40, window=4)
    k = 100.0 * torch.randn(1, 5, 2, 64, generator=torch.Generator().manual_seed(2)).to(DEV)
    pipeline.byte_append(cache, k, k, lens, slot_table=table)
    got = pipeline.byte_values(cache, table, lens + 5, dtype=torch.float32)
    at = kept[0].long()
    for i in range(2):
        assert torch.equal(got[i][0, :40], before[i][0, at])
        assert ((got[i][0, 40:45] - k[0]).abs() <= (0.5 + 2.0 ** -9) * cache.scales[0, table[0, 40:45].long(), :, i, None]).all()


@pytest.mark.parametrize("B,Tq,per_head,pool,dtype", [
    (1, 50, False, True, torch.bfloat16), (3, 7, True, True, torch.float16), (5, 4, False, False, torch.bfloat16),
    (3, 20, True, False, torch.float32), (37, 1, True, False, torch.bfloat16),
])
def test_read_in_slabs(monkeypatch, B, Tq, per_head, pool, dtype):
    """Query rows that go through in slabs: the bits of one piece, eagerly and in a graph."""
    g = torch.Generator().manual_seed(B)
    rows, W = 3000, 1300
    cache, _ = held(torch.int8, 16, rows, batch=1 if pool else B)
    q = torch.randn(B, Tq, 6, 64, generator=g).to(dtype).to(DEV)
    lead = (B, Tq, 2) if per_head else (B, Tq)
    ids = torch.randint(-1, rows, (*lead, W), generator=g).to(torch.int32).to(DEV)
    lens = torch.randint(0, W + 1, lead, generator=g).to(torch.int32).to(DEV)
    want = pipeline.byte_read(q, cache, ids, lens)
    one = module._abi.size("lsa_byte_read_scratch_bytes", 1, 6, 2, 64, module._read_splits(B * Tq * 2, W))
    assert one > 0
    for slab in (1, 3 * one, 11 * one + 5, (B * Tq - 1) * one):
        monkeypatch.setattr(module, "_SLAB_BYTES", slab)
        assert torch.equal(pipeline.byte_read(q, cache, ids, lens), want)
    monkeypatch.setattr(module, "_SLAB_BYTES", 3 * one)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
        out = pipeline.byte_read(q, cache, ids, lens)
    torch.cuda.synchronize()
    for _ in range(3):
        q.mul_(-1.0)
        graph.replay()
        monkeypatch.setattr(module, "_SLAB_BYTES", 1 << 28)
        eager = pipeline.byte_read(q, cache, ids, lens)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


@pytest.mark.parametrize("code", CODES)
def test_block_that_is_filled_token_by_token(code):
    """Each time its scale grows a block's codes are rounded again. int8: a token written before g growths is off by
    (g + 1) / 2 steps of the last scale, 2^-9 of a step more each time for the quotient. e4m3: by half a step of the
    code each time, which is 2^-3 of its power of two (at least 2^-9) and grows with what it is off by already."""
    B, T, D = 6, 64, 64
    g = torch.Generator().manual_seed(4)
    k = torch.randn(B, T, 2, D, generator=g)
    k[3:] *= 1.03 ** torch.arange(T).view(T, 1, 1)  # many tokens grow the scale
    k[5] = k[5].abs().clamp(max=1.0) * 1.03 ** torch.arange(T).view(T, 1, 1)  # every token does
    cache = pipeline.byte_cache(B, T, 2, D, 64, code, DEV)
    kd = k.to(DEV)
    scales = []
    for t in range(T):
        pipeline.byte_append(cache, kd[:, t:t + 1], kd[:, t:t + 1], torch.full((B,), t, dtype=torch.int32, device=DEV))
        scales.append(cache.scales[:, 0, :, 0].clone())
    scales = torch.stack(scales, 1).double().cpu()  # [B, T, 2] after each token
    assert (scales[:, 1:] >= scales[:, :-1]).all()
    x, half = k.double(), 0.5 + 2.0 ** -9
    lim = torch.zeros_like(x)
    for t in range(T):  # what tokens 0 .. t are off by at most after append t
        s = scales[:, t, None, :, None]
        again = torch.ones(B, t + 1, 2, 1, dtype=torch.bool)  # rounded by this append
        if t:
            again[:, :t] = (scales[:, t] > scales[:, t - 1])[:, None, :, None]
        step = s
        if code == torch.float8_e4m3fn:
            _, e = torch.frexp((x[:, :t + 1].abs() + lim[:, :t + 1]) / s)
            step = torch.exp2((e - 4).clamp(-9, 5).double()) * s
        lim[:, :t + 1] += torch.where(again, half * step, 0.0)
    grown = (scales[:, 1:] > scales[:, :-1]).sum(1)
    top = k.abs().amax(-1).cummax(1).values
    assert torch.equal(grown, (top[:, 1:] > top[:, :-1]).sum(1)) and (grown[5] == T - 1).all()
    got = pipeline.byte_values(cache, dtype=torch.float32)[0].double().cpu()
    off = (got - x).abs()
    assert (off <= lim).all(), f"off by {(off / lim).max():.2f} of the bound"
    last = scales[:, -1, None, :, None]
    print(f"{code}: grown {grown.tolist()}, off by {(off / last).amax((1, 2, 3)).tolist()} of the last scale, "
          f"rms {((off / last).square().mean((1, 2, 3)).sqrt() / (1 / 12) ** 0.5).tolist()} of one rounding's")
    bulk = pipeline.byte_cache(B, T, 2, D, 64, code, DEV)
    pipeline.byte_append(bulk, kd, kd, torch.zeros(B, dtype=torch.int32, device=DEV))
    assert torch.equal(bulk.scales, cache.scales)
    print("in one append: rms", [float(((pipeline.byte_values(bulk, dtype=torch.float32)[0].double().cpu() - x) / last)[b]
                                       .square().mean().sqrt() / (1 / 12) ** 0.5) for b in range(B)])


@pytest.mark.parametrize("code", CODES)
def test_a_weight_times_a_scale_keeps_24_bits_for_fp32_rows(code):
    """One key weighs 1, so the output is its code times V's scale: exact in three parts of 8 bits, whose products
    add up in two roundings of 2^-24. Two parts would be off by up to 2^-17."""
    cache, _ = held(code, 1, 500)
    cache.scales.copy_(0.5 + torch.rand(cache.scales.shape, generator=torch.Generator().manual_seed(8)))
    q = torch.randn(1, 500, 4, 64, generator=torch.Generator().manual_seed(9)).to(DEV)
    ids = torch.arange(500, dtype=torch.int32, device=DEV).view(1, 500, 1)
    got = pipeline.byte_read(q, cache, ids, torch.ones(1, 500, dtype=torch.int32, device=DEV))
    want = (cache.v.float().double() * cache.scales[..., 1:].double()).repeat_interleave(2, 2)
    assert ((got.double() - want).abs() <= 2.0 ** -22 * want.abs()).all()


@pytest.mark.parametrize("dtype,low", [(torch.float32, 2.0 ** -18), (torch.float16, 2.0 ** -9)])
def test_q_enters_exactly(dtype, low):
    """q's elements differ in their last part of 8 bits alone: 1 + 2^-9 + 2^-18 and -(1 + 2^-9 - 2^-18) in fp32, 1 + 2^-9
    and -(1 - 2^-9) in fp16. Against keys of 64 and of -64 every product and every sum of them is a multiple of 2^-12
    under 2^13: exact. The score is 64 low of a product that is 0 without that part; its exponential, the weights'
    sum, the products with V (1 and -1) and the division take eight roundings or so of 2^-24."""
    D = 128
    a = 1.0 + (2.0 ** -9 if dtype == torch.float32 else 0.0)
    row = torch.tensor([a + low, -(a - low)], dtype=torch.float64).repeat(D // 2)
    q = row.to(dtype).view(1, 1, 1, D)
    assert torch.equal(q.double().view(-1), row)
    signs = torch.tensor([64, -64], dtype=torch.int8).view(1, 2, 1, 1).expand(1, 2, 1, D).contiguous().to(DEV)
    scales = torch.tensor([1.0, 2.0 ** -6]).expand(1, 2, 1, 2).contiguous().to(DEV)
    cache = pipeline.ByteCache(signs, signs.clone(), scales, 1)
    ids = torch.tensor([0, 1], dtype=torch.int32, device=DEV).view(1, 1, 2)
    got = pipeline.byte_read(q.to(DEV), cache, ids, torch.tensor([[2]], device=DEV), scale=2.0 ** -7).double().cpu()
    want = math.tanh(64 * low)
    assert ((got - want).abs() <= torch.finfo(dtype).eps / 2 * want + 2.0 ** -20).all() and want > 2.0 ** -12.1


def test_read_of_scores_in_the_thousands():
    """By the scores' own error: a matrix instruction adds 32 exact products (and what came before) with four roundings
    of 2^-24 of their magnitudes or fewer, D / 32 of them follow each other, and the scale takes two more. A weight is
    then off by e^(2 d), the output by 2 d of the largest value; 2^-15 of it are the weights' parts and the sums."""
    D, n = 64, 80
    cache, _ = held(torch.int8, 16, 100, seed=3)
    g = torch.Generator().manual_seed(6)
    q = torch.randn(1, 9, 4, D, generator=g).to(torch.bfloat16)
    ids = torch.randint(0, 100, (1, 9, n), generator=g).to(torch.int32)
    k, v = (c.float().double().cpu() * cache.scales[..., i, None].double().cpu().repeat_interleave(16, 1)[:, :100]
            for i, c in enumerate((cache.k, cache.v)))
    got = pipeline.byte_read(q.to(DEV), cache, ids.to(DEV), torch.full((1, 9), n, device=DEV), scale=100.0).double().cpu()
    for t in range(9):
        for h in range(4):
            x, kk, vv = q[0, t, h].double(), k[0, ids[0, t].long(), h // 2], v[0, ids[0, t].long(), h // 2]
            s = 100.0 * kk @ x
            assert s.abs().max() > 1000
            d = (D / 32 * 2.0 ** -22 + 2.0 ** -23) * 100.0 * (kk.abs() @ x.abs()).max()
            want = torch.softmax(s, 0) @ vv
            lim = 2.0 ** -8 * want.abs() + (torch.expm1(2 * d) + 2.0 ** -15) * vv.abs().max()
            assert ((got[0, t, h] - want).abs() <= lim).all()


def test_threads_whose_reads_grow_the_scratch():
    """Four threads on one stream that has none yet, each with reads of growing size: the results of another stream."""
    import threading

    cache, _ = held(torch.float8_e4m3fn, 16, 5000)
    g = torch.Generator().manual_seed(13)
    calls = []
    for n in range(4):
        for rows in (1, 3, 17, 60, 150):
            q = torch.randn(1, rows + n, 8, 64, generator=g).to(torch.bfloat16).to(DEV)
            ids = torch.randint(0, 5000, (1, rows + n, 4000), generator=g).to(torch.int32).to(DEV)
            lens = torch.full((1, rows + n), 4000 - n, dtype=torch.int32, device=DEV)
            calls.append((n, q, ids, lens, pipeline.byte_read(q, cache, ids, lens)))
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    for kind in (module._abi.Workspace, module._abi.Counters):
        kind._buffers.pop((q.device.index, stream.cuda_stream, "byte_read"), None)
    bad, start = [], threading.Barrier(4)

    def work(me):
        start.wait()
        with torch.cuda.stream(stream):
            for n, q, ids, lens, want in calls:
                if n == me and not torch.equal(pipeline.byte_read(q, cache, ids, lens), want):
                    bad.append(me)

    before = len(module._abi.Workspace._retired)
    threads = [threading.Thread(target=work, args=(n,)) for n in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    torch.cuda.synchronize()
    assert not bad and len(module._abi.Workspace._retired) > before
