"""prefix_read, key_mass and the evictions among a program's other calls."""

import pytest
import torch

import test_gpu_prefix as prefix
from lsa_rocm_lab import _abi
from lsa_rocm_lab.port import eviction, pipeline

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rows_and_lists(dtype=torch.float32, B=3, Tq=1, Hq=8, Hkv=2, D=64, T=900, W=300, pool=False, seed=0):
    """q, K (a cache a row, or one pool) and lists, on the GPU."""
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(B, Tq, Hq, D, generator=g).to(dtype)
    k = torch.randn(1 if pool else B, T, Hkv, D, generator=g).to(dtype)
    ids = torch.randint(0, T, (B, Tq, W), generator=g, dtype=torch.int32)
    lens = torch.randint(1, W + 1, (B, Tq), generator=g, dtype=torch.int32)
    return [x.to(DEV) for x in (q, k, ids, lens)]


def test_words_a_decode_left_in_its_counters():
    """What a decode that gave up waiting may leave there changes no weight and no read."""
    q, k, ids, lens = rows_and_lists()
    steps = (lambda: pipeline.key_mass(q, k, ids, lens), lambda: pipeline.prefix_read(q, k[:1], k[:1], k, k, ids, lens))
    clean = [step() for step in steps]
    words = _abi.Counters.get(q.device, 4096)
    try:
        words.fill_(1)
        for step, want in zip(steps, clean):
            for _ in range(2):
                assert torch.equal(step(), want)
        assert (words == 1).all()
    finally:
        words.zero_()


@pytest.mark.parametrize("Tq,W", [(1, 64), (2, 64), (64, 4096)])
@pytest.mark.parametrize("pool", [False, True])
def test_weights_by_an_lse_that_is_too_low(Tq, W, pool):
    """A weight is at most 1, and no sum of such wraps: a key that fills every list of every row is the heaviest."""
    q, k, ids, lens = rows_and_lists(torch.bfloat16, 2, Tq, 16, 2, 64, 5, W, pool)
    k.zero_()
    ids.fill_(3)
    ids[:, :, 1::4] = 1
    lens.fill_(W)
    got = pipeline.key_mass(q, k, ids, lens, lse=torch.full((2, Tq, 16), -40.0, device=DEV))
    n = (2 if pool else 1) * Tq * W * 8  # whole numbers, exact in fp32
    assert got.shape == (1 if pool else 2, 2, 5)
    assert (got == torch.tensor([0.0, n / 4, 0.0, n * 3 / 4, 0.0], device=DEV)).all()


def test_a_slot_table_that_is_a_column_turned():
    q, pool, _, _ = rows_and_lists(torch.bfloat16, T=128, pool=True)
    v = pool * 2
    column = torch.randperm(128, device=DEV).to(torch.int32)[:90, None]
    assert torch.equal(pipeline.prefix_read(q, pool, v, prefix_slots=column.t()),
                       pipeline.prefix_read(q, pool, v, prefix_slots=column.flatten()[None].clone()))


def test_numbers_past_32_bits():
    """An id, slot, prefix or length that int32 does not hold: outside everything, as its int64 value is."""
    q, k, ids, lens = rows_and_lists(torch.bfloat16, T=200, W=40)
    far = torch.where(torch.arange(40, device=DEV) % 3 == 0, ids.long() + (1 << 32), ids.long())
    near = torch.where(far < 200, far, -1).to(torch.int32)
    assert torch.equal(pipeline.key_mass(q, k, far, lens), pipeline.key_mass(q, k, near, lens))
    rows = torch.tensor([0, 1 << 32, 1], device=DEV)  # the second: none
    args = (k[:2], k[:2] * 2, k, k)
    lengths = torch.tensor([(1 << 32) + 7, 90], device=DEV)
    assert torch.equal(
        pipeline.prefix_read(q, *args, far, lens.long(), prefix_rows=rows, prefix_lengths=lengths),
        pipeline.prefix_read(q, *args, near, lens, prefix_rows=rows.clamp(max=9).int(), prefix_lengths=lengths.clamp(max=200).int()))
    table = torch.arange(200, device=DEV)[None].expand(2, 200).clone()
    mass = torch.rand(1, 2, 200, device=DEV)
    none = table.clone()
    table[:, 5::9] += 1 << 32
    none[:, 5::9] = -1
    kept = pipeline.evict_slots(table, mass, 60, lens[:2].flatten().long() + (1 << 32))[2]
    assert torch.equal(kept, pipeline.evict_slots(none, mass, 60)[2])


@pytest.mark.parametrize("B,Tq,pool", [(13, 1, False), (13, 1, True), (5, 6, False), (5, 6, True)])
def test_key_weights_in_slabs_of_the_batch(monkeypatch, B, Tq, pool):
    """Batch rows that go through a few at a time: the same weights (where rows share a cache, sums in another order:
    2^-24 a step of an fp32 sum, and 2^-45 a weight)."""
    q, k, ids, lens = rows_and_lists(torch.bfloat16, B, Tq, pool=pool, seed=3)
    lse = torch.full((B, Tq, 8), 9.0, device=DEV)
    for wide in (None, lse):
        mass = torch.full((1 if pool else B, 2, 900), 0.5, device=DEV)
        whole = pipeline.key_mass(q, k, ids, lens, lse=wide), pipeline.key_mass(q, k, ids, lens, lse=wide, mass=mass.clone())
        for rows in (1, 3):
            monkeypatch.setattr(eviction, "_SLAB_BYTES", rows * (4 * 8 * 300 + (2 * 8 * 2 * 900 if Tq > 1 and not pool else 0)))
            got = pipeline.key_mass(q, k, ids, lens, lse=wide), pipeline.key_mass(q, k, ids, lens, lse=wide, mass=mass.clone())
            monkeypatch.undo()
            for x, y in zip(got, whole):
                if Tq == 1 and not pool:
                    assert torch.equal(x, y)
                else:
                    assert ((x.double() - y.double()).abs() <= B * Tq * (2.0 ** -23 * y.double() + 8 * 2.0 ** -44)).all()


SPREADS = {
    "one": lambda P, B: torch.full((B,), P - 2),
    "one and none": lambda P, B: torch.where(torch.arange(B) % 3 == 0, -1, P - 2),
    "two": lambda P, B: torch.where(torch.arange(B) % 5 == 0, 1, P - 1),
    "few": lambda P, B: (P * torch.linspace(0, 0.99, B) ** 5).long(),
    "none": lambda P, B: torch.full((B,), P),
}


@pytest.mark.parametrize("dtype,B,Tq,P,Tp,Hq,Hkv,D,paged", [
    (torch.bfloat16, 8, 1, 8, 2100, 8, 2, 128, 0),
    (torch.bfloat16, 40, 2, 30, 1500, 4, 1, 64, 16),   # several column blocks of one prefix
    (torch.float16, 6, 1, 1100, 600, 2, 1, 64, 16),    # past the first thousand
    (torch.float16, 70, 3, 5, 900, 8, 1, 128, 0),      # wide columns
    (torch.bfloat16, 5, 1, 2, 33000, 4, 1, 64, 0),     # 128 pieces
    (torch.bfloat16, 8, 1, 8, 9000, 8, 8, 64, 0),      # 4 pieces if the rows are spread, 32 if they crowd
    (torch.float16, 40, 2, 100, 2700, 8, 8, 64, 16),   # 1 or 10
    (torch.bfloat16, 150, 1, 30, 1100, 16, 4, 128, 0),  # 2 or 3, of several blocks
    (torch.float16, 30, 1, 200, 60, 4, 2, 64, 0),      # one piece at most, past the first 64
])
def test_rows_that_crowd_on_few_of_many_prefixes(dtype, B, Tq, P, Tp, Hq, Hkv, D, paged):
    """However the rows are spread, eagerly and from one graph whose rows change between replays."""
    c = prefix.make(dtype, B, Tq, P, Tp, Hq, Hkv, D, 20, 5, paged=paged, seed=61)
    c["plen"][1], c["plen"][P - 2:] = Tp // 3, Tp - 1
    t = {n: c[n].to(DEV) for n in ("q", "kp", "vp", "k", "v", "ids", "lens", "plen", "prow")}
    slots = prefix.dev(c["slots"])

    def step():
        return pipeline.prefix_read(t["q"], t["kp"], t["vp"], t["k"], t["v"], t["ids"], t["lens"], prefix_lengths=t["plen"],
                                    prefix_rows=t["prow"], prefix_slots=slots, return_lse=True)

    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for name, spread in SPREADS.items():
        print("crowd", dtype, B, Tq, P, Tp, name, flush=True)
        c["prow"] = spread(P, B).int()
        t["prow"].copy_(c["prow"])
        exact = prefix.want(c)
        eager = step()
        prefix.compare(eager, exact, c)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], eager[0]) and torch.equal(out[1], eager[1])
