"""What prefix_read, key_mass and the evictions hand their kernels: host logic, nothing is launched."""

import numpy as np
import pytest
import torch

from lsa_rocm_lab import _abi
from lsa_rocm_lab.port import eviction, pipeline, shared_prefix

GPU = torch.device("cuda", 0)


@pytest.fixture
def host(monkeypatch):
    """Buffers in host memory where a call asks for the device's; one stream, no capture."""
    for name in ("zeros", "empty"):
        make = getattr(torch, name)
        monkeypatch.setattr(torch, name, lambda *a, _make=make, device=None, **k: _make(*a, **k))
    monkeypatch.setattr(_abi, "_raw_stream", lambda index=None: 7)
    monkeypatch.setattr(_abi, "_capturing", lambda: False)
    for cls in (_abi.Workspace, _abi.Counters):
        monkeypatch.setattr(cls, "_buffers", {})
        monkeypatch.setattr(cls, "_retired", [])
    return monkeypatch


def test_counters_are_not_the_decodes(host):
    """A fused decode that gave up waiting may leave words in its counters; the calls around it, which do
    not ask whether one did, find theirs zero."""
    decode = _abi.Counters.get(GPU, 64)
    decode.fill_(3)
    for purpose in ("key_mass", "prefix_read"):
        _, counters, _ = _abi.call_memory(GPU, purpose, 16, 64)
        assert counters.data_ptr() != decode.data_ptr() and not counters.any()
        assert _abi.call_memory(GPU, purpose, 16, 64)[1] is counters  # kept from call to call
        assert _abi.call_memory(GPU, purpose, 16, 5000)[1].numel() >= 5000
    assert _abi.Counters.get(GPU, 64) is decode
    _abi.Counters.reset(GPU)
    assert not decode.any()


class OnGpu(torch.Tensor):
    """A CPU tensor that says it is on the GPU."""

    device = GPU


def fake(x):
    return x.as_subclass(OnGpu)


@pytest.fixture
def calls(host):
    """What the entry points are called with, in order; nothing is launched."""
    seen = []
    host.setattr(_abi, "current_device", lambda: 0)
    host.setattr(_abi, "call_in_order", lambda name, *args: seen.append((name, args)))
    host.setattr(_abi, "call", lambda name, *args: seen.append((name, args)))
    return seen


def test_a_slot_table_of_one_row_with_any_stride(calls):
    """A row axis of one has whatever stride its view left it; the table is dense all the same."""
    q, pool = fake(torch.zeros(2, 1, 4, 64)), fake(torch.zeros(1, 80, 2, 64))
    column = torch.arange(64, dtype=torch.int32)[:, None]
    for slots in (column.t(), column.t().contiguous().as_strided((1, 64), (1, 1))):
        pipeline.prefix_read(q, pool, pool, prefix_slots=fake(slots))
        name, args = calls.pop()
        assert name == "lsa_prefix_read" and args[6:8] == (1, 64)
        assert args[18] >= 64, "slot rows closer than their length are refused"


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32, torch.int16, torch.uint8])
def test_numbers_past_32_bits_stay_outside(dtype):
    """2^32 + 5 is no key, slot or prefix 5: numbers that int32 does not hold become its ends, which name nothing."""
    small = torch.tensor([[0, 5, 100]], dtype=dtype)
    assert shared_prefix.int32_on(small, small.device).tolist() == [[0, 5, 100]]
    if dtype == torch.uint8:
        assert shared_prefix.int32_on(torch.tensor([2 ** 32 - 1], dtype=torch.uint32), small.device).tolist() == [2 ** 31 - 1]
    if dtype == torch.int64:
        far = torch.tensor([2 ** 32 + 5, 2 ** 31, -(2 ** 31) - 1, -(2 ** 32) + 5, 2 ** 63 - 1, 2 ** 31 - 1, -1])
        got = shared_prefix.int32_on(far, far.device)
        top = 2 ** 31 - 1
        assert got.dtype == torch.int32 and got.tolist() == [top, top, -top - 1, -top - 1, top, top, -1]


def places(t):
    """The bytes that a tensor's elements lie at."""
    at = torch.tensor([t.data_ptr()])
    for n, step in zip(t.shape, t.stride()):
        at = (at[:, None] + torch.arange(n) * step * t.element_size()).flatten()
    return set((at[:, None] + torch.arange(t.element_size())).flatten().tolist())


def test_buffers_of_an_eviction_that_share_memory(calls):
    """K, V and mass to be filled: refused where two of them share a place among the rows that are written,
    taken where they lie between each other."""
    B, T, Hkv, D, budget = 2, 20, 2, 16, 6
    k = fake(torch.zeros(B, T, Hkv, D, dtype=torch.bfloat16))
    seen = fake(torch.zeros(B, Hkv, T))
    arena = torch.zeros(40000, dtype=torch.bfloat16)
    floats = arena.view(torch.float32)
    token, head = Hkv * D, D

    def rows(at, step=(9 * token, token, head), n=budget):
        return arena.as_strided((B, n, Hkv, D), (*step, 1), at)

    def masses(at, step=(Hkv * budget, budget)):
        return floats.as_strided((B, Hkv, budget), (*step, 1), at // 2)

    apart = masses(30000)
    wide = (100 * token, 2 * token, 2 * head)  # K and V of a head side by side
    byhead = (1000, D, 400)                    # head by head: K, V and masses in turn
    tried = {True: 0, False: 0}
    for k2, v2, m2 in [
        (rows(0), rows(5000), apart),
        (rows(0), rows(token), apart),                      # V a row behind K
        (rows(0), rows(5 * token), apart), (rows(0), rows(6 * token), apart), (rows(6 * token), rows(0), apart),
        (rows(0), rows(16 * token), apart), (rows(0), rows(17 * token), apart),
        (rows(0), rows(8), apart), (rows(8), rows(0), apart),
        (rows(0, wide), rows(D, wide), apart), (rows(0, wide), rows(8, wide), apart),
        (rows(0, wide), rows(token, wide), apart), (rows(0, wide), rows(2 * token, wide), apart),
        (rows(0, byhead), rows(D * budget, byhead), masses(2 * D * budget, (500, 200))),
        (rows(0, byhead), rows(D * budget, byhead), masses(2 * D * budget - 2, (500, 200))),
        (rows(0, byhead), rows(D * budget, byhead), masses(400 - 2 * budget, (500, 200))),
        (rows(0, byhead), rows(D * budget, byhead), masses(402 - 2 * budget, (500, 200))),
        (rows(0), rows(5000), masses(0)), (rows(0), rows(5000), masses(5000 + 100)),
        (rows(0), rows(5000), masses(6 * token)), (rows(0), rows(5000), masses(6 * token - 2)),
        (rows(0, n=9), rows(6 * token, n=9), masses(5000)),  # rows behind the budget are not written
    ]:
        k3, v3 = k2[:, :budget], v2[:, :budget]
        share = bool(places(k3) & places(v3) or places(k3) & places(m2) or places(v3) & places(m2))
        tried[share] += 1
        out = tuple(map(fake, (k2, v2, m2)))
        if share:
            with pytest.raises(ValueError, match="place of their own"):
                eviction.evict(k, k, seen, budget, out=out)
            assert not calls
        else:
            eviction.evict(k, k, seen, budget, out=out)
            assert [name for name, _ in calls] == ["lsa_evict_keep", "lsa_evict_rows"]
            calls.clear()
    assert min(tried.values()) >= 7


def test_shared_places_by_enumeration():
    """Nested views at random: whether they share a byte, against the bytes themselves."""
    rng = np.random.default_rng(0)
    arena = torch.zeros(4000, dtype=torch.float32)
    found = {True: 0, False: 0}
    for _ in range(1500):
        shape, steps, reach = [], [], 1
        for n in rng.integers(1, 5, 3).tolist():
            step = reach + int(rng.integers(0, 3)) * int(rng.integers(1, 4))
            shape.append(n), steps.append(step)
            reach = step * n
        turn = rng.permutation(3).tolist()
        view = lambda at: arena.as_strided([shape[i] for i in turn], [steps[i] for i in turn], at)  # noqa: B023, E731
        k, v = view(500), view(500 + int(rng.integers(-reach, reach)))
        assert eviction._apart(k)
        share = bool(places(k) & places(v))
        found[share] += 1
        assert eviction._meets_twin(k, v) == share == eviction._meets_twin(v, k)
        lo = k.data_ptr() + int(rng.integers(-20, 4 * reach))
        hi = lo + int(rng.integers(0, 40))
        assert eviction._meets(k, lo, hi) == any(lo <= x < hi for x in places(k))
    assert min(found.values()) > 300


@pytest.mark.parametrize("B,Tq,Hq,Hkv,T,W,pool,fresh", [
    (40, 1, 8, 2, 50, 30, False, True),      # rows of a decode batch, each with its cache
    (40, 1, 8, 2, 50, 30, True, True),       # over one pool
    (40, 1, 8, 2, 50, 30, True, False),
    (5, 7, 8, 2, 50, 30, False, True),
    (5, 7, 8, 2, 50, 30, True, False),
    (6, 3, 8, 2, 3000, 4, False, False),     # the integers of several rows' caches are most of it
    (1, 9, 8, 2, 40, 200, False, True),
    (3, 2, 8, 2, 40, 2000, False, True),     # one row's scores are more than a slab
    (2, 2, 8, 2, 10, 5, False, True),
])
def test_key_weights_in_slabs_of_memory(calls, B, Tq, Hq, Hkv, T, W, pool, fresh):
    """Every query row once, each slab of memory within the limit unless one query row's scores are more."""
    limit = 30000
    calls_of = eviction._SLAB_BYTES
    assert calls_of == 256 << 20
    q, k = fake(torch.zeros(B, Tq, Hq, 64)), fake(torch.zeros(1 if pool else B, T, Hkv, 64))
    ids, lens = fake(torch.zeros(B, Tq, W, dtype=torch.int32)), fake(torch.zeros(B, Tq, dtype=torch.int32))
    caches = k.shape[0]
    mass = None if fresh else fake(torch.zeros(caches, Hkv, T))
    eviction._SLAB_BYTES = limit
    try:
        got = pipeline.key_mass(q, k, ids, lens, mass=mass)
    finally:
        eviction._SLAB_BYTES = calls_of
    rows = []
    for name, a in calls:
        b, n, c = a[3], a[4], a[5]
        assert name == "lsa_key_mass" and a[6:10] == (T, Hq, Hkv, 64) and c == (1 if pool else b)
        at = (a[1] - k.data_ptr()) // (T * Hkv * 64 * 4)  # the slab's first cache
        assert (a[23] - got.data_ptr()) == at * Hkv * T * 4
        nbytes = a[22]
        whole = 8 * Hkv * T if b * n > 1 and c == 1 else 0  # the integers of one cache, whatever the slab
        sums = 8 * Hq * b * n * -(-W // 128)                # of spans of fp32 keys of 64
        assert nbytes - whole - sums <= limit + 64 or b * n == 1
        rows.append((at, b, n, a[19]))
    if pool:
        assert sum(b * n for _, b, n, _ in rows) == B * Tq
        assert [z for *_, z in rows] == [int(fresh)] + [0] * (len(rows) - 1)
    else:
        for cache in range(B):
            mine = [(n, z) for at, b, n, z in rows if at <= cache < at + b]
            assert sum(n for n, _ in mine) == Tq
            assert [z for _, z in mine] == [int(fresh)] + [0] * (len(mine) - 1)
    assert len(rows) == 1 or 4 * B * Tq * Hq * W + (0 if pool or Tq == 1 else 8 * B * Hkv * T) > limit


@pytest.mark.parametrize("B", [8, 32, 256])
@pytest.mark.parametrize("P", [8, 32, 2000])
def test_room_for_a_prefix_that_every_row_reads(B, P):
    """However many prefixes the table holds: where all rows read one of them it is cut into as many pieces
    as fill the chip (256 workgroups of 32 or more columns), so there is room for their partials."""
    need = _abi.size("lsa_prefix_read_scratch_bytes", _abi.LSA_BF16, B, 1, P, 32768, 32, 8, 128, 0)
    columns = -(-B // min(B, P)) * 4  # a prefix, if the rows are spread
    blocks = -(-B * 4 // next(n for n in (32, 64, 128, 256) if columns <= n or n == 256))
    pieces = max(1, 256 // (8 * blocks))
    assert need >= B * 8 * pieces * 4 * (128 + 2) * 4


def test_counters_that_creep_up(host):
    """Outgrown counters are kept for graphs that hold them: a buffer at least doubles, so they stay few."""
    for n in range(4000, 40000, 500):
        assert _abi.call_memory(GPU, "prefix_read", 0, n)[1].numel() >= n
    assert sum(x.numel() for x in _abi.Counters._retired) < 2 * 40000
