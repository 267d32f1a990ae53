"""prefix_read, key_mass and the evictions among a program's other calls."""

import pytest
import torch

from lsa_rocm_lab import _abi
from lsa_rocm_lab.port import pipeline

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
