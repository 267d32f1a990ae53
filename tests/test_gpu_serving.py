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
