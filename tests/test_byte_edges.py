"""Calls of rotate, byte_append and byte_read that are all edge, as far as the host goes: nothing is launched."""

import pytest
import torch

from lsa_rocm_lab.port import pipeline
from test_serving_memory import calls, fake, host  # noqa: F401 (fixtures)


def test_rotate_of_keys_alone(calls):
    """No query heads: the keys are normed and rotated all the same."""
    q, k = fake(torch.ones(2, 3, 0, 64)), fake(torch.ones(2, 3, 2, 64))
    pos, freq, w = fake(torch.arange(3)), fake(torch.ones(32)), fake(torch.ones(64))
    got = pipeline.rotate(q, k, pos, freq, k_weight=w)
    assert got[0].shape == q.shape and got[1].shape == k.shape
    (name, args), = calls
    assert name == "lsa_rotate" and args[0] == k.data_ptr() and args[5:8] == (2, 0, 64) and args[-3] == got[1].data_ptr()
    for empty in ((q, None), (q, fake(torch.ones(2, 3, 0, 64))), (fake(torch.ones(0, 3, 4, 64)), fake(torch.ones(0, 3, 2, 64)))):
        pipeline.rotate(*empty, pos, freq)
    assert len(calls) == 1
    with pytest.raises(ValueError, match="norm weights"):
        pipeline.rotate(q, k, pos, freq, q_weight=fake(torch.ones(32)))


def test_append_without_kv_heads_is_refused(calls):
    """A cache of no kv-heads takes nothing, and q is not handed back unwritten."""
    held = pipeline.ByteCache(*(fake(torch.zeros(2, 32, 0, 64, dtype=torch.int8)) for _ in range(2)),
                              fake(torch.zeros(2, 2, 0, 2)), 16)
    kv, starts = fake(torch.ones(2, 3, 0, 64)), fake(torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="kv-head"):
        pipeline.byte_append(held, kv, kv, starts, q=fake(torch.ones(2, 3, 4, 64)))
    assert not calls
