"""Calls of rotate, byte_append and byte_read that are all edge, as far as the host goes: nothing is launched."""

import ctypes

import pytest
import torch

from lsa_rocm_lab import _abi
from lsa_rocm_lab.port import byte_cache as module
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


def read_call(B, Tq, Hq, Hkv, D, W, per_head, pool):
    """byte_read of lists in host memory that nothing reads, and its tensors."""
    T = 64
    k, v = (fake(torch.zeros(1, 1, Hkv, D, dtype=torch.int8).expand(1 if pool else B, T, Hkv, D)) for _ in range(2))
    held = pipeline.ByteCache(k, v, fake(torch.zeros(k.shape[0], 4, Hkv, 2)), 16)
    held.k, held.v = (fake(torch.empty(k.shape, dtype=torch.int8)) for _ in range(2))
    lead = (B, Tq, Hkv) if per_head else (B, Tq)
    q, ids, lens = (fake(torch.empty(*s, dtype=t)) for s, t in (((B, Tq, Hq, D), torch.bfloat16), ((*lead, W), torch.int32),
                                                                (lead, torch.int32)))
    return q, held, ids, lens, pipeline.byte_read(q, held, ids, lens)


@pytest.mark.parametrize("B,Tq,Hq,Hkv,D,W,per_head,pool", [
    (1, 32768, 32, 8, 128, 4612, False, True),    # a 32k prompt: 262 144 units of 3 spans, 1.6 GB in one piece
    (8, 1024, 16, 8, 128, 32768, False, False),   # whole caches, 1024 rows of each
    (2, 4100, 128, 8, 128, 4612, True, False),
    (300, 17, 16, 1, 256, 9000, False, True),
])
def test_scratch_of_a_read_of_many_rows_is_bounded(calls, host, B, Tq, Hq, Hkv, D, W, per_head, pool):
    """256 MB of partials at most, in slabs that cover every query row once."""
    def copied(name, *args):  # with the cache as it is at the call
        calls.append((name, args, module._Cache.from_buffer_copy(ctypes.cast(args[1], ctypes.POINTER(module._Cache)).contents)))

    host.setattr(_abi, "call_in_order", copied)
    q, held, ids, lens, out = read_call(B, Tq, Hq, Hkv, D, W, per_head, pool)
    assert len(calls) > 1 and {name for name, *_ in calls} == {"lsa_byte_read"}
    size = q.element_size() * Hq * D
    lists = Hkv if per_head else 1
    scales = held.scales[0].numel() * 4
    done = 0
    for _, args, c in calls:
        q_at, _, _, b, t, *_ = args
        splits, nbytes, out_at = args[13], args[16], args[17]
        assert nbytes <= 256 << 20 and splits == calls[0][1][13] > 1
        n = b * t
        assert q_at == q.data_ptr() + done * size and out_at == out.data_ptr() + done * size
        assert args[8] == ids.data_ptr() + 4 * done * lists * W and args[9] == lens.data_ptr() + 4 * done * lists
        at = 0 if pool else done // Tq
        assert c.caches == (1 if pool else b) and (pool or t == Tq or b == 1)
        assert c.k == held.k.data_ptr() + at * held.k.stride(0) and c.scales == held.scales.data_ptr() + at * scales
        assert c.v == held.v.data_ptr() + at * held.v.stride(0)
        done += n
    assert done == B * Tq


def test_small_reads_are_one_call(calls):
    read_call(32, 1, 32, 8, 128, 4612, True, False)
    read_call(16, 1, 32, 8, 128, 32768, False, True)
    assert [args[3:5] for _, args in calls] == [(32, 1), (16, 1)]


def test_every_span_of_a_read_has_slots():
    """Spans are whole steps of 128 slots; as many are asked for as that leaves."""
    for units in (1, 8, 31, 160, 255, 256, 1000, 40000, 1 << 22):
        for width in (0, 1, 191, 192, 384, 577, 1300, 2816, 4612, 6336, 9001, 32768, 131072, 1 << 30):
            splits = module._read_splits(units, width)
            span = max(-(-(-(-width // splits)) // 128) * 128, 128)  # as the kernel cuts
            assert 1 <= splits <= 64 and (splits - 1) * span < max(width, 1)
    assert module._read_splits(8, 2816) == 11 and module._read_splits(128, 32768) == 20
