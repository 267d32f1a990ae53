"""What prefix_read, key_mass and the evictions hand their kernels: host logic, nothing is launched."""

import pytest
import torch

from lsa_rocm_lab import _abi
from lsa_rocm_lab.port import pipeline, shared_prefix

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
