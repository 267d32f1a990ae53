"""What prefix_read, key_mass, evict and evict_slots refuse, on the host before any launch."""

import pytest
import torch

from lsa_rocm_lab import _abi
from lsa_rocm_lab.port import eviction, pipeline, shared_prefix

BF16, P = _abi.LSA_BF16, 4096  # P: an aligned address that is never read


def prefix(**over):
    a = dict(q=P, kp=P, vp=P, dt=BF16, B=2, Tq=1, P=1, Tp=64, rows=64, Hq=8, Hkv=2, D=128, sb=0, st=256, sh=128, prow=None,
             plen=None, slots=None, slot_stride=0, k=P, v=P, Tk=32, kb=8192, kt=256, kh=128, ids=P, lens=P, W=4, per=0,
             scale=0.1, counters=None, ws=P, nbytes=1 << 40, out=P, lse=None, stream=None)
    a.update(over)
    return _abi.call("lsa_prefix_read", *a.values())


@pytest.mark.parametrize("over,match", [
    (dict(q=None), "NULL"), (dict(out=None), "NULL"), (dict(ids=None), "own lists"), (dict(dt=7), "dtype"),
    (dict(D=48), "LSA_ERR_SHAPE"), (dict(Hq=6), "LSA_ERR_SHAPE"), (dict(Hq=7), "LSA_ERR_SHAPE"), (dict(P=0), "prefixes"),
    (dict(Tp=-1), "LSA_ERR_SHAPE"), (dict(W=-1), "LSA_ERR_SHAPE"), (dict(rows=63), "prefix cache"),
    (dict(slots=P, slot_stride=63), "slot rows"), (dict(slots=P, slot_stride=64, rows=0), "slot rows"),
    (dict(q=P + 8), "aligned"), (dict(kt=257), "aligned"), (dict(st=100), "apart"), (dict(kh=64), "apart"),
    (dict(st=1 << 32), "strides past"), (dict(B=1 << 31), "LSA_ERR_SHAPE"),
])
def test_prefix_read_abi(over, match):
    with pytest.raises(ValueError, match=match):
        prefix(**over)


def test_prefix_read_of_several_prefixes_needs_their_rows():
    for over in (dict(P=3), dict(P=3, B=1)):
        with pytest.raises(ValueError, match="need prefix_rows"):
            prefix(**over)
    with pytest.raises(ValueError, match="LSA_ERR_SHAPE"):
        prefix(B=1 << 23)  # 2^24 rows of kv-heads


def test_prefix_read_needs_its_scratch():
    need = _abi.size("lsa_prefix_read_scratch_bytes", BF16, 2, 1, 1, 64, 8, 2, 128, 4)
    assert need > 0
    for over in (dict(ws=None), dict(nbytes=need - 1), dict(ws=P + 4)):
        with pytest.raises(_abi.LsaError, match="scratch"):
            prefix(**over)
    assert prefix(B=0) == 0 and _abi.size("lsa_prefix_read_scratch_bytes", BF16, 0, 1, 1, 64, 8, 2, 128, 4) == 0


def mass(**over):
    a = dict(q=P, k=P, dt=BF16, B=2, Tq=1, caches=2, Tk=32, Hq=8, Hkv=2, D=128, sb=8192, st=256, sh=128, ids=P, lens=P, W=4,
             per=0, scale=0.1, lse=None, zero=0, counters=None, ws=P, nbytes=1 << 40, mass=P, mb=64, mh=32, stream=None)
    a.update(over)
    return _abi.call("lsa_key_mass", *a.values())


@pytest.mark.parametrize("over,match", [
    (dict(k=None), "NULL"), (dict(mass=None), "NULL"), (dict(dt=5), "dtype"), (dict(D=80), "LSA_ERR_SHAPE"),
    (dict(Hq=24), "LSA_ERR_SHAPE"), (dict(caches=3), "LSA_ERR_SHAPE"), (dict(q=P + 2), "aligned"), (dict(st=260), "aligned"),
    (dict(sh=64), "apart"), (dict(zero=1, mh=40), "dense"), (dict(Tk=1 << 31), "LSA_ERR_SHAPE"),
])
def test_key_mass_abi(over, match):
    with pytest.raises(ValueError, match=match):
        mass(**over)


def test_key_mass_of_too_many_rows():
    """Their sums, and a launch's threads, have limits."""
    for over in (dict(Tq=(1 << 17) + 1), dict(caches=1, Tq=(1 << 16) + 1), dict(B=1 << 23, caches=1 << 23)):
        with pytest.raises(ValueError, match="LSA_ERR_SHAPE"):
            mass(**over)
    assert _abi.size("lsa_key_mass_scratch_bytes", BF16, 2, 1 << 17, 2, 32, 8, 2, 128, 4) > 0


def test_key_mass_needs_its_scratch():
    need = _abi.size("lsa_key_mass_scratch_bytes", BF16, 2, 1, 2, 32, 8, 2, 128, 4)
    assert need > 0
    # several rows of one cache add up in integers beside the scores
    assert _abi.size("lsa_key_mass_scratch_bytes", BF16, 2, 1, 1, 32, 8, 2, 128, 4) >= need + 8 * 2 * 32
    for over in (dict(ws=None), dict(nbytes=need - 1)):
        with pytest.raises(_abi.LsaError, match="scratch"):
            mass(**over)
    for over in (dict(B=0, caches=1), dict(W=0), dict(Tk=0)):
        assert mass(**over) == 0


def keep(**over):
    a = dict(mass=P, B=2, Hkv=2, T=100, mb=200, mh=100, lens=None, budget=10, window=4, sink=2, shared=0, table=None,
             stride=0, pool=0, ws=P, nbytes=1 << 30, kept=P, new=P, new_table=None, new_stride=0, stream=None)
    a.update(over)
    return _abi.call("lsa_evict_keep", *a.values())


@pytest.mark.parametrize("over,match", [
    (dict(mass=None), "NULL"), (dict(kept=None), "NULL"), (dict(budget=0), "budget"), (dict(budget=101), "budget"),
    (dict(window=9), "fit the budget"), (dict(window=-1), "fit the budget"), (dict(sink=-1), "fit the budget"),
    (dict(B=70000), "rows"), (dict(T=0), "positions"), (dict(T=(1 << 30) + 1), "positions"), (dict(table=P, stride=100, pool=5), "come together"),
    (dict(table=P, new_table=P, stride=100, new_stride=100, pool=5), "shared"),
    (dict(table=P, new_table=P, stride=99, new_stride=100, pool=5, shared=1), "strides"),
])
def test_evict_keep_abi(over, match):
    with pytest.raises(ValueError, match=match):
        keep(**over)


def test_evict_scratch():
    size = lambda *a: _abi.size("lsa_evict_scratch_bytes", *a)  # noqa: E731
    assert size(3, 2, 100, 1) == 1200 and size(3, 2, 100, 0) == 0 and size(3, 2, 32768, 0) == 0 < size(3, 2, 32769, 0)
    for over in (dict(nbytes=799), dict(ws=None), dict(ws=P + 8)):
        with pytest.raises(_abi.LsaError, match="scratch"):
            keep(shared=1, **over)


def rows(**over):
    a = dict(k=P, v=P, mass=P, dt=BF16, B=2, T=100, Hkv=2, D=64, sb=12800, st=128, sh=64, mb=200, mh=100, kept=P, shared=0,
             budget=10, k2=P, v2=P, ob=1280, ot=128, oh=64, m2=P, m2b=20, m2h=10, zero=1, stream=None)
    a.update(over)
    return _abi.call("lsa_evict_rows", *a.values())


@pytest.mark.parametrize("over,match", [
    (dict(v2=None), "NULL"), (dict(dt=9), "dtype"), (dict(D=60), "aligned|apart"), (dict(st=32), "apart"),
    (dict(k=P + 4), "aligned"), (dict(ot=132), "aligned"), (dict(budget=101), "budget"), (dict(B=65536), "B 65536"),
])
def test_evict_rows_abi(over, match):
    with pytest.raises(ValueError, match=match):
        rows(**over)


class OnGpu(torch.Tensor):
    """A CPU tensor that says it is on the GPU: the Python checks run, and nothing is launched."""

    device = torch.device("cuda", 0)


def fake(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype).as_subclass(OnGpu)


def test_tensors_off_the_gpu_are_refused():
    x = torch.zeros(1, 4, 2, 64)
    i = torch.zeros(1, 1, 4, dtype=torch.int32)
    for f in (lambda: pipeline.prefix_read(x, x, x), lambda: pipeline.key_mass(x[:, :1], x, i, i[..., 0]),
              lambda: pipeline.evict(x, x, torch.zeros(1, 2, 4), 2),
              lambda: pipeline.evict_slots(i[0], torch.zeros(1, 2, 4), 1)):
        with pytest.raises(ValueError, match="ROCm kernel"):
            f()
    with pytest.raises(ValueError, match="one device"):
        pipeline.prefix_read(fake(1, 1, 2, 64), x, x)


def test_prefix_read_arguments():
    q, kp = fake(3, 1, 8, 64), fake(1, 20, 2, 64)
    k, ids, lens = fake(3, 9, 2, 64), fake(3, 1, 4, dtype=torch.int32), fake(3, 1, dtype=torch.int32)
    for args, kw, match in [
        ((q, kp, kp, k), {}, "come together"),
        ((q[0], kp, kp), {}, "q \\[B, Tq, Hq, D\\]"),
        ((q, kp, kp[:, :5]), {}, "prefixes"),
        ((q, fake(1, 20, 3, 64), fake(1, 20, 3, 64)), {}, "query heads"),
        ((q, fake(1, 20, 2, 32), fake(1, 20, 2, 32)), {}, "query heads"),
        ((q, fake(1, 20, 2, 64, dtype=torch.float16), kp), {}, "one dtype"),
        ((fake(3, 1, 8, 64, dtype=torch.float64), *[fake(1, 20, 2, 64, dtype=torch.float64)] * 2), {}, "unsupported dtype"),
        ((q, fake(2, 20, 2, 64), fake(2, 20, 2, 64)), {}, "prefix_rows is needed"),
        ((q, kp, kp), dict(prefix_rows=lens[:2]), "prefix rows for 3"),
        ((q, kp, kp), dict(prefix_lengths=lens[:2]), "prefix lengths for 1"),
        ((q, fake(2, 20, 2, 64), fake(2, 20, 2, 64)), dict(prefix_slots=ids[0]), "over one pool"),
        ((q, kp, kp, fake(2, 9, 2, 64), fake(2, 9, 2, 64), ids, lens), {}, "k/v must be"),
        ((q, kp, kp, k, k, ids, lens[:2]), {}, "do not match"),
    ]:
        with pytest.raises(ValueError, match=match):
            shared_prefix.prefix_read(*args, **kw)


def test_key_mass_arguments():
    q, k = fake(3, 1, 8, 64), fake(3, 9, 2, 64)
    ids, lens = fake(3, 1, 4, dtype=torch.int32), fake(3, 1, dtype=torch.int32)
    f32 = torch.float32
    for args, kw, match in [
        ((q, fake(2, 9, 2, 64), ids, lens), {}, "key_mass: q"),
        ((q, fake(3, 9, 2, 64, dtype=torch.float16), ids, lens), {}, "dtypes differ"),
        ((q, fake(3, 9, 3, 64), ids, lens), {}, "do not group"),
        ((q, k, ids, lens[:1]), {}, "do not match"),
        ((q, k, ids, lens), dict(lse=fake(3, 1, 8)), "lse must be fp32"),
        ((q, k, ids, lens), dict(lse=fake(3, 8, dtype=f32)), "lse must be fp32"),
        ((q, k, ids, lens), dict(mass=fake(3, 2, 8, dtype=f32)), "mass must be fp32"),
        ((q, k, ids, lens), dict(mass=fake(3, 2, 9)), "mass must be fp32"),
        ((q, k, ids, lens), dict(mass=fake(3, 1, 9, dtype=f32).expand(3, 2, 9)), "place of its own"),
        ((q, k, ids, lens), dict(mass=fake(99, dtype=f32).as_strided((3, 2, 9), (9, 9, 1))), "place of its own"),
        ((q, k, ids, lens), dict(mass=fake(3, 9, 2, dtype=f32).transpose(1, 2)), "contiguous keys"),
    ]:
        with pytest.raises(ValueError, match=match):
            eviction.key_mass(*args, **kw)


def test_evict_arguments():
    k, m = fake(2, 20, 2, 64), fake(2, 2, 20, dtype=torch.float32)
    for args, kw, match in [
        ((k, k[:, :5], m, 4), {}, "of one dtype"),
        ((k, k, m[:, :, :5], 4), {}, "mass must be fp32"),
        ((k, k, m.to(torch.float16), 4), {}, "mass must be fp32"),
        ((k, k, m, 0), {}, "budget in"),
        ((k, k, m, 21), {}, "budget in"),
        ((k, k, m, 4), dict(window=4, sink=1), "fit the budget"),
        ((k, k, m, 4), dict(lengths=fake(3, dtype=torch.int32)), "3 lengths"),
        ((k, k, m, 4), dict(out=(fake(2, 3, 2, 64), fake(2, 3, 2, 64), fake(2, 2, 4, dtype=torch.float32))), "out k/v"),
        ((k, k, m, 4), dict(out=(fake(2, 4, 2, 64), fake(2, 4, 2, 64), fake(2, 2, 3, dtype=torch.float32))), "out mass"),
        ((k, k, m, 4), dict(out=(k[:, :4], fake(2, 4, 2, 64), fake(2, 2, 4, dtype=torch.float32))), "strides|overlap"),
        ((k, k, m, 4), dict(out=(k, k, fake(2, 2, 4, dtype=torch.float32))), "overlap"),
        ((k, k, m, 4), dict(out=(*[fake(2, 4, 2, 64)] * 2, fake(2, 2, 4, dtype=torch.float32))), "place of their own"),
        ((k, k, m, 4), dict(out=(fake(2, 4, 2, 64), fake(2, 4, 2, 64), fake(1, 2, 4, dtype=torch.float32).expand(2, 2, 4))),
         "place of their own"),
    ]:
        with pytest.raises(ValueError, match=match):
            eviction.evict(*args, **kw)
    t, pm = fake(2, 20, dtype=torch.int32), fake(1, 2, 50, dtype=torch.float32)
    for args, kw, match in [
        ((t[0], pm, 4), {}, "slot_table \\[R, T\\]"), ((t, fake(2, 2, 50, dtype=torch.float32), 4), {}, "mass \\[1"),
        ((t, pm, 21), {}, "budget in"), ((t, pm, 4), dict(sink=5), "fit the budget"),
        ((t, pm, 4), dict(lengths=t[:, :1][:1]), "1 lengths"),
    ]:
        with pytest.raises(ValueError, match=match):
            eviction.evict_slots(*args, **kw)
