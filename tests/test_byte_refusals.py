"""What rotate, byte_append, byte_values and byte_read refuse, on the host before any launch, and the rotary
frequencies, which are computed there."""

import ctypes
import math

import pytest
import torch

from lsa_rocm_lab import _abi
from lsa_rocm_lab.port import byte_cache as module
from lsa_rocm_lab.port import pipeline, rotary
from test_serving_refusals import BF16, P, fake


def turn(**over):
    a = dict(frequencies=P, q_weight=None, k_weight=P, pairs=64, frequencies_f64=0, interleaved=0, weights_f32=0, eps=1e-6,
             magnitude=1.0)
    a.update(over)
    return ctypes.addressof(_keep(rotary._Turn(*a.values())))


def held(**over):
    a = dict(k=P, v=P, scales=P, code=0, block=16, caches=2, tokens=100, sb=25600, st=256, sh=128)
    a.update(over)
    return ctypes.addressof(_keep(module._Cache(*a.values())))


_alive = []


def _keep(x):
    _alive.append(x)
    return x


def call_rotate(t=None, **over):
    a = dict(q=P, k=P, dt=BF16, B=2, T=3, Hq=8, Hkv=2, D=128, qsb=0, qst=1024, qsh=128, ksb=0, kst=256, ksh=128, pos=P,
             i64=0, ps=3, turn=t or turn(), qo=P, ko=P, stream=None)
    a.update(over)
    return _abi.call("lsa_rotate", *a.values())


@pytest.mark.parametrize("over,match", [
    (dict(q=None), "NULL"), (dict(ko=None), "NULL"), (dict(turn=None), "NULL"), (dict(pos=None), "NULL positions"),
    (dict(dt=4), "dtype"), (dict(D=96), "head dim"), (dict(Hq=0), "LSA_ERR_SHAPE"), (dict(Hkv=-1), "LSA_ERR_SHAPE"),
    (dict(T=1 << 25), "2\\^26"), (dict(q=P + 8), "aligned"), (dict(kst=258), "aligned"), (dict(ps=-1), "position stride"),
])
def test_rotate_abi(over, match):
    with pytest.raises(ValueError, match=match):
        call_rotate(**over)


@pytest.mark.parametrize("over,match", [
    (dict(pairs=65), "65 pairs"), (dict(pairs=-1), "pairs"), (dict(frequencies=None), "NULL freq"),
    (dict(k_weight=P + 4), "weights"), (dict(eps=-1.0), "eps"), (dict(eps=math.nan), "eps"),
])
def test_turn_abi(over, match):
    with pytest.raises(ValueError, match=match):
        call_rotate(turn(**over))
    assert call_rotate(turn(pairs=0, frequencies=None), B=0) == 0


def append(c=None, t=None, **over):
    a = dict(cache=c or held(), k=P, v=P, q=P, dt=BF16, B=2, T=3, Hq=8, Hkv=2, D=128, ksb=0, kst=256, ksh=128, vsb=0, vst=256,
             vsh=128, qsb=0, qst=1024, qsh=128, starts=P, lens=None, slots=None, turn=t or turn(), out=P, stream=None)
    a.update(over)
    return _abi.call("lsa_byte_append", *a.values())


@pytest.mark.parametrize("over,match", [
    (dict(k=None), "NULL"), (dict(starts=None), "NULL"), (dict(out=None), "NULL"), (dict(cache=None), "NULL cache"),
    (dict(dt=3), "dtype"), (dict(D=48), "head dim"), (dict(Hq=0), "LSA_ERR_SHAPE"), (dict(T=-1), "LSA_ERR_SHAPE"),
    (dict(T=1 << 24), "2\\^24"), (dict(B=3), "2 caches"), (dict(v=P + 2), "aligned"), (dict(vsh=100), "aligned"),
])
def test_append_abi(over, match):
    with pytest.raises(ValueError, match=match):
        append(**over)


@pytest.mark.parametrize("over,match", [
    (dict(scales=None), "NULL cache"), (dict(code=2), "code 2"), (dict(block=3), "LSA_ERR_POW2"), (dict(block=128), "LSA_ERR_POW2"),
    (dict(block=0), "LSA_ERR_POW2"), (dict(caches=3), "3 caches"), (dict(tokens=1 << 31), "LSA_ERR_SHAPE"),
    (dict(st=100), "apart"), (dict(sh=64), "apart"), (dict(st=1 << 31), "apart"), (dict(sb=8), "aligned"),
    (dict(k=P + 8), "aligned"), (dict(scales=P + 4), "aligned"), (dict(caches=1), "slot map"),
])
def test_cache_abi(over, match):
    with pytest.raises(ValueError, match=match):
        append(held(**over))


def values(c=None, **over):
    a = dict(cache=c or held(), rows=P, rs=9, lens=None, R=2, W=9, Hkv=2, D=128, dt=BF16, ko=P, vo=P, stream=None)
    a.update(over)
    return _abi.call("lsa_byte_values", *a.values())


@pytest.mark.parametrize("over,match", [
    (dict(ko=None), "NULL"), (dict(dt=-1), "dtype"), (dict(R=-1), "LSA_ERR_SHAPE"), (dict(W=1 << 31), "LSA_ERR_SHAPE"),
    (dict(R=3), "2 caches"), (dict(vo=P + 4), "aligned"), (dict(D=16), "head dim"),
])
def test_values_abi(over, match):
    with pytest.raises(ValueError, match=match):
        values(**over)


def read(c=None, **over):
    a = dict(q=P, cache=c or held(), dt=BF16, B=2, Tq=1, Hq=8, Hkv=2, D=128, ids=P, lens=P, W=500, per=0, scale=0.1, splits=4,
             counters=P, ws=P, nbytes=1 << 40, out=P, stream=None)
    a.update(over)
    return _abi.call("lsa_byte_read", *a.values())


@pytest.mark.parametrize("over,match", [
    (dict(q=None), "NULL"), (dict(ids=None), "NULL"), (dict(lens=None), "NULL"), (dict(dt=3), "dtype"), (dict(D=100), "head dim"),
    (dict(Hq=7), "must group"), (dict(Hq=1), "must group"), (dict(splits=0), "splits"), (dict(splits=65), "splits"),
    (dict(W=-1), "negative"), (dict(W=(1 << 30) + 1), "2\\^30"), (dict(B=4), "2 caches"), (dict(Tq=1 << 23), "under 2\\^24"), (dict(Tq=1 << 40), "too many"), (dict(Tq=1 << 21, ws=P), "2\\^24 workgroups"),
    (dict(out=P + 8), "aligned"),
])
def test_read_abi(over, match):
    with pytest.raises(ValueError, match=match):
        read(**over)


def test_read_needs_its_scratch():
    need = _abi.size("lsa_byte_read_scratch_bytes", 2, 8, 2, 128, 4)
    assert need == 2 * 2 * 4 * (4 * 128 + 8) * 4
    assert _abi.size("lsa_byte_read_scratch_bytes", 2, 80, 2, 128, 4) == 2 * 2 * 3 * 4 * (16 * 128 + 32) * 4
    for over in (dict(ws=None), dict(nbytes=need - 1), dict(ws=P + 8)):
        with pytest.raises(_abi.LsaError, match="scratch"):
            read(**over)
    assert _abi.size("lsa_byte_read_scratch_bytes", 2, 8, 2, 128, 1) == 0
    assert read(held(caches=0), B=0) == 0


def test_tensors_off_the_gpu_are_refused():
    x, n = torch.zeros(1, 4, 2, 64), torch.zeros(1, dtype=torch.int32)
    c = pipeline.byte_cache(1, 16, 2, 64, 16, torch.int8, "cpu")
    for f in (lambda: pipeline.rotate(x, x, None, None), lambda: pipeline.byte_append(c, x, x, n), lambda: pipeline.byte_values(c),
              lambda: pipeline.byte_read(x, c, n.view(1, 1, 1).expand(1, 4, 1), n.expand(1, 4))):
        with pytest.raises(ValueError, match="ROCm kernel"):
            f()
    with pytest.raises(ValueError, match="one device"):
        pipeline.rotate(fake(1, 4, 2, 64), x, None, None)


def test_rotate_arguments():
    q, k, f32 = fake(3, 5, 8, 64), fake(3, 5, 2, 64), torch.float32
    pos, freq = fake(3, 5, dtype=torch.int32), fake(32, dtype=f32)
    for args, kw, match in [
        ((q[0], k, pos, freq), {}, "q \\[B, T, Hq, D\\]"),
        ((q, fake(3, 4, 2, 64), pos, freq), {}, "q \\[B, T, Hq, D\\]"),
        ((q, fake(3, 5, 2, 32), pos, freq), {}, "q \\[B, T, Hq, D\\]"),
        ((q, fake(3, 5, 2, 64, dtype=torch.float16), pos, freq), {}, "dtypes differ"),
        ((fake(3, 5, 8, 64, dtype=torch.float64), None, pos, freq), {}, "unsupported dtype"),
        ((q, k, None, freq), {}, "positions"),
        ((q, k, pos[:, :4], freq), {}, "positions"),
        ((q, k, pos.float(), freq), {}, "int32 or int64"),
        ((q, k, pos, fake(33, dtype=f32)), {}, "33 pairs"),
        ((q, k, pos, fake(32, 1, dtype=f32)), {}, "frequencies \\[pairs\\]"),
        ((q, k, pos, fake(32)), {}, "fp32 or fp64"),
        ((q, k, pos, torch.zeros(32)), {}, "on cuda:0"),
        ((q, k, pos, freq), dict(q_weight=fake(32)), "norm weights"),
        ((q, k, pos, freq), dict(k_weight=fake(64, dtype=torch.float16)), "norm weights"),
        ((q, k, pos, freq), dict(eps=-1e-6), "eps"),
        ((fake(3, 5, 8, 96), None, pos, freq), {}, "head dim 96"),
    ]:
        with pytest.raises(ValueError, match=match):
            pipeline.rotate(*args, **kw)


def fake_cache(batch=3, tokens=40, heads=2, dim=64, block=16, dtype=torch.int8):
    k, v = (fake(batch, tokens, heads, dim, dtype=dtype) for _ in range(2))
    return pipeline.ByteCache(k, v, fake(batch, -(-tokens // block), heads, 2, dtype=torch.float32), block)


def test_append_arguments():
    k, n = fake(3, 5, 2, 64), fake(3, dtype=torch.int32)
    table = fake(3, 40, dtype=torch.int32)
    c, pool = fake_cache(), fake_cache(1, 160)
    shared = pipeline.ByteCache(c.k, c.k, c.scales, 16)
    wide = fake(3, 40, 2, 128, dtype=torch.int8)
    for args, kw, match in [
        ((c, k, k[:, :4], n), {}, "k and v"),
        ((c, fake(3, 5, 1, 64), fake(3, 5, 1, 64), n), {}, "k and v"),
        ((c, k, k.to(torch.float16), n), {}, "one dtype"),
        ((c, k, k, n), dict(q=fake(3, 5, 8, 64, dtype=torch.float16)), "one dtype"),
        ((c, k, k, n), dict(q=fake(3, 4, 8, 64)), "q \\[3, 5, Hq, 64\\]"),
        ((pool, k, k, n), {}, "or a pool of one with a slot_table"),
        ((c, k, k, n), dict(slot_table=table), "or a pool of one with a slot_table"),
        ((c, k, k, n), dict(slot_rows=n), "slot_rows without"),
        ((c, k, k, n[:2]), {}, "starts and lengths"),
        ((c, k, k, n), dict(lengths=n[:1]), "starts and lengths"),
        ((shared, k, k, n), {}, "place of their own"),
        ((pipeline.ByteCache(fake(1, 40, 2, 64, dtype=torch.int8).expand(3, -1, -1, -1),
                             fake(1, 40, 2, 64, dtype=torch.int8).expand(3, -1, -1, -1), c.scales, 16), k, k, n), {},
         "place of their own"),
        ((pipeline.ByteCache(wide[..., :64], wide[..., 32:96], c.scales, 16), k, k, n), {}, "place of their own"),
        ((pipeline.ByteCache(c.k, c.v, c.scales, 12), k, k, n), {}, "blocks of"),
        ((pipeline.ByteCache(c.k, c.v, c.scales[:, :2], 16), k, k, n), {}, "contiguous fp32 scales"),
        ((pipeline.ByteCache(c.k, c.v, c.scales.to(torch.bfloat16), 16), k, k, n), {}, "contiguous fp32 scales"),
        ((pipeline.ByteCache(c.k.to(torch.uint8), c.v.to(torch.uint8), c.scales, 16), k, k, n), {}, "int8 or float8_e4m3fn"),
        ((pipeline.ByteCache(c.k, c.v[:, :39], c.scales, 16), k, k, n), {}, "a cache \\[B, T, Hkv, D\\]"),
        ((pipeline.ByteCache(c.k.transpose(2, 3), c.v.transpose(2, 3), fake(3, 3, 64, 2, dtype=torch.float32), 16),
          fake(3, 5, 64, 2), fake(3, 5, 64, 2), n), {}, "contiguous rows"),
    ]:
        with pytest.raises(ValueError, match=match):
            pipeline.byte_append(*args, **kw)


def test_values_and_read_arguments():
    c, ids, lens = fake_cache(), fake(3, 1, 9, dtype=torch.int32), fake(3, 1, dtype=torch.int32)
    q = fake(3, 1, 8, 64)
    for f, match in [
        (lambda: pipeline.byte_values(c, ids), "rows \\[R, W\\]"),
        (lambda: pipeline.byte_values(c, ids[:2, 0]), "rows \\[R, W\\]"),
        (lambda: pipeline.byte_values(c, ids[:, 0], lens[:2]), "2 lengths"),
        (lambda: pipeline.byte_values(c, dtype=torch.int8), "unsupported dtype"),
        (lambda: pipeline.byte_read(q[0], c, ids, lens), "q \\[B, Tq, Hq, D\\]"),
        (lambda: pipeline.byte_read(fake(3, 1, 7, 64), c, ids, lens), "q \\[B, Tq, Hq, D\\]"),
        (lambda: pipeline.byte_read(fake(3, 1, 8, 128), c, ids, lens), "q \\[B, Tq, Hq, D\\]"),
        (lambda: pipeline.byte_read(fake(2, 1, 8, 64), c, ids[:2], lens[:2]), "a cache of 2 rows"),
        (lambda: pipeline.byte_read(q, c, ids, lens[:2]), "do not match"),
        (lambda: pipeline.byte_read(q.double(), c, ids, lens), "unsupported dtype"),
        (lambda: pipeline.byte_cache(1, 16, 2, 64, 24), "blocks of"),
        (lambda: pipeline.byte_cache(1, 16, 2, 64, 16, torch.uint8), "int8 or float8_e4m3fn"),
    ]:
        with pytest.raises(ValueError, match=match):
            f()


def test_frequencies():
    f = pipeline.rotary_frequencies(8, 10000.0, dtype=torch.float64)
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-14)
    assert pipeline.rotary_frequencies(8).dtype == torch.float32
    assert torch.equal(pipeline.rotary_frequencies(8, scaling="linear", factor=4.0, dtype=torch.float64), f / 4.0)
    g = pipeline.rotary_frequencies(8, scaling="base", factor=4.0, dtype=torch.float64)
    assert g[0] == 1.0 and abs(g[3] / f[3] - 0.25) < 1e-12 and (g <= f).all()
    # turns in a context of 1000: 159, 15.9, 1.59, 0.159; between 1 and 4 turns in part
    p = pipeline.rotary_frequencies(8, scaling="parts", factor=4.0, original=1000, dtype=torch.float64)
    keep = (1000 * 0.01 / (2 * math.pi) - 1.0) / 3.0
    assert torch.equal(p[:2], f[:2]) and abs(p[2] / f[2] - (keep + (1 - keep) / 4)) < 1e-12 and abs(p[3] / f[3] - 0.25) < 1e-12
    for args, kw in [((7,), {}), ((0,), {}), ((8, -1.0), {}), ((8,), dict(scaling="other")), ((8,), dict(factor=0.0)),
                     ((8,), dict(scaling="parts")), ((8,), dict(scaling="parts", original=10, low=2.0, high=2.0)),
                     ((8,), dict(dtype=torch.float16))]:
        with pytest.raises(ValueError, match="rotary_frequencies"):
            pipeline.rotary_frequencies(*args, **kw)
