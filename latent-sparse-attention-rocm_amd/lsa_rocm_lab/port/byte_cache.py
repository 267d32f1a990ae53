"""A K/V cache held in 8 bits, with a scale for each block of tokens and kv-head.

``byte_cache`` allocates one, dense or a pool of pages; ``byte_append`` norms, rotates, rounds and
writes new tokens; ``byte_values`` gives back what it holds, as numbers (``segment_buckets`` and its
like build an index over these); ``byte_read`` is ``lsa_read`` over it. A key costs half of what it
costs in 16 bits, in memory and in a read. No counterpart in the reference.
"""

from __future__ import annotations

import ctypes
import functools
from dataclasses import dataclass

import torch

from lsa_rocm_lab import _abi
from lsa_rocm_lab.port.eviction import _apart, _meets_twin
from lsa_rocm_lab.port.rotary import head_rows, turn_of
from lsa_rocm_lab.port.shared_prefix import aligned, int32_on, launch_device, lists_of, one_device

_CODES = {torch.int8: 0, torch.float8_e4m3fn: 1}


@dataclass
class ByteCache:
    """Keys and values in 8 bits: row t of kv-head h stands for ``code * scale``, with the scale of
    the ``block`` tokens that t is among. A pool that is read through slot tables is one batch row;
    any table serves to read it. To be written through one its pages are multiples of ``block``: a table
    that ``evict_slots`` has made, whose slots move one by one, is appended to with ``block`` 1."""

    k: torch.Tensor  # [B or 1, T, Hkv, D] int8 or float8_e4m3fn
    v: torch.Tensor
    scales: torch.Tensor  # [B or 1, ceil(T / block), Hkv, 2] fp32: K's, V's
    block: int


class _Cache(ctypes.Structure):
    """``lsa_byte_cache`` (include/lsa_rocm.h)."""

    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("scales", ctypes.c_void_p), ("code", ctypes.c_int32),
                ("block", ctypes.c_int32), ("caches", ctypes.c_int64), ("tokens", ctypes.c_int64),
                ("batch_stride", ctypes.c_int64), ("token_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64)]


def byte_cache(batch: int, tokens: int, heads_kv: int, head_dim: int, block: int = 64, dtype: torch.dtype = torch.int8,
               device: torch.device | str = "cuda") -> ByteCache:
    """An empty 8-bit cache (zeros): ``dtype`` int8 or float8_e4m3fn, ``block`` 1, 2, 4 .. 64 tokens."""
    if dtype not in _CODES:
        raise ValueError(f"byte_cache: int8 or float8_e4m3fn, got {dtype}")
    if block not in (1, 2, 4, 8, 16, 32, 64):
        raise ValueError(f"byte_cache: blocks of 1, 2, 4 .. 64 tokens, got {block}")
    shape = (batch, tokens, heads_kv, head_dim)
    k, v = (torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
    return ByteCache(k, v, torch.zeros(batch, -(-tokens // block), heads_kv, 2, dtype=torch.float32, device=device), block)


def _cache_of(what: str, cache: ByteCache) -> _Cache:
    """``lsa_byte_cache`` of a cache, checked. Its rows are read and written in place: no copy is made."""
    k, v, scales, block = cache.k, cache.v, cache.scales, cache.block
    code = _CODES.get(k.dtype)
    if code is None or v.dtype != k.dtype:
        raise ValueError(f"{what}: a cache of int8 or float8_e4m3fn, got {k.dtype} / {v.dtype}")
    if k.dim() != 4 or k.shape != v.shape:
        raise ValueError(f"{what}: a cache [B, T, Hkv, D], got {tuple(k.shape)} / {tuple(v.shape)}")
    if block not in (1, 2, 4, 8, 16, 32, 64):
        raise ValueError(f"{what}: blocks of 1, 2, 4 .. 64 tokens, got {block}")
    n, T, H, D = k.shape
    if scales.dtype is not torch.float32 or scales.shape != (n, -(-T // block), H, 2) or not scales.is_contiguous():
        raise ValueError(f"{what}: contiguous fp32 scales {[n, -(-T // block), H, 2]}, got {scales.dtype} "
                         f"{tuple(scales.shape)}")
    strides = k.stride()
    if strides != v.stride() or strides[3] != 1:
        raise ValueError(f"{what}: K and V codes at one layout with contiguous rows, got strides {strides} / {v.stride()}")
    return _Cache(k.data_ptr(), v.data_ptr(), scales.data_ptr(), code, block, n, T, strides[0] if n > 1 else 0,
                  strides[1] if T > 1 else D, strides[2] if H > 1 else D)


def byte_append(
    cache: ByteCache,
    k: torch.Tensor,
    v: torch.Tensor,
    starts: torch.Tensor,
    lengths: torch.Tensor | None = None,
    slot_table: torch.Tensor | None = None,
    slot_rows: torch.Tensor | None = None,
    q: torch.Tensor | None = None,
    frequencies: torch.Tensor | None = None,
    q_weight: torch.Tensor | None = None,
    k_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    interleaved: bool = False,
    magnitude: float = 1.0,
) -> torch.Tensor | None:
    """Writes each row's new tokens behind its cache; returns q normed and rotated (None without q).

    k, v [B, T, Hkv, D] (fp32, bf16 or fp16): the first ``lengths[b]`` (default T) tokens of row b go to
    positions ``starts[b]``, ``starts[b] + 1``, ..; k is normed (with ``k_weight``) and rotated (with
    ``frequencies``) first, as ``rotate`` does, and so is q [B, T, Hq, D] (zeros behind a row's
    length); where a token's position is not its place in the cache (after an eviction, say), ``rotate``
    first and give no ``frequencies``. ``cache`` has B rows, or is a pool [1, rows, Hkv, D] that ``slot_table`` [n, width] and
    ``slot_rows`` [B] (as in the selects) map positions to, whole blocks at a time. Positions outside
    are dropped, and so are new tokens of a block of positions whose slots are not a block of the pool:
    ``block`` rows in order from a multiple of it on (slots behind the new tokens may also name no row
    of the pool). Dropped tokens change no row and have no part in a scale. No block may be written to
    twice in a call (by two rows, or two entries of a table).

    A block's scale is its largest magnitude over 127 (int8) or 448 (e4m3), at least 2^-100, and
    codes are rounded to nearest. Tokens before ``starts[b]`` in the first block stay: where its scale
    grows, their codes are rescaled and rounded again, by at most half a step. That adds up: a token of a
    block that is filled token by token is off by up to g + 1 half steps where the scale grew g times
    behind it. Rows of N(0, 1) grow it 3 to 6 times in 64 tokens, for 1.2 to 1.6 times the error of one
    append in rms (e4m3 2.0); magnitudes that rise by 3% with every token, less than a code's step, 11
    times (e4m3 40: the codes stay and their values rise with the scale). With ``block`` 1 a token is
    rounded once. What the block held from ``starts[b]`` on is given up, so a row may be taken back by
    appending at an earlier position. NaN and infinities stay out of the scale; a NaN is held as e4m3's
    NaN or as 0, an infinity as the largest code.
    """
    from lsa_rocm_lab.port.pipeline import _slot_args

    device = one_device("byte_append", k, v, cache.k, cache.v, cache.scales, q)
    if k.dim() != 4 or k.shape != v.shape or k.shape[2:] != cache.k.shape[2:]:
        raise ValueError(f"byte_append: k and v [B, T, Hkv, D] for a cache {tuple(cache.k.shape)}, got {tuple(k.shape)} / "
                         f"{tuple(v.shape)}")
    if k.dtype != v.dtype or (q is not None and q.dtype != k.dtype):
        raise ValueError(f"byte_append: one dtype, got {k.dtype} {v.dtype} {None if q is None else q.dtype}")
    dt = _abi.dtype_code(k.dtype)
    held = _cache_of("byte_append", cache)
    k8, v8 = cache.k, cache.v
    if not (k8.is_contiguous() and abs(v8.data_ptr() - k8.data_ptr()) >= k8.numel()) and (
            not (_apart(k8) and _apart(v8)) or _meets_twin(k8, v8)):
        raise ValueError("byte_append: the cache's codes must each have a place of their own")
    B, T, Hkv, D = k.shape
    if Hkv < 1:
        raise ValueError(f"byte_append: k and v of a kv-head or more, got {tuple(k.shape)}")
    if q is not None and (q.dim() != 4 or q.shape[:2] != k.shape[:2] or q.shape[3] != D):
        raise ValueError(f"byte_append: q [{B}, {T}, Hq, {D}], got {tuple(q.shape)}")
    if held.caches != (B if slot_table is None else 1):
        raise ValueError(f"byte_append: a cache of {B} rows, or a pool of one with a slot_table; got {held.caches}")
    starts = int32_on(starts, device)
    lens = None if lengths is None else int32_on(lengths, device)
    if starts.numel() != B or (lens is not None and lens.numel() != B):
        raise ValueError(f"byte_append: starts and lengths [{B}]")
    if slot_table is not None:  # numbers past 32 bits are rows of no cache
        if slot_table.dtype is not torch.int32:
            slot_table = int32_on(slot_table, device)
        slot_rows = None if slot_rows is None else int32_on(slot_rows, device)
    turn, _keep = turn_of("byte_append", device, D, k.dtype, frequencies, q_weight, k_weight, eps, interleaved, magnitude)
    slots, _slots = _slot_args(slot_table, slot_rows, B, device)
    out, Hq, qsb, qst, qsh = None, 0, 0, 0, 0
    if q is not None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        Hq = q.shape[2]
    if k.numel() == 0:
        return out
    if q is not None:
        q, qsb, qst, qsh = head_rows(q)
    k, ksb, kst, ksh = head_rows(k)
    v, vsb, vst, vsh = head_rows(v)
    with launch_device(device):
        _abi.call("lsa_byte_append", ctypes.addressof(held), k.data_ptr(), v.data_ptr(), _abi.ptr(q), dt, B, T, Hq, Hkv, D,
                  ksb, kst, ksh, vsb, vst, vsh, qsb, qst, qsh, starts.data_ptr(), _abi.ptr(lens), slots,
                  ctypes.addressof(turn), _abi.ptr(out), _abi.stream(device))
    return out


def byte_values(cache: ByteCache, rows: torch.Tensor | None = None, lengths: torch.Tensor | None = None,
                dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
    """What the cache holds, as numbers: (k, v) [R, W, Hkv, D] in ``dtype`` (fp32, bf16 or fp16).

    ``rows`` [R, W]: the cache rows of each list (a slot table's, say; of batch row r, or of a pool),
    default all of every batch row. Rows outside the cache, and those from ``lengths[r]`` on, are zeros.
    """
    device = one_device("byte_values", cache.k, cache.v, cache.scales)
    dt = _abi.dtype_code(dtype)
    held = _cache_of("byte_values", cache)
    Hkv, D = cache.k.shape[2:]
    R, W = cache.k.shape[:2]
    if rows is not None:
        if rows.dim() != 2 or held.caches not in (rows.shape[0], 1):
            raise ValueError(f"byte_values: rows [R, W] of a cache of R batch rows or one, got {tuple(rows.shape)} of "
                             f"{held.caches}")
        rows = int32_on(rows, device)
        R, W = rows.shape
    lens = None if lengths is None else int32_on(lengths, device)
    if lens is not None and lens.numel() != R:
        raise ValueError(f"byte_values: {lens.numel()} lengths for {R} rows")
    k = torch.empty((R, W, Hkv, D), dtype=dtype, device=device)
    v = torch.empty_like(k)
    if R * W * Hkv:
        with launch_device(device):
            _abi.call("lsa_byte_values", ctypes.addressof(held), _abi.ptr(rows), W, _abi.ptr(lens), R, W, Hkv, D, dt,
                      k.data_ptr(), v.data_ptr(), _abi.stream(device))
    return k, v


_READ_SPLITS = 64
_SLAB_BYTES = 256 << 20  # partials held at once (more query rows go through in slabs)


@functools.lru_cache(maxsize=4096)
def _read_splits(units: int, width: int) -> int:
    """Spans of a list, a workgroup each. 256 units (a CU each) and more read theirs whole, fewer are cut until
    there are about 512 workgroups, lists of any number past 1500 slots, so that lengths that differ even out and rows
    that walk the same keys meet in the caches; a span has 192 slots or more, below which its start costs more
    than it saves, in whole steps of 128. Measured, us, by spans: 8 units of 2816 slots 4: 12.6, 8: 9.4, 11: 9.0,
    22: 9.3; 256 of them 1: 30.8, 2: 35.2, 8: 36.4; 160 of 6336 2: 56, 4: 41.4, 8: 46; 128 of 32768 4: 196, 16: 173,
    32: 168; 16384 of 4608 1: 2492, 3: 2417, 8: 2463; 32768 of 32768 1: 33100, 4: 26800, 16: 22800, 20: 23400."""
    few = -(-512 // units) if units < 256 else 1
    splits = max(1, min(_READ_SPLITS, width // 192, max(few, width // 1500), (1 << 23) // units))
    span = -(-(-(-width // splits)) // 128) * 128
    return max(1, -(-width // max(span, 1)))


def _even(n: int, most: int) -> int:
    """The size of even pieces of n, of at most ``most``."""
    return -(-n // -(-n // most))


def byte_read(q: torch.Tensor, cache: ByteCache, read_lists: torch.Tensor, lengths: torch.Tensor,
              scale: float | None = None) -> torch.Tensor:
    """Attention of every query row over its read list of an 8-bit cache: ``lsa_read``'s contract.

    q [B, Tq, Hq, D] (fp32, bf16 or fp16); ``cache`` of B rows or a pool; ``read_lists`` [B, Tq, W], shared
    by the heads, or [B, Tq, Hkv, W], with ``lengths`` to match: cache rows, those outside the cache
    skipped, duplicates counted per occurrence. A slot table and its rows' lengths read a whole paged
    cache. Any number of query heads a kv-head. A row with no keys gives zeros; the output is like q.
    Keys enter exactly, q exactly; softmax weights times V's scale are rounded to 16 bits of mantissa
    (24 for fp32 rows), the sum that divides them is of the unrounded ones.
    """
    device = one_device("byte_read", q, cache.k, cache.v, cache.scales)
    held = _cache_of("byte_read", cache)
    Hkv = cache.k.shape[2]
    if q.dim() != 4 or q.shape[3] != cache.k.shape[3] or Hkv < 1 or q.shape[2] % Hkv:
        raise ValueError(f"byte_read: q [B, Tq, Hq, D] for a cache {tuple(cache.k.shape)}, got {tuple(q.shape)}")
    dt = _abi.dtype_code(q.dtype)
    B, Tq, Hq, D = q.shape
    if held.caches not in (B, 1):
        raise ValueError(f"byte_read: a cache of {B} rows or a pool of one, got {held.caches}")
    ids, lens, W, per_head = lists_of(read_lists, lengths, B * Tq, Hkv, device)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if out.numel() == 0:
        return out
    q = aligned(q)
    rows = B * Tq
    units = rows * Hkv * -(-Hq // Hkv // 16)
    splits = _read_splits(units, W)
    nbytes = _abi.shape_size("lsa_byte_read_scratch_bytes", rows, Hq, Hkv, D, splits)
    slabs = nbytes > _SLAB_BYTES and rows > 1
    if slabs:
        if held.caches == 1:  # all of the rows are of one cache
            B, Tq = 1, rows
        most = max(1, _SLAB_BYTES // (nbytes // rows))
        many, step = (_even(B, most // Tq), Tq) if Tq <= most else (1, _even(Tq, most))  # batch rows, query rows of each
        nbytes, units = nbytes // rows * many * step, units // rows * many * step
    scale = float(D ** -0.5 if scale is None else scale)
    q_at, out_at, ids_at, lens_at = q.data_ptr(), out.data_ptr(), ids.data_ptr(), lens.data_ptr()
    with launch_device(device):
        ws, counters, stream = _abi.call_memory(device, "byte_read", nbytes, units if nbytes else 0)

        def launch(part, m, n, at):  # n query rows of m batch rows, the first of them row `at`
            first, row = at * Hq * D * q.element_size(), 4 * at * (Hkv if per_head else 1)
            _abi.call_in_order("lsa_byte_read", q_at + first, ctypes.addressof(part), dt, m, n, Hq, Hkv, D,
                               ids_at + row * W, lens_at + row, W, 1 if per_head else 0, scale, splits,
                               _abi.ptr(counters), _abi.ptr(ws), nbytes, out_at + first, stream)

        if not slabs:
            launch(held, B, Tq, 0)
            return out
        for b in range(0, B, many):
            m = min(many, B - b)
            part = held
            if m < B:  # caches b .. b + m
                k, v, scales = (x[b:b + m].data_ptr() for x in (cache.k, cache.v, cache.scales))
                part = _Cache(k, v, scales, held.code, held.block, m, held.tokens, held.batch_stride, held.token_stride,
                              held.head_stride)
            for t in range(0, Tq, step):
                launch(part, m, min(step, Tq - t), b * Tq + t)
    return out
