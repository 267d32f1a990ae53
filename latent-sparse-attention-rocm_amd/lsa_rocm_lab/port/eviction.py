"""A cache that is cut down to the keys that carry attention weight.

``key_mass`` adds up the softmax weight each listed key received (from decode steps as they run,
or from a prompt's last rows); ``evict`` keeps the heaviest keys of a dense cache, beside its
first and last ones, and ``evict_slots`` does so for a paged cache by reordering its slot table.
The kept keys stay in their order, so bucket tables are built over the smaller cache as over any
other (``pipeline.segment_buckets``, ``build_buckets``). No counterpart in the reference.
"""

from __future__ import annotations

import torch

from lsa_rocm_lab import _abi
from lsa_rocm_lab.port.shared_prefix import aligned, cache_pair, cache_strides, int32_on, launch_device, lists_of, one_device

# Batch rows and their query rows go through in slabs: of so many bytes of scratch, so many softmaxes a cache
# (their sums are 64-bit integers) and so many kv-heads of rows (a launch's limit)
_SLAB_BYTES, _SLAB_SUMS, _SLAB_UNITS = 256 << 20, 1 << 19, (1 << 24) - 1


def _apart(t: torch.Tensor) -> bool:
    """Whether a tensor that is written has every element in a place of its own."""
    reach = 1
    for step, n in sorted((step, n) for step, n in zip(t.stride(), t.shape) if n > 1):
        if step < reach:
            return False
        reach = step * n
    return True


def key_mass(
    q: torch.Tensor,
    k: torch.Tensor,
    read_lists: torch.Tensor,
    lengths: torch.Tensor,
    scale: float | None = None,
    lse: torch.Tensor | None = None,
    mass: torch.Tensor | None = None,
) -> torch.Tensor:
    """The attention weight that each listed key receives, summed over the query rows of its
    cache and the query heads of its kv-head.

    q [B, Tq, Hq, D], k [B, Tk, Hkv, D] (or one pool [1, Tk, Hkv, D] for every row),
    ``read_lists`` / ``lengths`` as ``lsa_read`` takes them (``[B, Tq, W]`` or ``[B, Tq, Hkv, W]``;
    ids outside the cache are skipped, a key listed twice counts twice). The weights are of the
    softmax over the row's list, or, with ``lse`` [B, Tq, Hq] (``prefix_read(return_lse=True)``'s),
    of the wider softmax it belongs to (whose weights are at most 1: by an ``lse`` that is too low
    they are 1). A row whose sum is not a number gives none, as it reads as no keys in
    ``lsa_read``. Where several query rows share a cache a weight is rounded to a multiple of 2^-44
    (by a given ``lse`` and lists of n > 2^19 slots times heads, of n 2^-63). Returns
    [B or 1, Hkv, Tk] fp32: new, or ``mass`` with the weights added in place. The bits do not
    depend on the order in which rows and workgroups run.
    """
    device = one_device("key_mass", q, k, lse, mass)
    if q.dim() != 4 or k.dim() != 4 or k.shape[0] not in (q.shape[0], 1) or k.shape[3] != q.shape[3]:
        raise ValueError(f"key_mass: q [B, Tq, Hq, D] and k [B or 1, Tk, Hkv, D], got {tuple(q.shape)} and "
                         f"{tuple(k.shape)}")
    if q.dtype != k.dtype:
        raise ValueError(f"key_mass: q/k dtypes differ: {q.dtype} {k.dtype}")
    dt = _abi.dtype_code(q.dtype)
    B, Tq, Hq, D = q.shape
    caches, Tk, Hkv = k.shape[:3]
    if Hkv < 1 or Hq % Hkv:
        raise ValueError(f"key_mass: {Hq} query heads do not group onto {Hkv} kv-heads")
    ids, lens, W, per_head = lists_of(read_lists, lengths, B * Tq, Hkv, device)
    if lse is not None and (tuple(lse.shape) != (B, Tq, Hq) or lse.dtype != torch.float32):
        raise ValueError(f"key_mass: lse must be fp32 [{B}, {Tq}, {Hq}], got {lse.dtype} {tuple(lse.shape)}")
    fresh = mass is None
    if fresh:
        mass = torch.empty(caches, Hkv, Tk, dtype=torch.float32, device=device)
    elif (tuple(mass.shape) != (caches, Hkv, Tk) or mass.dtype != torch.float32 or (Tk > 1 and mass.stride(2) != 1)
          or not _apart(mass)):
        raise ValueError(f"key_mass: mass must be fp32 [{caches}, {Hkv}, {Tk}] with contiguous keys, each in a place of "
                         f"its own, got {mass.dtype} {tuple(mass.shape)} at strides {mass.stride()}")
    if B * Tq == 0 or W == 0 or Tk == 0:
        return mass.zero_() if fresh else mass
    q = aligned(q)
    if k.stride(-1) != 1 or k.data_ptr() % 16:
        k = aligned(k)
    sb, st, sh = cache_strides(k)
    lse = None if lse is None else lse.contiguous()
    scale = float(D ** -0.5 if scale is None else scale)
    # every query row's scores are held until its sums are known, beside the integers that several rows of a cache
    # add up in (twice its masses: a pool's, or one cache's, are not cut)
    many, step = B, Tq
    scores, cell = 4 * Hq * W, 8 * Hkv * Tk if caches == B and Tq > 1 else 0  # bytes of a query row, of a cache
    if B * (Tq * scores + cell) > _SLAB_BYTES or B * Tq * Hq > _SLAB_SUMS:
        group = Hq // Hkv
        many = max(1, min(B, _SLAB_BYTES // (scores + 2 * cell), _SLAB_SUMS // group if caches < B else B,
                          _SLAB_UNITS // Hkv))
        step = max(1, min(Tq, (_SLAB_BYTES - many * cell) // (many * scores),
                          _SLAB_SUMS // (group if caches == B else many * group), _SLAB_UNITS // (many * Hkv)))
    with launch_device(device):
        for b in range(0, B, many):
            m = min(many, B - b)
            own, kb, mb = (1, k, mass) if caches < B else (m, k[b:b + m], mass[b:b + m])
            for t in range(0, Tq, step):
                n = min(step, Tq - t)
                part, pids, plens, plse = q, ids, lens, lse
                if (m, n) != (B, Tq):  # rows t .. t + n of batch rows b .. b + m
                    part = q[b:b + m, t:t + n].contiguous()
                    pids = ids.view(B, Tq, -1)[b:b + m, t:t + n].contiguous()
                    plens = lens.view(B, Tq, -1)[b:b + m, t:t + n].contiguous()
                    plse = None if lse is None else lse[b:b + m, t:t + n].contiguous()
                nbytes = _abi.shape_size("lsa_key_mass_scratch_bytes", dt, m, n, own, Tk, Hq, Hkv, D, W)
                ws, counters, stream = _abi.call_memory(device, "key_mass", nbytes, m * Hkv if n == 1 and own == m else 0)
                first = fresh and t == 0 and (b == 0 or caches == B)
                _abi.call_in_order("lsa_key_mass", part.data_ptr(), kb.data_ptr(), dt, m, n, own, Tk, Hq, Hkv, D, sb, st,
                                   sh, pids.data_ptr(), plens.data_ptr(), W, 1 if per_head else 0, scale, _abi.ptr(plse),
                                   1 if first else 0, _abi.ptr(counters), _abi.ptr(ws), nbytes, mb.data_ptr(),
                                   mass.stride(0) if own > 1 else Hkv * Tk, mass.stride(1) if Hkv > 1 else Tk, stream)
    return mass


def _check_keep(what: str, T: int, budget: int, window: int, sink: int) -> None:
    if not 1 <= budget <= T:
        raise ValueError(f"{what}: a budget in 1..{T}, got {budget}")
    if window < 0 or sink < 0 or window + sink > budget:
        raise ValueError(f"{what}: window {window} and sink {sink} must fit the budget {budget}")


def _row_lengths(what: str, lengths: torch.Tensor | None, B: int, device: torch.device) -> torch.Tensor | None:
    if lengths is None:
        return None
    lens = int32_on(lengths, device)
    if lens.numel() != B:
        raise ValueError(f"{what}: {lens.numel()} lengths for {B} rows")
    return lens


def _dense_mass(what: str, mass: torch.Tensor, shape: tuple[int, int, int]) -> torch.Tensor:
    if tuple(mass.shape) != shape or mass.dtype != torch.float32:
        raise ValueError(f"{what}: mass must be fp32 {list(shape)}, got {mass.dtype} {tuple(mass.shape)}")
    return mass if shape[2] <= 1 or mass.stride(2) == 1 else mass.contiguous()


def _extent(t: torch.Tensor) -> tuple[int, int]:
    """The addresses between which a tensor's elements lie."""
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride())) if t.numel() else -1
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _axes(t: torch.Tensor) -> list[tuple[int, int]]:
    """(step in bytes, size) of a tensor's axes, the largest step first; elements that follow each other
    are one axis, the last, of step 1. Of an ``_apart`` tensor each step holds all of the smaller ones."""
    size = t.element_size()
    found = [(1, size)]
    for step, n in sorted((step * size, n) for step, n in zip(t.stride(), t.shape) if n > 1):
        found = [*found[:-1], (1, n * step)] if len(found) == 1 and step == found[-1][1] else [*found, (step, n)]
    return [*found[:0:-1], found[0]]


def _meets_twin(k: torch.Tensor, v: torch.Tensor) -> bool:
    """Whether two ``_apart`` tensors of the same shape and steps share a byte."""
    axes = _axes(k)

    def hit(rest: int, i: int) -> bool:  # rest: a sum of steps, each taken fewer than its size of times either way?
        step, n = axes[i]
        if i == len(axes) - 1:
            return abs(rest) < n
        return any(abs(x) < n and hit(rest - x * step, i + 1) for x in (rest // step, rest // step + 1))

    return k.numel() > 0 and hit(v.data_ptr() - k.data_ptr(), 0)


def _meets(t: torch.Tensor, lo: int, hi: int) -> bool:
    """Whether an ``_apart`` tensor has a byte at an address in [lo, hi)."""
    axes = _axes(t)

    def hit(at: int, i: int) -> bool:
        step, n = axes[i]
        reach = sum((m - 1) * s for s, m in axes[i + 1:]) + 1  # bytes from the first to past the last of one index
        first, last = max(0, (lo - at - reach) // step + 1), min(n - 1, (hi - 1 - at) // step)  # whose bytes' span meets it
        if first > last or i == len(axes) - 1 or last - first > 1:  # of three in a line it holds the middle one
            return first <= last
        return any(hit(at + x * step, i + 1) for x in range(first, last + 1))

    return t.numel() > 0 and lo < hi and hit(t.data_ptr(), 0)


def _places_apart(k: torch.Tensor, v: torch.Tensor, mass: torch.Tensor) -> bool:
    """Whether what is written of ``evict``'s out (K and V at the same steps) has a place of its own."""
    if not (_apart(k) and _apart(v) and _apart(mass)) or _meets_twin(k, v):
        return False
    lo, hi = _extent(mass)
    if not (_meets(k, lo, hi) or _meets(v, lo, hi)):
        return True
    *outer, (_, run) = _axes(mass)
    starts = [mass.data_ptr()]
    for step, n in outer:
        starts = [at + x * step for at in starts for x in range(n)]
    return not any(_meets(x, at, at + run) for at in starts for x in (k, v))


def evict(
    k: torch.Tensor,
    v: torch.Tensor,
    mass: torch.Tensor,
    budget: int,
    lengths: torch.Tensor | None = None,
    window: int = 0,
    sink: int = 0,
    shared: bool = False,
    out: tuple[torch.Tensor, torch.Tensor, torch.Tensor] | None = None,
):
    """The ``budget`` keys of each row and kv-head worth keeping, and the cache cut down to them.

    k/v [B, T, Hkv, D], mass [B, Hkv, T] fp32 (``key_mass``'s, accumulated). Of a row's
    ``lengths[b]`` positions (default T) the first ``sink`` and the last ``window`` stay, and of the
    others those of largest mass; ties go to the lower position, a NaN weighs least; a row of at
    most ``budget`` positions keeps all. ``shared``: the kv-heads keep the same positions, by the sum
    of their masses (as lists over an index-space table need it).

    Returns ``(k, v, mass, kept, lengths)``: the kept rows in their order, [B, budget, Hkv, D], their
    masses [B, Hkv, budget], their positions in the old cache [B, Hkv, budget] int32 (shared:
    [B, budget]; -1 past the row's new length) and the new lengths [B] int32. New tensors hold
    zeros past the new length. ``out`` = (k, v, mass) buffers of ``budget`` rows or more (not the
    inputs: two caches take turns; each written element in a place of its own), whose rows past the
    new length are left as they were.
    """
    device = one_device("evict", k, v, mass)
    if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype:
        raise ValueError(f"evict: k/v [B, T, Hkv, D] of one dtype, got {k.dtype} {tuple(k.shape)} / {v.dtype} "
                         f"{tuple(v.shape)}")
    B, T, Hkv, D = k.shape
    dt = _abi.dtype_code(k.dtype)
    budget, window, sink = int(budget), int(window), int(sink)
    _check_keep("evict", T, budget, window, sink)
    mass = _dense_mass("evict", mass, (B, Hkv, T))
    lens = _row_lengths("evict", lengths, B, device)
    k, v, (sb, st, sh) = cache_pair(k, v)
    if out is None:
        k2, v2 = (torch.empty(B, budget, Hkv, D, dtype=k.dtype, device=device) for _ in range(2))
        m2 = torch.empty(B, Hkv, budget, dtype=torch.float32, device=device)
    else:
        k2, v2, m2 = out
        one_device("evict", k, k2, v2, m2)
        if (k2.dim() != 4 or k2.shape != v2.shape or k2.shape[1] < budget or (k2.shape[0], *k2.shape[2:]) != (B, Hkv, D)
                or k2.dtype != k.dtype or v2.dtype != k.dtype or k2.stride(-1) != 1 or v2.stride(-1) != 1
                or cache_strides(k2) != cache_strides(v2) or k2.data_ptr() % 16 or v2.data_ptr() % 16):
            raise ValueError(f"evict: out k/v must be {k.dtype} [{B}, >= {budget}, {Hkv}, {D}] of contiguous, 16-byte "
                             f"aligned rows at the same strides, got {tuple(k2.shape)} / {tuple(v2.shape)}")
        if (m2.dim() != 3 or tuple(m2.shape[:2]) != (B, Hkv) or m2.shape[2] < budget or m2.dtype != torch.float32
                or (m2.shape[2] > 1 and m2.stride(2) != 1)):
            raise ValueError(f"evict: out mass must be fp32 [{B}, {Hkv}, >= {budget}] with contiguous keys, got "
                             f"{tuple(m2.shape)}")
        for new in out:
            a, b = _extent(new)
            if any(a < hi and lo < b for lo, hi in map(_extent, (k, v, mass))):
                raise ValueError("evict: out must not overlap the cache it is made from")
        if not _places_apart(k2[:, :budget], v2[:, :budget], m2[..., :budget]):
            raise ValueError("evict: out k, v and mass need a place of their own for every element")
    ob, ot, oh = cache_strides(k2)
    kept = torch.empty((B, budget) if shared else (B, Hkv, budget), dtype=torch.int32, device=device)
    new_lengths = torch.empty(B, dtype=torch.int32, device=device)
    if B:
        one = 1 if shared else 0
        nbytes = _abi.shape_size("lsa_evict_scratch_bytes", B, Hkv, T, one)
        with launch_device(device):
            ws, _, stream = _abi.call_memory(device, "evict", nbytes)
            _abi.call_in_order("lsa_evict_keep", mass.data_ptr(), B, Hkv, T, mass.stride(0), mass.stride(1),
                               _abi.ptr(lens), budget, window, sink, one, None, 0, 0, _abi.ptr(ws), nbytes,
                               kept.data_ptr(), new_lengths.data_ptr(), None, 0, stream)
            _abi.call("lsa_evict_rows", k.data_ptr(), v.data_ptr(), mass.data_ptr(), dt, B, T, Hkv, D, sb, st, sh,
                      mass.stride(0), mass.stride(1), kept.data_ptr(), one, budget, k2.data_ptr(), v2.data_ptr(), ob,
                      ot, oh, m2.data_ptr(), m2.stride(0), m2.stride(1), 1 if out is None else 0, stream)
    return k2, v2, m2, kept, new_lengths


def evict_slots(
    slot_table: torch.Tensor,
    mass: torch.Tensor,
    budget: int,
    lengths: torch.Tensor | None = None,
    window: int = 0,
    sink: int = 0,
):
    """``evict`` for a paged cache: no K/V row moves, the slot table changes.

    ``slot_table`` [R, T] int32 (a row a sequence: logical position -> cache row), mass
    [1, Hkv, pool] fp32 (``key_mass``'s over the pool). What row r keeps of its ``lengths[r]``
    positions (default T) is decided as in ``evict`` with ``shared``; a position without a cache row
    (outside the pool) weighs least.

    Returns ``(slot_table, lengths, kept)``: each row with the cache rows it keeps first, in their
    order, then the ones it gave up, in theirs (the sequence's next tokens may take them, or an
    allocator), then what was behind its length; the new lengths [R] and the kept positions
    [R, budget] (-1 past the new length), int32. The masses stay with their cache rows: clear
    those that are given to a new token.
    """
    device = one_device("evict_slots", slot_table, mass)
    if slot_table.dim() != 2 or slot_table.shape[1] < 1:
        raise ValueError(f"evict_slots: slot_table [R, T], got {tuple(slot_table.shape)}")
    if mass.dim() != 3 or mass.shape[0] != 1 or mass.shape[1] < 1 or mass.shape[2] < 1:
        raise ValueError(f"evict_slots: mass [1, Hkv, pool], got {tuple(mass.shape)}")
    R, T = slot_table.shape
    Hkv, pool = mass.shape[1:]
    budget, window, sink = int(budget), int(window), int(sink)
    _check_keep("evict_slots", T, budget, window, sink)
    mass = _dense_mass("evict_slots", mass, (1, Hkv, pool))
    lens = _row_lengths("evict_slots", lengths, R, device)
    table = int32_on(slot_table, device)
    new_table = torch.empty(R, T, dtype=torch.int32, device=device)
    kept = torch.empty(R, budget, dtype=torch.int32, device=device)
    new_lengths = torch.empty(R, dtype=torch.int32, device=device)
    if R:
        nbytes = _abi.shape_size("lsa_evict_scratch_bytes", R, Hkv, T, 1)
        with launch_device(device):
            ws, _, stream = _abi.call_memory(device, "evict", nbytes)
            _abi.call_in_order("lsa_evict_keep", mass.data_ptr(), R, Hkv, T, 0, mass.stride(1), _abi.ptr(lens), budget,
                               window, sink, 1, table.data_ptr(), T, pool, _abi.ptr(ws), nbytes, kept.data_ptr(),
                               new_lengths.data_ptr(), new_table.data_ptr(), T, stream)
    return new_table, new_lengths, kept
