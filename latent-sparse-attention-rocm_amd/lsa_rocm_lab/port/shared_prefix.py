"""Attention of a decode batch over a prefix that its rows share.

Requests behind one system prompt hold the same keys at its start. ``prefix_read`` keeps those
once and joins them in one softmax with what each row reads of its own cache (a read list, as
``lsa_read``). bf16 and fp16 rows of head dim 64 or 128 read them once for the whole batch (up to
256 query rows times heads a kv-head at a time); fp32, head dims 32 and 256 and a scale that is not
positive read them once a query row. No counterpart in the reference.
"""

from __future__ import annotations

import contextlib

import torch

from lsa_rocm_lab import _abi


_HERE = contextlib.nullcontext()
_SLAB_BYTES = 256 << 20  # partials held at once (more query rows go through in slabs)


def launch_device(device: torch.device):
    """A context in which a launch on a tensor's ``device`` finds it current (nothing where it is)."""
    return _HERE if device.index == _abi.current_device() else torch.cuda.device(device)


def one_device(what: str, *tensors: torch.Tensor | None) -> torch.device:
    """The ROCm device that all of the tensors are on; anything else raises ``ValueError``."""
    device = tensors[0].device
    index = device.index  # compared in a fraction of a device's time
    for t in tensors:
        if t is not None and t.get_device() != index and (t.device != device or device.type != "cuda"):
            raise ValueError(f"{what} is a ROCm kernel over tensors of one device, got {device} and {t.device}")
    return device


def int32_on(t: torch.Tensor, device: torch.device) -> torch.Tensor:
    """``t`` as a kernel reads it: int32, contiguous, on ``device``. A number past 32 bits becomes the
    nearest that they hold (an id, slot or prefix outside every cache, a length past every row)."""
    if t.dtype is torch.int32 and (t.get_device() == device.index or t.device == device) and t.is_contiguous():
        return t
    if t.dtype is not torch.int32 and t.dtype.itemsize >= 4:
        t = t.to(torch.int64).clamp(-(1 << 31), (1 << 31) - 1)
    return t.to(device=device, dtype=torch.int32).contiguous()


def cache_strides(x: torch.Tensor) -> tuple[int, int, int]:
    """Batch, token and head strides of a cache [B, T, Hkv, D] (an axis of one has none of its own)."""
    sb, st, sh, _ = x.stride()
    nb, nt, nh, D = x.shape
    return sb if nb > 1 else 0, st if nt > 1 else D, sh if nh > 1 else D


def cache_pair(k: torch.Tensor, v: torch.Tensor):
    """K and V as a kernel reads them (rows of contiguous elements at the same strides; other
    layouts are made dense) and their strides."""
    ks, vs = k.stride(), v.stride()
    if (ks[3] != 1 or vs[3] != 1 or (ks != vs and cache_strides(k) != cache_strides(v))
            or (k.data_ptr() | v.data_ptr()) % 16):
        k, v = aligned(k), aligned(v)
    return k, v, cache_strides(k)


def aligned(x: torch.Tensor) -> torch.Tensor:
    """``x`` dense and 16-byte aligned (a contiguous view may begin off that)."""
    x = x.contiguous()
    return x.clone() if x.data_ptr() % 16 else x


def lists_of(read_lists: torch.Tensor, lengths: torch.Tensor, rows: int, heads_kv: int, device: torch.device):
    """Read lists of ``rows`` query rows as ``lsa_read`` takes them: ids [n, W], lengths [n], and
    whether every kv-head has its own."""
    width = read_lists.shape[-1]
    ids, lens = int32_on(read_lists, device), int32_on(lengths, device)
    n = lens.numel()
    per_head = heads_kv > 1 and n == rows * heads_kv and n != rows
    if n != (rows * heads_kv if per_head else rows) or ids.numel() != n * width:
        raise ValueError(f"read lists {tuple(read_lists.shape)} / lengths {tuple(lengths.shape)} do not match "
                         f"{rows} query rows (x {heads_kv} kv-heads)")
    return ids, lens, width, per_head


def prefix_read(
    q: torch.Tensor,
    k_prefix: torch.Tensor,
    v_prefix: torch.Tensor,
    k: torch.Tensor | None = None,
    v: torch.Tensor | None = None,
    read_lists: torch.Tensor | None = None,
    lengths: torch.Tensor | None = None,
    scale: float | None = None,
    prefix_lengths: torch.Tensor | None = None,
    prefix_rows: torch.Tensor | None = None,
    prefix_slots: torch.Tensor | None = None,
    return_lse: bool = False,
):
    """One softmax over a shared prefix and each row's own read list.

    q [B, Tq, Hq, D] (fp32, bf16 or fp16; D 32, 64, 128 or 256; 1, 2, 4 or 8 query heads a
    kv-head). ``k_prefix`` / ``v_prefix`` [P, Tp, Hkv, D] hold P prefixes, or, with
    ``prefix_slots`` [P, Tp] (logical position -> cache row, as a slot table), are one pool
    [1, slots, Hkv, D]; slots outside it are skipped. Every query row reads the first
    ``prefix_lengths[p]`` keys (default: all) of prefix p = ``prefix_rows[b]`` of its batch row
    (default: the only prefix, or prefix b where there are B; one outside [0, P) means none).
    ``k``, ``v``, ``read_lists``, ``lengths``: the own part, as ``lsa_read`` (lists
    [B, Tq, W] or [B, Tq, Hkv, W]; k/v [B or 1, Tk, Hkv, D]); all four or none.
    Where the prefix is read once for the batch its softmax weights are rounded to q's type (by half
    a step at most; the sum that divides them adds the rounded ones); the row forms and ``lsa_read``
    keep them in fp32.

    Returns the output, like q, or with ``return_lse`` also the softmax's logarithm of sums
    [B, Tq, Hq] in fp32 (``key_mass`` takes it). A row with no keys gives zeros and -inf.
    """
    none = k is None
    if (v is None) != none or (read_lists is None) != none or (lengths is None) != none:
        raise ValueError("prefix_read: k, v, read_lists and lengths come together")
    device = one_device("prefix_read", q, k_prefix, v_prefix, k, v)
    if q.dim() != 4 or k_prefix.dim() != 4 or k_prefix.shape != v_prefix.shape:
        raise ValueError(f"prefix_read: q [B, Tq, Hq, D] and prefixes [P, Tp, Hkv, D], got {tuple(q.shape)}, "
                         f"{tuple(k_prefix.shape)} / {tuple(v_prefix.shape)}")
    B, Tq, Hq, D = q.shape
    Hkv = k_prefix.shape[2]
    if k_prefix.shape[3] != D or Hkv < 1 or Hq % Hkv:
        raise ValueError(f"prefix_read: {Hq} query heads of {D} on prefixes {tuple(k_prefix.shape)}")
    dtype = q.dtype
    if k_prefix.dtype != dtype or v_prefix.dtype != dtype or (k is not None and (k.dtype != dtype or v.dtype != dtype)):
        raise ValueError("prefix_read: q, the prefixes and k/v must have one dtype")
    dt = _abi.dtype_code(dtype)
    slots = None
    if prefix_slots is not None:
        if prefix_slots.dim() != 2 or prefix_slots.shape[0] < 1 or k_prefix.shape[0] != 1:
            raise ValueError(f"prefix_read: prefix_slots [P, Tp] over one pool, got {tuple(prefix_slots.shape)} over "
                             f"{tuple(k_prefix.shape)}")
        slots = int32_on(prefix_slots, device)
        P, Tp = slots.shape
        if k_prefix.shape[1] == 0:  # an empty pool: no slot names a row of it
            Tp, slots = 0, None
    else:
        P, Tp = k_prefix.shape[:2]
    if P < 1:
        raise ValueError("prefix_read: no prefix")
    plen = None if prefix_lengths is None else int32_on(prefix_lengths, device)
    if plen is not None and plen.numel() != P:
        raise ValueError(f"prefix_read: {plen.numel()} prefix lengths for {P} prefixes")
    if prefix_rows is not None:
        prow = int32_on(prefix_rows, device)
        if prow.numel() != B:
            raise ValueError(f"prefix_read: {prow.numel()} prefix rows for {B} batch rows")
    elif P in (1, B):
        prow = None
    else:
        raise ValueError(f"prefix_read: prefix_rows is needed: {P} prefixes for {B} batch rows")
    q = aligned(q)
    k_prefix, v_prefix, (psb, pst, psh) = cache_pair(k_prefix, v_prefix)
    Tk = W = sb = st = sh = 0
    ids = lens = None
    per_head = False
    if k is not None:
        if k.dim() != 4 or k.shape != v.shape or k.shape[0] not in (B, 1) or tuple(k.shape[2:]) != (Hkv, D):
            raise ValueError(f"prefix_read: k/v must be [B={B} or 1, Tk, {Hkv}, {D}], got {tuple(k.shape)} / "
                             f"{tuple(v.shape)}")
        Tk = k.shape[1]
        k, v, (sb, st, sh) = cache_pair(k, v)
        ids, lens, W, per_head = lists_of(read_lists, lengths, B * Tq, Hkv, device)
        if Tk == 0:
            W = 0
    out = torch.empty_like(q)
    lse = torch.empty(B, Tq, Hq, dtype=torch.float32, device=device) if return_lse else None
    if B * Tq:
        nbytes = _abi.shape_size("lsa_prefix_read_scratch_bytes", dt, B, Tq, P, Tp, Hq, Hkv, D, W)
        if nbytes > _SLAB_BYTES and B * Tq > 1:  # in halves: query rows, then batch rows
            axis = 1 if Tq > 1 else 0
            if prow is None and P > 1:
                prow = torch.arange(B, dtype=torch.int32, device=device)
            own = [None] * 4
            if W:
                heads = (Hkv,) if per_head else ()
                own = [k, v, ids.view(B, Tq, *heads, W), lens.view(B, Tq, *heads)]
            n = q.shape[axis]
            for at, m in ((0, n // 2), (n // 2, n - n // 2)):
                cut = [x if x is None or (i < 2 and (axis == 1 or x.shape[0] == 1)) else x.narrow(axis, at, m)
                       for i, x in enumerate(own)]
                rows = prow if prow is None or axis == 1 else prow.narrow(0, at, m)
                part = prefix_read(q.narrow(axis, at, m), k_prefix, v_prefix, *cut, scale, plen if Tp else None, rows,
                                   slots, return_lse=True)
                out.narrow(axis, at, m).copy_(part[0])
                if return_lse:
                    lse.narrow(axis, at, m).copy_(part[1])
            return (out, lse) if return_lse else out
        with launch_device(device):
            ws, counters, stream = _abi.call_memory(device, "prefix_read", nbytes, B * Tq * Hkv)
            _abi.call_in_order("lsa_prefix_read", q.data_ptr(), k_prefix.data_ptr(), v_prefix.data_ptr(), dt, B, Tq, P, Tp,
                               k_prefix.shape[1], Hq, Hkv, D, psb, pst, psh, _abi.ptr(prow), _abi.ptr(plen),
                               _abi.ptr(slots), Tp, _abi.ptr(k), _abi.ptr(v),
                               Tk, sb, st, sh, _abi.ptr(ids), _abi.ptr(lens), W, 1 if per_head else 0,
                               float(D ** -0.5 if scale is None else scale), _abi.ptr(counters), _abi.ptr(ws), nbytes,
                               out.data_ptr(), _abi.ptr(lse), stream)
    return (out, lse) if return_lse else out
