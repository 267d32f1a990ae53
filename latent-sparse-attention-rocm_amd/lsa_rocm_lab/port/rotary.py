"""Norms of query and key heads and their rotary positions.

``rotate`` takes the heads of a projection to what the index and the reads work on: each head's RMS
norm (where its weight is given), then its rotary position, in one pass over q and k.
``rotary_frequencies`` makes the pairs' frequencies, also for contexts longer than trained on.
``byte_append`` does the same on the way into an 8-bit cache. No counterpart in the reference.
"""

from __future__ import annotations

import ctypes
import math

import torch

from lsa_rocm_lab import _abi
from lsa_rocm_lab.port.shared_prefix import aligned, launch_device, one_device


def rotary_frequencies(
    dim: int,
    base: float = 10000.0,
    scaling: str = "none",
    factor: float = 1.0,
    original: int = 0,
    low: float = 1.0,
    high: float = 4.0,
    device: torch.device | str | None = None,
    dtype: torch.dtype = torch.float32,
) -> torch.Tensor:
    """Frequencies [dim / 2] of the pairs of a head's ``dim`` rotated dims: ``base ** (-2 j / dim)``.

    ``scaling`` for contexts ``factor`` times as long: ``"linear"`` divides all of them by it;
    ``"base"`` raises the base by ``factor ** (dim / (dim - 2))``, so that the slowest pair slows by
    ``factor`` and the fastest not at all; ``"parts"`` goes by how often a pair turns in the
    ``original`` context: at most ``low`` times, divided by ``factor``; at least ``high`` times,
    kept; linear in the turns between. Computed in fp64 and rounded to ``dtype`` (fp32 or fp64).
    """
    if dim < 2 or dim % 2:
        raise ValueError(f"rotary_frequencies: an even number of dims, got {dim}")
    if dtype not in (torch.float32, torch.float64):
        raise ValueError(f"rotary_frequencies: fp32 or fp64, got {dtype}")
    if not (base > 0.0 and math.isfinite(base) and factor > 0.0 and math.isfinite(factor)):
        raise ValueError(f"rotary_frequencies: base {base} and factor {factor} must be positive")
    j = torch.arange(dim // 2, dtype=torch.float64)
    if scaling == "base" and dim > 2:
        base = base * factor ** (dim / (dim - 2))
    freq = base ** (-2.0 * j / dim)
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "parts":
        if original < 1 or not low < high:
            raise ValueError(f"rotary_frequencies: parts of an original context, low < high; got {original}, {low}, {high}")
        keep = ((original * freq / (2.0 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
        freq = freq * (keep + (1.0 - keep) / factor)
    elif scaling not in ("none", "base"):
        raise ValueError(f"rotary_frequencies: scaling none|linear|base|parts, got {scaling!r}")
    return freq.to(device=device, dtype=dtype)


class _Turn(ctypes.Structure):
    """``lsa_turn`` (include/lsa_rocm.h)."""

    _fields_ = [("frequencies", ctypes.c_void_p), ("q_weight", ctypes.c_void_p), ("k_weight", ctypes.c_void_p),
                ("pairs", ctypes.c_int32), ("frequencies_f64", ctypes.c_int32), ("interleaved", ctypes.c_int32),
                ("weights_f32", ctypes.c_int32), ("eps", ctypes.c_float), ("magnitude", ctypes.c_float)]


def turn_of(what: str, device: torch.device, D: int, dtype: torch.dtype, frequencies, q_weight, k_weight, eps: float,
            interleaved: bool, magnitude: float):
    """``const lsa_turn*`` of a call, and the tensors it points at (alive until the launch)."""
    pairs = f64 = 0
    if D not in (32, 64, 128, 256):
        raise ValueError(f"{what}: head dim {D} not in 32, 64, 128, 256")
    if frequencies is not None:
        if frequencies.dim() != 1 or frequencies.device != device:
            raise ValueError(f"{what}: frequencies [pairs] on {device}, got {tuple(frequencies.shape)} on {frequencies.device}")
        pairs = frequencies.shape[0]
        if 2 * pairs > D:
            raise ValueError(f"{what}: {pairs} pairs in heads of {D}")
        if frequencies.dtype not in (torch.float32, torch.float64):
            raise ValueError(f"{what}: frequencies in fp32 or fp64, got {frequencies.dtype}")
        if pairs > 1 and frequencies.stride(0) != 1:
            frequencies = frequencies.contiguous()
        f64 = 1 if frequencies.dtype is torch.float64 else 0
    if not eps >= 0.0:
        raise ValueError(f"{what}: eps {eps}")
    f32 = 0
    qw = kw = None
    if q_weight is not None or k_weight is not None:
        for w in (q_weight, k_weight):
            if w is None:
                continue
            if w.shape != (D,) or w.device != device or (w.dtype is not dtype and w.dtype is not torch.float32):
                raise ValueError(f"{what}: norm weights [{D}] in {dtype} or fp32 on {device}, got {w.dtype} "
                                 f"{tuple(w.shape)} on {w.device}")
            if w.dtype is torch.float32:
                f32 = 1
        qw, kw = _weight(q_weight, f32), _weight(k_weight, f32)
    turn = _Turn(frequencies.data_ptr() if pairs else None, None if qw is None else qw.data_ptr(),
                 None if kw is None else kw.data_ptr(), pairs, f64, 1 if interleaved else 0, f32, eps, magnitude)
    return turn, (frequencies, qw, kw)


def _weight(w: torch.Tensor | None, f32: int) -> torch.Tensor | None:
    """A norm's weight as the kernels read it: dense, 16-byte aligned, in fp32 where one of the two is."""
    if w is None:
        return None
    if f32 and w.dtype is not torch.float32:
        w = w.float()
    return w if w.stride(0) == 1 and not w.data_ptr() & 15 else aligned(w)


def head_rows(x: torch.Tensor):
    """Heads [B, T, H, D] as a kernel reads them (a view of a wider projection in place, if its rows are
    contiguous and 16-byte aligned; else made dense) and their batch, token and head strides."""
    sb, st, sh, sd = x.stride()
    B, T, H, _ = x.shape
    sb, st, sh = sb if B > 1 else 0, st if T > 1 else 0, sh if H > 1 else 0
    if sd != 1 or x.data_ptr() & 15 or (sb | st | sh) & (3 if x.dtype is torch.float32 else 7):
        x = aligned(x)
        sb, st, sh, _ = x.stride()
    return x, sb, st, sh


def rotate(
    q: torch.Tensor,
    k: torch.Tensor | None,
    positions: torch.Tensor | None,
    frequencies: torch.Tensor | None,
    q_weight: torch.Tensor | None = None,
    k_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    interleaved: bool = False,
    magnitude: float = 1.0,
):
    """The heads of q [B, T, Hq, D] and k [B, T, Hkv, D] (or None), normed and rotated.

    With a weight [D] a head x becomes ``x / sqrt(mean(x^2) + eps) * weight``. Its first
    ``2 * len(frequencies)`` dims are then rotated in pairs, by ``position * frequencies[j]``: dims j and
    j + len(frequencies), or, ``interleaved``, 2j and 2j + 1; cosine and sine are multiplied by
    ``magnitude``; the other dims stay. ``positions`` [B, T] or [T], int32 or int64. fp32, bf16 or fp16;
    D 32, 64, 128 or 256; views with contiguous, 16-byte aligned rows are read in place. Angles are
    taken in fp64, the rest in fp32 and rounded once. Returns (q, k), new and dense.
    """
    device = one_device("rotate", q, k)
    if q.dim() != 4 or (k is not None and (k.dim() != 4 or k.shape[:2] != q.shape[:2] or k.shape[3] != q.shape[3])):
        raise ValueError(f"rotate: q [B, T, Hq, D] and k [B, T, Hkv, D], got {tuple(q.shape)} and "
                         f"{None if k is None else tuple(k.shape)}")
    if k is not None and k.dtype != q.dtype:
        raise ValueError(f"rotate: q/k dtypes differ: {q.dtype} {k.dtype}")
    dt = _abi.dtype_code(q.dtype)
    B, T, Hq, D = q.shape
    turn, _keep = turn_of("rotate", device, D, q.dtype, frequencies, q_weight, k_weight, eps, interleaved, magnitude)
    i64 = stride = 0
    if turn.pairs:
        if positions is None or positions.shape not in ((B, T), (T,)) or positions.device != device:
            raise ValueError(f"rotate: positions [{B}, {T}] or [{T}] on {device}, got "
                             f"{None if positions is None else (tuple(positions.shape), positions.device)}")
        if positions.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"rotate: positions in int32 or int64, got {positions.dtype}")
        i64 = 1 if positions.dtype is torch.int64 else 0
        if T > 1 and positions.stride(-1) != 1:
            positions = positions.contiguous()
        stride = positions.stride(0) if positions.dim() == 2 and B > 1 else 0
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if Hq == 0 and k is not None and k.numel():  # the keys alone
        return q_out, rotate(k, None, positions, frequencies, k_weight, None, eps, interleaved, magnitude)[0]
    k_out = None if k is None else torch.empty_like(k, memory_format=torch.contiguous_format)
    if q.numel() == 0:
        return q_out, k_out
    q, qsb, qst, qsh = head_rows(q)
    Hkv = ksb = kst = ksh = 0
    if k is not None:
        Hkv = k.shape[2]
        k, ksb, kst, ksh = head_rows(k)
    with launch_device(device):
        _abi.call("lsa_rotate", q.data_ptr(), _abi.ptr(k), dt, B, T, Hq, Hkv, D, qsb, qst, qsh, ksb, kst, ksh,
                  _abi.ptr(positions) if turn.pairs else None, i64, stride, ctypes.addressof(turn), q_out.data_ptr(),
                  _abi.ptr(k_out), _abi.stream(device))
    return q_out, k_out
