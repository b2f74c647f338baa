"""Rotary positions on gfx950 (through libbyteprof_amd.so): queries and keys turned by position x frequency in one launch, and the
frequencies, scaled for contexts longer than a model was trained on."""

from __future__ import annotations

import math
import struct

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from .. import _lib
from .attention import _VALUES, _launch, _no_derivative, _same_device, _span

MAX_HEAD_DIM = 1024
_DESCRIPTION = struct.Struct("6Q9q7if")  # BpRotary of byteprof_amd.h


def rotary_frequencies(dim: int, theta: float = 10000.0, *, scaling: str = "none", factor: float = 1.0, trained: int | None = None,
                       slow: float = 1.0, fast: float = 32.0, device=None) -> tuple[torch.Tensor, float]:
    """(inv_freq [dim / 2] float32, the factor on cosine and sine) for `rotary`: theta ** (-2 i / dim), made for a context
    `factor` times as long as the `trained` positions by

      "none"    nothing
      "linear"  every frequency divided by factor
      "base"    theta replaced by theta factor ** (dim / (dim - 2)): the fastest frequency kept, the slowest divided by factor
      "parts"   frequencies that turn fewer than `slow` times in `trained` positions divided by factor, those that turn more than
                `fast` times kept, a linear ramp in turns between; cosine and sine times 0.1 ln(factor) + 1

    Made on the host, once for a model."""
    if dim < 2 or dim % 2 or not 0.0 < theta < math.inf:
        raise ValueError("rotary_frequencies: dim must be even and positive, theta positive and finite")
    if not 1.0 <= factor < math.inf:
        raise ValueError("rotary_frequencies: factor must be finite and at least 1")
    power = torch.arange(0, dim, 2, dtype=torch.float64) / dim
    freq, by = theta ** -power, 1.0
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "base":
        if dim < 4:
            raise ValueError("rotary_frequencies: a scaled base needs a dim of at least 4")
        freq = (theta * factor ** (dim / (dim - 2))) ** -power
    elif scaling == "parts":
        if trained is None or trained < 1 or not 0.0 <= slow < fast:
            raise ValueError("rotary_frequencies: parts needs the trained positions, and slow below fast")
        keep = ((trained * freq / (2 * math.pi) - slow) / (fast - slow)).clamp(0.0, 1.0)
        freq, by = freq * keep + freq / factor * (1.0 - keep), 0.1 * math.log(factor) + 1.0
    elif scaling != "none":
        raise ValueError(f"rotary_frequencies: no scaling {scaling!r}")
    return freq.float().to(device), by


def _disjoint(x: torch.Tensor, y: torch.Tensor) -> bool:
    """Whether x and y [tokens, heads, D] share no element: their ranges are apart, or they have one token stride and lie in
    different columns of it (slices of one projection)."""
    (a, b), (c, d) = _span(x), _span(y)
    if b <= c or d <= a:
        return True
    step = x.stride(0) * x.element_size()
    if x.shape[0] < 2 or step != y.stride(0) * y.element_size() or step <= 0:
        return False
    rx, ry = (_span(t[:1])[1] - _span(t[:1])[0] for t in (x, y))
    at = (c - a) % step
    return rx <= at and at + ry <= step


def _writable(t: torch.Tensor) -> bool:
    """Whether no two elements of t [tokens, heads, D] share memory."""
    (n, h, d), (st, sh, _) = t.shape, t.stride()
    st, sh = st if n > 1 else h * max(sh, d), sh if h > 1 else d
    return sh >= d and st >= (h - 1) * sh + d or st >= d and sh >= (n - 1) * st + d


_POSITIONS = {torch.int64: 8, torch.int32: 4}


def _outputs(what: str, q: torch.Tensor, k: torch.Tensor | None, out: tuple) -> tuple:
    """out as (q_out, k_out), each like its input and of elements of its own."""
    out = tuple(out)
    if len(out) != 2 or out[0] is None or (out[1] is None) != (k is None):
        raise ValueError(f"{what}: out must be (q_out, k_out), as q and k are given")
    for x, y in zip((q, k), out):
        if y is not None and (y.shape != x.shape or y.dtype != x.dtype or (
                y.numel() and (y.stride(2) != 1 and y.shape[2] > 1 or not _writable(y)))):
            raise ValueError(f"{what}: an output must be like its input, contiguous in the head dimension, each element its own")
    return out


def _apart(what: str, q: torch.Tensor, k: torch.Tensor | None, q_out: torch.Tensor, k_out: torch.Tensor | None,
           *read: torch.Tensor) -> None:
    """Refuses outputs that are neither their own input nor apart from everything else."""
    for y, own, others in ((q_out, q, (k, k_out)), (k_out, k, (q, q_out))):
        if y is None or not y.numel():
            continue
        a, b = _span(y)
        if not (y.data_ptr() == own.data_ptr() and y.stride() == own.stride()) and not _disjoint(y, own) or not all(
                t is None or _disjoint(y, t) for t in others) or any(c < b and a < e for c, e in map(_span, read)):
            raise ValueError(f"{what}: an output must be its own input or apart from everything else")


def rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, inv_freq: torch.Tensor, *, interleaved: bool = False,
           factor: float = 1.0, out: tuple | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """q [tokens, Hq, D] and k [tokens, Hk, D] (or None) at positions [tokens] (int64 or int32): of every head, the first
    2 len(inv_freq) columns in pairs (i, i + len(inv_freq)), interleaved (2 i, 2 i + 1), become
    factor (x1 cos a - x2 sin a, x2 cos a + x1 sin a), a = position x inv_freq[i] (float32); the other columns stay as they are.
    Angles are reduced in 64 bits (right to float32 up to positions of 2 ** 28). bf16, fp16 or fp32, any strides with the last dimension contiguous
    (slices of one projection as they lie). Returns (q, k), contiguous, or in `out` = (q_out, k_out): q and k themselves, or tensors
    of any such strides apart from everything else. Forward only: tensors that require a gradient or carry a forward-mode tangent
    are refused."""
    what = "rotary"
    shape, dtype = q.shape, _VALUES.get(q.dtype)
    if len(shape) != 3:
        raise ValueError(f"{what}: q must be [tokens, Hq, D] and k [tokens, Hk, D]")
    tokens, hq, d = shape
    q_st, hk, k_st = q.stride(), 0, (0, 0, 1)
    if k is not None:
        k_shape, k_st = k.shape, k.stride()
        if len(k_shape) != 3 or k_shape[0] != tokens or k_shape[2] != d:
            raise ValueError(f"{what}: q must be [tokens, Hq, D] and k [tokens, Hk, D]")
        hk = k_shape[1]
    if dtype is None or (k is not None and k.dtype is not q.dtype):
        raise ValueError(f"{what}: q and k must share one dtype, bfloat16, float16 or float32")
    if d > MAX_HEAD_DIM:
        raise ValueError(f"{what}: a head may have {MAX_HEAD_DIM} columns, not {d}")
    if positions.dtype not in _POSITIONS or positions.dim() != 1 or positions.numel() != tokens:
        raise ValueError(f"{what}: positions must be int64 or int32 [tokens]")
    if inv_freq.dtype is not torch.float32 or inv_freq.dim() != 1 or 2 * inv_freq.numel() > d:
        raise ValueError(f"{what}: inv_freq must be float32 [pairs], of at most half of a head's columns")
    if not -3e38 <= factor <= 3e38:
        raise ValueError(f"{what}: factor must be finite in float32")
    if (q_st[2] != 1 or k_st[2] != 1) and d > 1 and (q.numel() if q_st[2] != 1 else k.numel()):
        raise ValueError(f"{what}: q and k must be contiguous in the head dimension")
    q_out, k_out = (None, None) if out is None else _outputs(what, q, k, out)
    index = _same_device(what, q, k, positions, inv_freq, q_out, k_out)
    if q.requires_grad or inv_freq.requires_grad or (k is not None and k.requires_grad) or forward_ad._current_level >= 0:
        _no_derivative(what, q, inv_freq, *(() if k is None else (k,)))
    positions, inv_freq = positions.contiguous(), inv_freq.contiguous()
    if out is None:
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
        if k is not None:
            k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
    else:
        _apart(what, q, k, q_out, k_out, positions, inv_freq)
        increment_version([y for y in (q_out, k_out) if y is not None])
    if tokens and d and (hq or hk):
        k_at, k_out_at, k_out_st = (0, 0, k_st) if k is None else (k.data_ptr(), k_out.data_ptr(), k_out.stride())
        _launch(index, "bp_rotary", _DESCRIPTION.pack(
            q.data_ptr(), k_at, q_out.data_ptr(), k_out_at, positions.data_ptr(), inv_freq.data_ptr(), tokens, *q_st[:2], *k_st[:2],
            *q_out.stride()[:2], *k_out_st[:2], dtype, _POSITIONS[positions.dtype], hq, hk, d, 2 * inv_freq.numel(), interleaved,
            factor))
    return q_out, k_out
