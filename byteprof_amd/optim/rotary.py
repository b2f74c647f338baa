"""Rotary positions on gfx950 (through libbyteprof_amd.so): queries and keys turned by position x frequency in one launch, and the
frequencies, scaled for contexts longer than a model was trained on."""

from __future__ import annotations

import math

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from .. import _lib
from .attention import _VALUES, _launch, _no_derivative, _same_device, _span

MAX_HEAD_DIM = 1024


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


def rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, inv_freq: torch.Tensor, *, interleaved: bool = False,
           factor: float = 1.0, out: tuple | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """q [tokens, Hq, D] and k [tokens, Hk, D] (or None) at positions [tokens] (int64 or int32): of every head, the first
    2 len(inv_freq) columns in pairs (i, i + len(inv_freq)), interleaved (2 i, 2 i + 1), become
    factor (x1 cos a - x2 sin a, x2 cos a + x1 sin a), a = position x inv_freq[i] (float32); the other columns stay as they are.
    Angles are right at any position (reduced in 64 bits). bf16, fp16 or fp32, any strides with the last dimension contiguous
    (slices of one projection as they lie). Returns (q, k), contiguous, or in `out` = (q_out, k_out): q and k themselves, or tensors
    of any such strides apart from everything else. Forward only: tensors that require a gradient or carry a forward-mode tangent
    are refused."""
    what = "rotary"
    if q.dim() != 3 or (k is not None and (k.dim() != 3 or k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2])):
        raise ValueError(f"{what}: q must be [tokens, Hq, D] and k [tokens, Hk, D]")
    tokens, hq, d = q.shape
    dtype = _VALUES.get(q.dtype)
    if dtype is None or (k is not None and k.dtype != q.dtype):
        raise ValueError(f"{what}: q and k must share one dtype, bfloat16, float16 or float32")
    if d > MAX_HEAD_DIM:
        raise ValueError(f"{what}: a head may have {MAX_HEAD_DIM} columns, not {d}")
    if positions.dtype not in (torch.int64, torch.int32) or positions.shape != (tokens,):
        raise ValueError(f"{what}: positions must be int64 or int32 [tokens]")
    if inv_freq.dtype is not torch.float32 or inv_freq.dim() != 1 or 2 * inv_freq.shape[0] > d:
        raise ValueError(f"{what}: inv_freq must be float32 [pairs], of at most half of a head's columns")
    if not math.isfinite(factor) or abs(factor) > 3e38:
        raise ValueError(f"{what}: factor must be finite in float32")
    given = [t for t in (q, k) if t is not None]
    if any(t.stride(2) != 1 and d > 1 and t.numel() for t in given):
        raise ValueError(f"{what}: q and k must be contiguous in the head dimension")
    outs = (None, None) if out is None else tuple(out)
    if len(outs) != 2 or (out is not None and (outs[0] is None or (outs[1] is None) != (k is None))):
        raise ValueError(f"{what}: out must be (q_out, k_out), as q and k are given")
    index = _same_device(what, q, k, positions, inv_freq, *outs)
    if any(t.requires_grad for t in given) or inv_freq.requires_grad or forward_ad._current_level >= 0:
        _no_derivative(what, *given, inv_freq)
    positions, inv_freq = positions.contiguous(), inv_freq.contiguous()
    if out is None:
        outs = tuple(None if t is None else torch.empty_like(t, memory_format=torch.contiguous_format) for t in (q, k))
    else:
        for i, (t, y) in enumerate(zip((q, k), outs)):
            if y is None:
                continue
            if y.shape != t.shape or y.dtype != t.dtype or (y.stride(2) != 1 and d > 1) or (y.numel() and not _writable(y)):
                raise ValueError(f"{what}: an output must be like its input, contiguous in the head dimension, each element its own")
            others = [x for j, x in enumerate((q, k)) if x is not None
                      and not (i == j and x.data_ptr() == y.data_ptr() and x.stride() == y.stride())]
            others += [x for j, x in enumerate(outs) if x is not None and j != i]
            a, b = _span(y)
            apart = all(_disjoint(y, x) for x in others) and all(
                b <= c or e <= a for c, e in map(_span, (positions, inv_freq)))
            if y.numel() and not apart:
                raise ValueError(f"{what}: an output must be its own input or apart from everything else")
        increment_version([y for y in outs if y is not None])
    if tokens == 0 or d == 0:
        return outs
    (q_t, q_h, _), (qo_t, qo_h, _) = q.stride(), outs[0].stride()
    hk = k_t = k_h = ko_t = ko_h = 0
    if k is not None:
        hk, (k_t, k_h, _), (ko_t, ko_h, _) = k.shape[1], k.stride(), outs[1].stride()
    if hq + hk:
        _launch(index, "bp_rotary", dtype, q.data_ptr(), _lib.ptr(k), outs[0].data_ptr(), _lib.ptr(outs[1]), positions.data_ptr(),
                positions.element_size(), inv_freq.data_ptr(), tokens, hq, hk, d, 2 * inv_freq.shape[0], interleaved, factor, q_t, q_h,
                k_t, k_h, qo_t, qo_h, ko_t, ko_h)
    return outs
