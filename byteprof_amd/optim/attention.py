"""Attention of several sequences on gfx950 (through libbyteprof_amd.so): packed prompts, and chunks of new tokens over a
cache in pages, with the append that writes it.

  packed_attention  whole sequences one after another in [tokens, heads, head_dim]
  paged_append      a chunk's keys and values into the pages
  paged_attention   a chunk of each sequence (one token in a decode step, drafts in a verify round, a part of a prompt) over
                    everything its sequence has in the cache

Offsets, lengths and page tables are int32 tensors on the GPU that the kernels read: the calls neither copy nor synchronise,
and one captured graph serves whatever the tensors hold when it is replayed. bf16 or fp16, softmax and sums in fp32; any
number of query heads to a key head; head_dim a multiple of 8 up to 256. Forward only: a tensor that requires a gradient or
carries a forward-mode tangent is refused. A key or value that a row may not see (past its causal limit) still takes part with
probability 0 where its tile is read, so it has to be finite; what lies past a sequence's length or in other sequences is
never read.
"""

from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from .. import _lib

MAX_HEAD_DIM = 256
UNDIVIDED_KEYS = 256  # a sequence's keys up to here are never divided: no workspace


_FLOATS = {torch.bfloat16: _lib.DT_BF16, torch.float16: _lib.DT_F16}


def _same_device(what: str, x: torch.Tensor, *tensors: torch.Tensor | None) -> int:
    """The index of the GPU that all tensors are on."""
    index = x.get_device()
    if index < 0:
        raise ValueError(f"{what}: the tensors must be on a GPU (there is no CPU path)")
    for t in tensors:
        if t is not None and t.get_device() != index:
            raise ValueError(f"{what}: all tensors must be on {x.device}, got {t.device}")
    return index


def _no_derivative(what: str, *tensors: torch.Tensor) -> None:
    """Refuses tensors that a gradient or (inside a forward-mode level) a tangent would have to be taken through."""
    for t in tensors:
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{what} has no backward pass: detach its inputs or use torch.no_grad()")
        if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError(f"{what} has no forward-mode derivative: pass the primal (torch.autograd.forward_ad.unpack_dual)")


def _ints(what: str, name: str, t: torch.Tensor, dims: int) -> None:
    if t.dtype is not torch.int32 or t.dim() != dims or not (t.is_contiguous() or t.stride(-1) == 1):
        raise ValueError(f"{what}: {name} must be an int32 tensor of {dims} dimension(s), contiguous in the last")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t [.., .., D] itself where the kernel's 16-byte loads can take it as it lies, else a contiguous copy."""
    s0, s1, s2 = t.stride()
    if s2 == 1 and not (t.data_ptr() & 15 or (s0 | s1) & 7):
        return t
    t = t.contiguous()
    return t.clone() if t.data_ptr() & 15 else t


def _scale(what: str, scale: float | None, d: int) -> float:
    if scale is None:
        return d ** -0.5
    scale = float(scale)
    # the kernels multiply by scale log2(e) in float32; a scale that vanishes there would be no scale
    if not 0.0 < ctypes.c_float(ctypes.c_float(scale).value * math.log2(math.e)).value < math.inf:
        raise ValueError(f"{what}: scale must be positive and finite, and so must scale log2(e) in float32")
    return scale


def _dtype(what: str, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> int:
    code = _FLOATS.get(q.dtype)
    if code is None or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"{what}: q, keys and values must share one dtype, bfloat16 or float16")
    return code


def _heads(what: str, hq: int, hk: int, d: int, dk: int) -> None:
    if hk < 1 or hq < 1 or hq % hk:
        raise ValueError(f"{what}: {hq} query heads are no multiple of {hk} key heads")
    if d != dk or d < 8 or d > MAX_HEAD_DIM or d % 8:
        raise ValueError(f"{what}: head_dim must be the same everywhere, a multiple of 8 up to {MAX_HEAD_DIM}")


def _span(t: torch.Tensor) -> tuple[int, int]:
    """The bytes that t reaches over, first and one past the last."""
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride())) if t.numel() else -1
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _output(what: str, q: torch.Tensor, out: torch.Tensor | None, *read: torch.Tensor) -> torch.Tensor:
    if out is None:
        return torch.empty_like(q, memory_format=torch.contiguous_format)
    if out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous() or out.data_ptr() & 15:
        raise ValueError(f"{what}: out must be a contiguous 16-byte aligned {tuple(q.shape)} {q.dtype} tensor")
    first, end = _span(out)
    for t in read if out.data_ptr() == q.data_ptr() and q.is_contiguous() else (q, *read):
        a, b = _span(t)
        if first < b and a < end:
            raise ValueError(f"{what}: out must not overlap what the call reads (but it may be q itself)")
    increment_version(out)  # a graph that has saved it for its backward pass finds out
    return out


def _workspace(tokens: int, seqs: int, hq: int, hk: int, d: int, max_keys: int, device: torch.device):
    if max_keys <= UNDIVIDED_KEYS:
        return None, 0
    need = _lib.lib().bp_attn_workspace_bytes(tokens, seqs, hq, hk, d, max_keys)
    return (torch.empty(need, dtype=torch.uint8, device=device), need) if need else (None, 0)


def _launch(index: int, name: str, *args) -> None:
    """One call of the library on torch's current stream of GPU `index`."""
    if index != torch._C._cuda_getDevice():
        with torch.cuda.device(index):
            return _launch(index, name, *args)
    status = getattr(_lib.lib(), name)(*args, torch._C._cuda_getCurrentRawStream(index))
    if status:
        _lib.check(status, name)


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu: torch.Tensor, *, causal: bool = True,
                     scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of sequences packed one after another: q [tokens, Hq, D], k, v [tokens, Hk, D] (slices of one projection
    may be passed as they lie), cu [sequences + 1] int32 on the GPU with the sequences' first tokens and the end of the last.
    A token sees the tokens of its own sequence, with `causal` those up to itself. scale: D ** -0.5 by default. Rows that no
    sequence covers (a batch padded to a fixed size) come out as zeros. Returns [tokens, Hq, D], in `out` when given:
    q itself or a tensor apart from q, k and v."""
    what = "packed_attention"
    if q.dim() != 3 or k.dim() != 3 or v.shape != k.shape or k.shape[0] != q.shape[0]:
        raise ValueError(f"{what}: q must be [tokens, Hq, D] and k, v [tokens, Hk, D]")
    tokens, hq, d = q.shape
    _, hk, dk = k.shape
    dtype = _dtype(what, q, k, v)
    _heads(what, hq, hk, d, dk)
    _ints(what, "cu", cu, 1)
    seqs = cu.shape[0] - 1
    if seqs < 0:
        raise ValueError(f"{what}: cu needs at least one entry")
    index = _same_device(what, q, k, v, cu, out)
    if q.requires_grad or k.requires_grad or v.requires_grad or forward_ad._current_level >= 0:
        _no_derivative(what, q, k, v)
    scale = _scale(what, scale, d)
    q, k, v = _rows(q), _rows(k), _rows(v)
    y = _output(what, q, out, k, v)
    if tokens == 0:
        return y
    ws, need = _workspace(tokens, seqs, hq, hk, d, tokens, q.device)
    q_t, q_h, _ = q.stride()
    k_t, k_h, _ = k.stride()
    v_t, v_h, _ = v.stride()
    _launch(index, "bp_attn_packed", dtype, q.data_ptr(), k.data_ptr(), v.data_ptr(), y.data_ptr(), cu.data_ptr(), tokens,
            seqs, hq, hk, d, q_t, q_h, k_t, k_h, v_t, v_h, causal, scale, _lib.ptr(ws), need)
    return y


def _pages(what: str, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor,
           cu: torch.Tensor) -> tuple:
    """(pages, page size, Hk, D), the caches' strides, the sequences and the table's width and stride."""
    shape = k_pages.shape
    if len(shape) != 4 or v_pages.shape != shape or shape[1] < 1:
        raise ValueError(f"{what}: the caches must be [pages, page size, Hk, D], keys and values alike")
    kst, vst = k_pages.stride(), v_pages.stride()
    if kst[3] != 1 or vst[3] != 1:
        raise ValueError(f"{what}: the caches must be contiguous in the head dimension")
    _ints(what, "table", table, 2)
    _ints(what, "lengths", lengths, 1)
    _ints(what, "cu", cu, 1)
    (seqs, most), (row, _) = table.shape, table.stride()
    if lengths.shape[0] != seqs or cu.shape[0] != seqs + 1:
        raise ValueError(f"{what}: table [sequences, pages], lengths [sequences] and cu [sequences + 1] disagree")
    if most * shape[1] >= 1 << 29:
        raise ValueError(f"{what}: a sequence may have fewer than 2 ** 29 positions")
    return shape, kst, vst, seqs, most, row


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor,
                    cu: torch.Tensor, *, scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of chunks of new tokens over a cache in pages: q [tokens, Hq, D] with the chunks one after another (cu
    [sequences + 1]), caches [pages, page size, Hk, D], table [sequences, most pages] (position p of sequence b in page
    table[b, p // page size]; entries past its length are not read), lengths [sequences]: a sequence's positions in the
    cache, its chunk's among them (append first). A chunk's tokens are the last positions; each sees all up to its own. Rows
    that no chunk covers come out as zeros. A row that sees a position whose page id is outside the cache is NaN; so may other
    rows of its chunk be.
    Returns [tokens, Hq, D], in `out` when given: q itself or a tensor apart from q and the caches."""
    what = "paged_attention"
    if q.dim() != 3:
        raise ValueError(f"{what}: q must be [tokens, Hq, D]")
    (pool, page, hk, dk), kst, vst, seqs, most, row = _pages(what, k_pages, v_pages, table, lengths, cu)
    tokens, hq, d = q.shape
    dtype = _dtype(what, q, k_pages, v_pages)
    _heads(what, hq, hk, d, dk)
    k_ptr, v_ptr = k_pages.data_ptr(), v_pages.data_ptr()
    if (k_ptr | v_ptr) & 15 or (kst[0] | kst[1] | kst[2] | vst[0] | vst[1] | vst[2]) & 7 and any(
            n > 1 and (a | b) & 7 for n, a, b in zip((pool, page, hk), kst, vst)):
        raise ValueError(f"{what}: the caches must be 16-byte aligned, with strides of whole multiples of 8 elements")
    index = _same_device(what, q, k_pages, v_pages, table, lengths, cu, out)
    if q.requires_grad or k_pages.requires_grad or v_pages.requires_grad or forward_ad._current_level >= 0:
        _no_derivative(what, q, k_pages, v_pages)
    scale = _scale(what, scale, d)
    q = _rows(q)
    y = _output(what, q, out, k_pages, v_pages)
    if tokens == 0:
        return y
    ws, need = _workspace(tokens, seqs, hq, hk, d, page * most, q.device)
    q_t, q_h, _ = q.stride()
    _launch(index, "bp_attn_paged", dtype, q.data_ptr(), k_ptr, v_ptr, y.data_ptr(), table.data_ptr(), row, lengths.data_ptr(),
            cu.data_ptr(), tokens, seqs, pool, page, most, hq, hk, d, q_t, q_h, kst[0], kst[1], kst[2], vst[0], vst[1], vst[2],
            scale, _lib.ptr(ws), need)
    return y


def paged_append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor,
                 lengths: torch.Tensor, cu: torch.Tensor) -> None:
    """The chunks' keys and values k, v [tokens, Hk, D] (any strides with the last dimension contiguous) into the caches, at
    the last positions of each sequence: token i of a chunk of c at position lengths[b] - c + i. Tokens of no chunk, positions
    outside the table (also where lengths[b] is past it, which paged_attention takes as the table's end) and pages outside the
    cache are left out. Any dtype of 1, 2 or 4 bytes; the caches' dtype is k's."""
    what = "paged_append"
    if k.dim() != 3 or v.shape != k.shape:
        raise ValueError(f"{what}: k and v must be [tokens, Hk, D]")
    (pool, page, hk, d), kst, vst, seqs, most, row = _pages(what, k_pages, v_pages, table, lengths, cu)
    tokens, heads, dim = k.shape
    if heads != hk or dim != d:
        raise ValueError(f"{what}: the caches hold {hk} heads of {d}, k and v {heads} of {dim}")
    dtype, size = k.dtype, k.element_size()
    if v.dtype != dtype or k_pages.dtype != dtype or v_pages.dtype != dtype or size not in (1, 2, 4):
        raise ValueError(f"{what}: k, v and the caches must share one dtype of 1, 2 or 4 bytes")
    k_t, k_h, k_d = k.stride()
    v_t, v_h, v_d = v.stride()
    if (k_d != 1 or v_d != 1) and k.numel():
        raise ValueError(f"{what}: k and v must be contiguous in the head dimension")
    index = _same_device(what, k, v, k_pages, v_pages, table, lengths, cu)
    if k.requires_grad or v.requires_grad or k_pages.requires_grad or v_pages.requires_grad or forward_ad._current_level >= 0:
        _no_derivative(what, k, v, k_pages, v_pages)
    if tokens == 0 or hk == 0 or d == 0:
        return
    _launch(index, "bp_paged_append", size, k.data_ptr(), v.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
            table.data_ptr(), row, lengths.data_ptr(), cu.data_ptr(), tokens, seqs, pool, page, most, hk, d, k_t, k_h, v_t, v_h,
            kst[0], kst[1], kst[2], vst[0], vst[1], vst[2])
    increment_version((k_pages, v_pages))
