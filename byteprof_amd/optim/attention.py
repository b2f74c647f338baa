"""Attention of several sequences on gfx950 (through libbyteprof_amd.so): packed prompts, and chunks of new tokens over a
cache in pages, with the append that writes it.

  packed_attention  whole sequences one after another in [tokens, heads, head_dim]
  paged_append      a chunk's keys and values into the pages
  paged_attention   a chunk of each sequence (one token in a decode step, drafts in a verify round, a part of a prompt) over
                    everything its sequence has in the cache

Offsets, lengths and page tables are int32 tensors on the GPU that the kernels read: the calls neither copy nor synchronise,
and one captured graph serves whatever the tensors hold when it is replayed. bf16 or fp16, softmax and sums in fp32; any
number of query heads to a key head; head_dim a multiple of 8 up to 256. Forward only: a tensor that requires a gradient is
refused. A key or value that a row may not see (past its causal limit) still takes part with probability 0 where its tile is
read, so it has to be finite; what lies past a sequence's length or in other sequences is never read.
"""

from __future__ import annotations

import torch

from .. import _lib

MAX_HEAD_DIM = 256


def _same_device(what: str, device: torch.device, *tensors: torch.Tensor | None) -> None:
    if device.type != "cuda":
        raise ValueError(f"{what}: the tensors must be on a GPU (there is no CPU path)")
    for t in tensors:
        if t is not None and t.device != device:
            raise ValueError(f"{what}: all tensors must be on {device}, got {t.device}")


def _no_grad(what: str, *tensors: torch.Tensor) -> None:
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise ValueError(f"{what} has no backward pass: detach its inputs or use torch.no_grad()")


def _ints(what: str, name: str, t: torch.Tensor, dims: int) -> None:
    if t.dtype != torch.int32 or t.dim() != dims or (t.numel() > 0 and t.stride(-1) != 1):
        raise ValueError(f"{what}: {name} must be an int32 tensor of {dims} dimension(s), contiguous in the last")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t itself where the kernel's 16-byte loads can take it as it lies, else a contiguous copy."""
    st = t.stride()
    if st[-1] == 1 and t.data_ptr() % 16 == 0 and all(s % 8 == 0 for s in st[:-1]):
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _scale(what: str, scale: float | None, d: int) -> float:
    scale = d ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < float("inf"):
        raise ValueError(f"{what}: scale must be positive and finite")
    return scale


def _heads(what: str, q: torch.Tensor, hk: int, d: int, *others: torch.Tensor) -> None:
    if q.dtype not in (torch.bfloat16, torch.float16) or any(t.dtype != q.dtype for t in others):
        raise ValueError(f"{what}: q, keys and values must share one dtype, bfloat16 or float16")
    if hk < 1 or q.shape[1] < 1 or q.shape[1] % hk:
        raise ValueError(f"{what}: {q.shape[1]} query heads are no multiple of {hk} key heads")
    if q.shape[2] != d or d < 8 or d > MAX_HEAD_DIM or d % 8:
        raise ValueError(f"{what}: head_dim must be the same everywhere, a multiple of 8 up to {MAX_HEAD_DIM}")


def _output(what: str, q: torch.Tensor, out: torch.Tensor | None) -> torch.Tensor:
    if out is None:
        return torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError(f"{what}: out must be a contiguous 16-byte aligned {tuple(q.shape)} {q.dtype} tensor")
    return out


def _workspace(tokens: int, seqs: int, hq: int, hk: int, d: int, max_keys: int, device: torch.device):
    need = _lib.lib().bp_attn_workspace_bytes(tokens, seqs, hq, hk, d, max_keys)
    return (torch.empty(need, dtype=torch.uint8, device=device), need) if need else (None, 0)


def _launch(device: torch.device, name: str, *args) -> None:
    """One call of the library on torch's current stream of `device`."""
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _launch(device, name, *args)
    _lib.check(getattr(_lib.lib(), name)(*args, _lib.stream_ptr(device)), name)


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu: torch.Tensor, *, causal: bool = True,
                     scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of sequences packed one after another: q [tokens, Hq, D], k, v [tokens, Hk, D] (slices of one projection
    may be passed as they lie), cu [sequences + 1] int32 on the GPU with the sequences' first tokens and the end of the last.
    A token sees the tokens of its own sequence, with `causal` those up to itself. scale: D ** -0.5 by default. Rows that no
    sequence covers (a batch padded to a fixed size) come out as zeros. Returns [tokens, Hq, D], in `out` when given."""
    what = "packed_attention"
    if q.dim() != 3 or k.dim() != 3 or v.shape != k.shape or k.shape[0] != q.shape[0]:
        raise ValueError(f"{what}: q must be [tokens, Hq, D] and k, v [tokens, Hk, D]")
    tokens, hq, d = q.shape
    hk = k.shape[1]
    _heads(what, q, hk, k.shape[2], k, v)
    _ints(what, "cu", cu, 1)
    if cu.shape[0] < 1:
        raise ValueError(f"{what}: cu needs at least one entry")
    _same_device(what, q.device, k, v, cu, out)
    _no_grad(what, q, k, v)
    scale = _scale(what, scale, d)
    q, k, v = _rows(q), _rows(k), _rows(v)
    y = _output(what, q, out)
    if tokens == 0:
        return y
    seqs = cu.shape[0] - 1
    ws, need = _workspace(tokens, seqs, hq, hk, d, tokens, q.device)
    _launch(q.device, "bp_attn_packed", _lib.TORCH_DT[q.dtype], q.data_ptr(), k.data_ptr(), v.data_ptr(), y.data_ptr(),
            cu.data_ptr(), tokens, seqs, hq, hk, d, q.stride(0), q.stride(1), k.stride(0), k.stride(1), v.stride(0),
            v.stride(1), int(causal), scale, _lib.ptr(ws), need)
    return y


def _pages(what: str, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor,
           cu: torch.Tensor) -> None:
    if k_pages.dim() != 4 or v_pages.shape != k_pages.shape or k_pages.shape[1] < 1:
        raise ValueError(f"{what}: the caches must be [pages, page size, Hk, D], keys and values alike")
    if k_pages.stride(3) != 1 or v_pages.stride(3) != 1:
        raise ValueError(f"{what}: the caches must be contiguous in the head dimension")
    _ints(what, "table", table, 2)
    _ints(what, "lengths", lengths, 1)
    _ints(what, "cu", cu, 1)
    if cu.shape[0] < 1 or lengths.shape[0] != cu.shape[0] - 1 or table.shape[0] != lengths.shape[0]:
        raise ValueError(f"{what}: table [sequences, pages], lengths [sequences] and cu [sequences + 1] disagree")
    if table.shape[1] * k_pages.shape[1] >= 1 << 29:
        raise ValueError(f"{what}: a sequence may have fewer than 2 ** 29 positions")


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor,
                    cu: torch.Tensor, *, scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of chunks of new tokens over a cache in pages: q [tokens, Hq, D] with the chunks one after another (cu
    [sequences + 1]), caches [pages, page size, Hk, D], table [sequences, most pages] (position p of sequence b in page
    table[b, p // page size]; entries past its length are not read), lengths [sequences]: a sequence's positions in the
    cache, its chunk's among them (append first). A chunk's tokens are the last positions; each sees all up to its own. Rows
    that no chunk covers come out as zeros; rows of a sequence with a page id outside the cache below its length as NaN.
    Returns [tokens, Hq, D], in `out` when given."""
    what = "paged_attention"
    if q.dim() != 3:
        raise ValueError(f"{what}: q must be [tokens, Hq, D]")
    _pages(what, k_pages, v_pages, table, lengths, cu)
    tokens, hq, d = q.shape
    pool, page, hk, _ = k_pages.shape
    _heads(what, q, hk, k_pages.shape[3], k_pages, v_pages)
    for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
        if t.data_ptr() % 16 or any(s % 8 for s in t.stride()[:3]):
            raise ValueError(f"{what}: {name} must be 16-byte aligned, with strides of whole multiples of 8 elements")
    _same_device(what, q.device, k_pages, v_pages, table, lengths, cu, out)
    _no_grad(what, q, k_pages, v_pages)
    scale = _scale(what, scale, d)
    q = _rows(q)
    y = _output(what, q, out)
    if tokens == 0:
        return y
    seqs, most = table.shape
    ws, need = _workspace(tokens, seqs, hq, hk, d, page * most, q.device)
    kst, vst = k_pages.stride(), v_pages.stride()
    _launch(q.device, "bp_attn_paged", _lib.TORCH_DT[q.dtype], q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
            y.data_ptr(), table.data_ptr(), table.stride(0), lengths.data_ptr(), cu.data_ptr(), tokens, seqs, pool, page, most,
            hq, hk, d, q.stride(0), q.stride(1), kst[0], kst[1], kst[2], vst[0], vst[1], vst[2], scale, _lib.ptr(ws), need)
    return y


def paged_append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor,
                 lengths: torch.Tensor, cu: torch.Tensor) -> None:
    """The chunks' keys and values k, v [tokens, Hk, D] (any strides with the last dimension contiguous) into the caches, at
    the last positions of each sequence: token i of a chunk of c at position lengths[b] - c + i. Tokens of no chunk, positions
    outside the table and pages outside the cache are left out. Any dtype of 1, 2 or 4 bytes; the caches' dtype is k's."""
    what = "paged_append"
    if k.dim() != 3 or v.shape != k.shape:
        raise ValueError(f"{what}: k and v must be [tokens, Hk, D]")
    _pages(what, k_pages, v_pages, table, lengths, cu)
    pool, page, hk, d = k_pages.shape
    if k.shape[1:] != (hk, d):
        raise ValueError(f"{what}: the caches hold {hk} heads of {d}, k and v {k.shape[1]} of {k.shape[2]}")
    if k.dtype != v.dtype or k_pages.dtype != k.dtype or v_pages.dtype != k.dtype or k.element_size() not in (1, 2, 4):
        raise ValueError(f"{what}: k, v and the caches must share one dtype of 1, 2 or 4 bytes")
    if k.numel() and (k.stride(2) != 1 or v.stride(2) != 1):
        raise ValueError(f"{what}: k and v must be contiguous in the head dimension")
    _same_device(what, k.device, v, k_pages, v_pages, table, lengths, cu)
    _no_grad(what, k, v, k_pages, v_pages)
    if k.numel() == 0:
        return
    seqs, most = table.shape
    kst, vst = k_pages.stride(), v_pages.stride()
    _launch(k.device, "bp_paged_append", k.element_size(), k.data_ptr(), v.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
            table.data_ptr(), table.stride(0), lengths.data_ptr(), cu.data_ptr(), k.shape[0], seqs, pool, page, most, hk, d,
            k.stride(0), k.stride(1), v.stride(0), v.stride(1), kst[0], kst[1], kst[2], vst[0], vst[1], vst[2])
