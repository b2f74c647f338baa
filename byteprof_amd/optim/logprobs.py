"""Log probabilities of given tokens with the entropy and the most likely tokens, on gfx950 (through libbyteprof_amd.so): one
pass over the logits of a language model's head."""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from .. import _lib
from .attention import _launch, _no_derivative, _same_device

MAX_TOP = 32


class TokenLogprobs(NamedTuple):
    """logprob [rows] (None without targets) and entropy [rows] in nats, top_ids [rows, top] int64, top_logprobs [rows, top];
    float32 but for the ids."""

    logprob: torch.Tensor | None
    entropy: torch.Tensor
    top_ids: torch.Tensor
    top_logprobs: torch.Tensor


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor | None = None, *, top: int = 0) -> TokenLogprobs:
    """logits [rows, vocab] (bf16, fp16 or fp32; each row contiguous, rows any distance apart), targets [rows] int64: the log
    softmax at each row's target (NaN for one outside the vocabulary), the entropy of the row, and its `top` (up to MAX_TOP)
    most likely tokens in order; equal logits in order of their ids. -inf logits are tokens that cannot come. A row with a
    NaN or +inf has NaN probabilities (NaN counts as greatest in the order), and so has a row of nothing but -inf. Forward
    only: logits that require a gradient or carry a forward-mode tangent are refused."""
    what = "token_logprobs"
    if logits.dim() != 2:
        raise ValueError(f"{what}: logits must be [rows, vocab], each row contiguous")
    rows, vocab = logits.shape
    row, inner = logits.stride()
    if (inner != 1 and vocab > 1) or row < 0:
        raise ValueError(f"{what}: logits must be [rows, vocab], each row contiguous")
    dtype = _lib.TORCH_DT.get(logits.dtype, _lib.DT_I8)
    if dtype == _lib.DT_I8:
        raise ValueError(f"{what}: logits must be bfloat16, float16 or float32")
    if not 0 <= top <= MAX_TOP or (rows and top > vocab):
        raise ValueError(f"{what}: top must be 0..{MAX_TOP} and at most the vocabulary, got {top}")
    if rows and not 1 <= vocab < 1 << 30:
        raise ValueError(f"{what}: the vocabulary must have 1 to 2 ** 30 - 1 tokens")
    if targets is not None and (targets.dtype != torch.int64 or targets.shape != (rows,)):
        raise ValueError(f"{what}: targets must be int64 [rows]")
    index = _same_device(what, logits, targets)
    if logits.requires_grad or forward_ad._current_level >= 0:
        _no_derivative(what, logits)
    dev = logits.device
    f32 = torch.float32
    logprob = None if targets is None else torch.empty_strided((rows,), (1,), dtype=f32, device=dev)
    entropy = torch.empty_strided((rows,), (1,), dtype=f32, device=dev)
    ids = torch.empty_strided((rows, top), (top, 1), dtype=torch.int64, device=dev)
    tops = torch.empty_strided((rows, top), (top, 1), dtype=f32, device=dev)
    out = TokenLogprobs(logprob, entropy, ids, tops)
    if rows == 0:
        return out
    if targets is not None and rows > 1:
        targets = targets.contiguous()
    need = _lib.lib().bp_logprobs_workspace_bytes(dtype, rows, vocab, top)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _launch(index, "bp_logprobs", dtype, logits.data_ptr(), row, _lib.ptr(targets), _lib.ptr(logprob), entropy.data_ptr(),
            ids.data_ptr(), tops.data_ptr(), rows, vocab, top, _lib.ptr(ws), need)
    return out
