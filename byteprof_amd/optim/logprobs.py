"""Log probabilities of given tokens with the entropy and the most likely tokens, on gfx950 (through libbyteprof_amd.so): one
pass over the logits of a language model's head."""

from __future__ import annotations

from typing import NamedTuple

import torch

from .. import _lib
from .attention import _launch, _no_grad, _same_device

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
    only: logits that require a gradient are refused."""
    what = "token_logprobs"
    if logits.dim() != 2 or (logits.numel() and (logits.stride(1) != 1 or logits.stride(0) < 0)):
        raise ValueError(f"{what}: logits must be [rows, vocab], each row contiguous")
    rows, vocab = logits.shape
    if logits.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise ValueError(f"{what}: logits must be bfloat16, float16 or float32")
    if not 0 <= top <= MAX_TOP or (rows and top > vocab):
        raise ValueError(f"{what}: top must be 0..{MAX_TOP} and at most the vocabulary, got {top}")
    if rows and not 1 <= vocab < 1 << 30:
        raise ValueError(f"{what}: the vocabulary must have 1 to 2 ** 30 - 1 tokens")
    if targets is not None and (targets.dtype != torch.int64 or targets.shape != (rows,)):
        raise ValueError(f"{what}: targets must be int64 [rows]")
    _same_device(what, logits.device, targets)
    _no_grad(what, logits)
    dev = logits.device
    f32 = lambda *shape: torch.empty(*shape, dtype=torch.float32, device=dev)  # noqa: E731
    out = TokenLogprobs(None if targets is None else f32(rows), f32(rows),
                        torch.empty(rows, top, dtype=torch.int64, device=dev), f32(rows, top))
    if rows == 0:
        return out
    if targets is not None:
        targets = targets.contiguous()
    dt = _lib.TORCH_DT[logits.dtype]
    need = _lib.lib().bp_logprobs_workspace_bytes(dt, rows, vocab, top)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _launch(dev, "bp_logprobs", dt, logits.data_ptr(), logits.stride(0), _lib.ptr(targets), _lib.ptr(out.logprob),
            out.entropy.data_ptr(), out.top_ids.data_ptr(), out.top_logprobs.data_ptr(), rows, vocab, top, _lib.ptr(ws), need)
    return out
