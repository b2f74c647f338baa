"""Several sequences at once on an OlmoDecoder's weights: prompts run packed (packed_attention), their keys and values go into
a cache in pages (paged_append) that the steps of all sequences read together (paged_attention), and tokens come with their log
probabilities (token_logprobs). The single-sequence loops of olmo.py are not touched; the linears are the decoder's own
(skinny_mm on its bf16, int8 or int4 weights, rows independent of each other), so are the norm and SiLU kernels.

  batch = OlmoBatch(dec, pages=512)
  scores = batch.score([ids_a, ids_b], top=5)             # of every prompt token after the first
  outs = batch.generate([ids_a, ids_b], max_new_tokens=32, top=5)

The cache may be held in 8 bits (cache=torch.float8_e4m3fn or torch.int8: half the memory, and the steps' attention reads half as
much; prompts still run over their own 16-bit keys and values), and positions may turn by frequencies of the program's own
(rotary=rotary_frequencies(...), made for contexts longer than the decoder's).

Greedy; a sequence ends after an EOS id or max_new_tokens. Pages are taken when a call begins and given back when it ends.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from .. import _lib
from . import skinny as S
from .attention import packed_attention, paged_append, paged_attention
from .logprobs import MAX_TOP, TokenLogprobs, token_logprobs
from .olmo import OlmoDecoder, OptimizeError
from .rotary import rotary as rotate


class Generated(NamedTuple):
    """The new tokens [n] of one sequence with, per token, its log probability [n], the entropy [n] of the distribution it was
    taken from, and that distribution's most likely tokens [n, top]."""

    tokens: torch.Tensor
    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_ids: torch.Tensor
    top_logprobs: torch.Tensor


class OlmoBatch:
    """pages x page positions of cache for every layer of `dec`, of dtype `cache`: bfloat16, or (pages of a multiple of 4 positions)
    8-bit codes with a scale for each head and block of 16 positions (12, 8 or 4 where 16 does not divide a page). rotary:
    (inv_freq [head_dim / 2], factor) on the decoder's device; by default the decoder's own frequencies, their angles rounded to
    float32 as its own loops have them where the cache is bfloat16. That takes several launches of elementary torch a layer:
    rotary=(dec.inv_freq, 1.0) turns by the same frequencies in one (8 sequences, 16 layers of 16 heads of 128 columns: a step of
    3.7 ms becomes 2.4)."""

    def __init__(self, dec: OlmoDecoder, pages: int, page: int = 16, *, cache: torch.dtype = torch.bfloat16,
                 rotary: tuple[torch.Tensor, float] | None = None):
        if pages < 1 or page < 1:
            raise ValueError("the cache needs at least one page of at least one position")
        if cache not in (torch.bfloat16, torch.float8_e4m3fn, torch.int8):
            raise ValueError(f"the cache is held in bfloat16, float8_e4m3fn or int8, not {cache}")
        if cache != torch.bfloat16 and page % 4:
            raise ValueError(f"an 8-bit cache needs pages of a multiple of 4 positions, not {page}")
        cfg = dec.cfg
        if rotary is not None:
            inv_freq, factor = rotary if isinstance(rotary, (tuple, list)) and len(rotary) == 2 else (None, 0.0)
            if (not isinstance(inv_freq, torch.Tensor) or inv_freq.dtype is not torch.float32 or inv_freq.shape != (cfg.head_dim // 2,)
                    or inv_freq.device != dec.inv_freq.device or not -3e38 <= factor <= 3e38):
                raise ValueError(f"rotary must be (inv_freq, factor): float32 [{cfg.head_dim // 2}] on {dec.inv_freq.device}, a finite number")
        self.dec, self.page = dec, page
        shape = (cfg.layers, pages, page, cfg.heads, cfg.head_dim)
        self.k_pages, self.v_pages = (torch.zeros(shape, dtype=cache, device=dec.device) for _ in range(2))
        self.scales: list[dict] = [{}] * cfg.layers
        if cache != torch.bfloat16:
            block = next(b for b in (16, 12, 8, 4) if page % b == 0)
            shape = (2, cfg.layers, pages, page // block, cfg.heads)
            k_scales, v_scales = torch.zeros(shape, dtype=torch.uint8, device=dec.device).view(torch.float8_e8m0fnu)
            self.scales = [{"k_scales": k, "v_scales": v} for k, v in zip(k_scales, v_scales)]
            rotary = rotary or (dec.inv_freq, 1.0)
        self.rotary = rotary
        self.free = list(range(pages))

    def _ints(self, xs: list) -> torch.Tensor:
        return torch.tensor(xs, dtype=torch.int32, device=self.dec.device)

    def _prompts(self, prompts: list[torch.Tensor], top: int) -> list[list[int]]:
        if not 0 <= top <= min(MAX_TOP, self.dec.cfg.vocab):
            raise ValueError(f"top must be 0..{MAX_TOP} and at most the vocabulary, got {top}")
        ids = [p.reshape(-1).tolist() for p in prompts]
        if not ids or min(len(i) for i in ids) < 1:
            raise OptimizeError("need at least one prompt, each of at least one token")
        if any(min(i) < 0 or max(i) >= self.dec.cfg.vocab for i in ids):
            raise OptimizeError("token id outside the vocabulary")
        return ids

    def _norm(self, x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
        out = torch.empty_like(x)
        _lib.check(_lib.lib().bp_decode_norm_residual_rows(
            x.data_ptr(), weight.data_ptr(), _lib.ptr(residual), out.data_ptr(), x.shape[1], self.dec.cfg.eps, x.shape[0],
            _lib.stream_ptr(self.dec.device)), "bp_decode_norm_residual_rows")
        return out

    def _rope(self, x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
        """bf16(x cos + rotate_half(x) sin) in fp32, x [tokens, hidden] -> [tokens, heads, head_dim]."""
        x = x.view(-1, self.dec.cfg.heads, self.dec.cfg.head_dim).float()
        a, b = x.chunk(2, dim=-1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1).to(torch.bfloat16)

    def _forward(self, ids: torch.Tensor, positions: torch.Tensor, attend, keep: torch.Tensor | None = None) -> torch.Tensor:
        """Logits of the tokens `ids` at `positions` (of the rows `keep` only, when given); attend(layer, q, k, v) is the
        attention of a layer, [tokens, heads, head_dim] each."""
        dec, cfg = self.dec, self.dec.cfg
        st = _lib.stream_ptr(dec.device)
        if self.rotary is None:
            angle = positions[:, None].float() * dec.inv_freq[None, :]
            cos, sin = angle.cos()[:, None], angle.sin()[:, None]
        x = dec.embed[ids]
        for i, w in enumerate(dec.layers):
            q, k, v = S.skinny_mm(x, *w["qkv"]).split(cfg.hidden, dim=1)
            q, k = self._norm(q.contiguous(), w["q_norm"]), self._norm(k.contiguous(), w["k_norm"])
            if self.rotary is None:
                q, k = self._rope(q, cos, sin), self._rope(k, cos, sin)
            else:
                q, k = (t.view(-1, cfg.heads, cfg.head_dim) for t in (q, k))
                rotate(q, k, positions, self.rotary[0], factor=self.rotary[1], out=(q, k))
            a = attend(i, q, k, v.unflatten(1, (cfg.heads, cfg.head_dim)))
            x = self._norm(S.skinny_mm(a.view(-1, cfg.hidden), *w["o"]), w["post_attn"], x)
            gate_up = S.skinny_mm(x, *w["gate_up"])
            act = torch.empty(x.shape[0], cfg.ffn, dtype=torch.bfloat16, device=dec.device)
            _lib.check(_lib.lib().bp_decode_silu_mul_rows(gate_up.data_ptr(), act.data_ptr(), cfg.ffn, x.shape[0], 1, st),
                       "bp_decode_silu_mul_rows")
            x = self._norm(S.skinny_mm(act, *w["down"]), w["post_ff"], x)
        if keep is not None:
            x = x[keep]
        return S.skinny_mm(self._norm(x, dec.norm), *dec.lm_head)

    def _pack(self, ids: list[list[int]]) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """The prompts' tokens one after another, their positions, and the offsets."""
        cu = [0]
        for i in ids:
            cu.append(cu[-1] + len(i))
        dev = self.dec.device
        flat = torch.tensor([t for i in ids for t in i], dtype=torch.int64, device=dev)
        positions = torch.tensor([p for i in ids for p in range(len(i))], dtype=torch.int64, device=dev)
        return flat, positions, self._ints(cu)

    @torch.no_grad()
    def score(self, prompts: list[torch.Tensor], top: int = 0) -> list[TokenLogprobs]:
        """Of every prompt, the log probabilities of its tokens after the first, given those before ([L - 1] each)."""
        ids = self._prompts(prompts, top)
        flat, positions, cu = self._pack(ids)
        logits = self._forward(flat, positions, lambda i, q, k, v: packed_attention(q, k, v, cu))
        # row t of a prompt predicts its token t + 1; a prompt's last row (whose target is the next prompt's) is dropped
        out = token_logprobs(logits, torch.roll(flat, -1), top=top)
        parts, at = [], 0
        for i in ids:
            parts.append(TokenLogprobs(*(t[at:at + len(i) - 1] for t in out)))
            at += len(i)
        return parts

    @torch.no_grad()
    def generate(self, prompts: list[torch.Tensor], max_new_tokens: int, eos_token_id=None, top: int = 0) -> list[Generated]:
        """The greedy continuation of every prompt: one packed pass over the prompts, then one step for all sequences at a
        time until every one has ended."""
        ids = self._prompts(prompts, top)
        if max_new_tokens < 1:
            raise OptimizeError("need at least one new token")
        eos = {eos_token_id} if isinstance(eos_token_id, int) else set(eos_token_id or ())
        need = [-(-(len(i) + max_new_tokens - 1) // self.page) for i in ids]
        if sum(need) > len(self.free):
            raise OptimizeError(f"{sum(need)} pages asked for, {len(self.free)} free")
        taken = [[self.free.pop() for _ in range(n)] for n in need]
        try:
            return self._generate(ids, taken, max_new_tokens, eos, top)
        finally:
            self.free.extend(p for pages in taken for p in pages)

    def _generate(self, ids: list[list[int]], taken: list[list[int]], max_new: int, eos: set, top: int) -> list[Generated]:
        flat, positions, cu = self._pack(ids)
        table = self._ints([pages + [-1] * (max(map(len, taken)) - len(pages)) for pages in taken])
        lengths = self._ints([len(i) for i in ids])

        def prompt(i: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
            paged_append(k, v, self.k_pages[i], self.v_pages[i], table, lengths, cu, **self.scales[i])
            return packed_attention(q, k, v, cu)

        def step(i: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
            paged_append(k, v, self.k_pages[i], self.v_pages[i], table, lengths, ones, **self.scales[i])
            return paged_attention(q, self.k_pages[i], self.v_pages[i], table, lengths, ones, **self.scales[i])

        n = len(ids)
        ones = torch.arange(n + 1, dtype=torch.int32, device=self.dec.device)
        logits = self._forward(flat, positions, prompt, keep=cu[1:].long() - 1)
        steps, ended, count = [], [False] * n, [0] * n
        while True:
            best = token_logprobs(logits, top=max(1, top))
            steps.append(best)
            tokens = best.top_ids[:, 0]
            for b, t in enumerate(tokens.tolist()):
                if not ended[b]:
                    count[b] += 1
                    ended[b] = t in eos or count[b] == max_new
            if all(ended):
                break
            lengths += 1  # (a sequence that has ended goes on within its pages; nobody reads what it writes)
            logits = self._forward(tokens, lengths.long() - 1, step)
        top_ids = torch.stack([s.top_ids for s in steps], 1)
        top_lps = torch.stack([s.top_logprobs for s in steps], 1)
        entropy = torch.stack([s.entropy for s in steps], 1)
        return [Generated(top_ids[b, :c, 0], top_lps[b, :c, 0], entropy[b, :c], top_ids[b, :c, :top], top_lps[b, :c, :top])
                for b, c in enumerate(count)]
