"""OlmoBatch over a cache held in 8 bits and with frequencies of its own: against steps whose attention is taken in float64 over what
the cache stands for, against the CPU oracle with the same frequencies, and against the batch without either."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from byteprof_amd.optim import attention as A
from byteprof_amd.optim import olmo as OG
from byteprof_amd.optim.olmo_batch import OlmoBatch
from byteprof_amd.optim.rotary import rotary_frequencies
from oracle import olmo as OO
from tests.test_attention_gpu import reference
from tests.test_olmo_batch_gpu import CFG, DEV, LOGITS_TOL, oracle_rows, prompts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache,page", [(torch.float8_e4m3fn, 16), (torch.int8, 16), (torch.int8, 4), (torch.float8_e4m3fn, 24)])
def test_generated_tokens_against_attention_over_what_the_cache_stands_for(cache, page):
    """Every step again on a batch of its own, its attention in float64 over paged_read's values, fed with the first batch's tokens:
    every token is the best there but for the errors of the two paths' logits, and so are the log probabilities."""
    dec = OG.OlmoDecoder(CFG, OG.random_weights(CFG, DEV, seed=11))
    first = OlmoBatch(dec, pages=60, page=page, cache=cache)
    ps, new = prompts((5, 23, 1, 40), seed=7), 18
    outs = first.generate(ps, max_new_tokens=new, top=2)
    assert len(first.free) == 60

    batch = OlmoBatch(dec, pages=60, page=page, cache=cache)
    ids = [p.tolist() for p in ps]
    need = [-(-(len(i) + new) // page) for i in ids]
    table = torch.full((len(ps), max(need)), -1, dtype=torch.int32, device=DEV)
    for b, n in enumerate(need):
        table[b, :n] = torch.arange(sum(need[:b]), sum(need[:b]) + n, device=DEV)
    for t in range(new):
        lens = [len(i) + t for i in ids]
        lengths = torch.tensor(lens, dtype=torch.int32, device=DEV)
        every = torch.tensor(np.cumsum([0] + lens), dtype=torch.int32, device=DEV)

        def attend(i, q, k, v):
            A.paged_append(k, v, batch.k_pages[i], batch.v_pages[i], table, lengths, cu, **batch.scales[i])
            if t == 0:
                return A.packed_attention(q, k, v, cu)
            kr, vr = A.paged_read(batch.k_pages[i], batch.v_pages[i], table, lengths, every, sum(lens), **batch.scales[i])
            rows = [reference(q[b:b + 1], kr[every[b]:every[b + 1]], vr[every[b]:every[b + 1]], lens[b] - 1, CFG.head_dim ** -0.5)[0]
                    for b in range(len(lens))]
            return torch.cat(rows).to(torch.bfloat16).to(DEV)

        with torch.no_grad():
            if t == 0:
                flat, positions, cu = batch._pack(ids)
                logits = batch._forward(flat, positions, attend, keep=cu[1:].long() - 1)
            else:
                cu = torch.arange(len(ps) + 1, dtype=torch.int32, device=DEV)
                logits = batch._forward(torch.stack([o.tokens[t - 1] for o in outs]), lengths.long() - 1, attend)
        lp = torch.log_softmax(logits.double(), -1).cpu()
        tol = 4 * LOGITS_TOL * logits.abs().max().item()  # both paths' logits are off by LOGITS_TOL of the largest at most
        for b, got in enumerate(outs):
            mine = lp[b, got.tokens[t].cpu()]
            assert mine >= lp[b].max() - tol
            assert abs(got.logprobs[t].item() - mine.item()) <= tol


def test_frequencies_of_its_own_against_the_oracle(monkeypatch):
    W = OG.random_weights(CFG, DEV, seed=12)
    dec = OG.OlmoDecoder(CFG, W)
    inv, factor = rotary_frequencies(CFG.head_dim, CFG.rope_theta, scaling="linear", factor=4.0, device=DEV)
    assert factor == 1.0
    batch = OlmoBatch(dec, pages=16, rotary=(inv, factor))
    plain = OO.inv_freq
    monkeypatch.setattr(OO, "inv_freq", lambda cfg: (plain(cfg) / 4).astype(np.float32))
    ps = prompts((30, 14), seed=8)
    for p, got in zip(ps, batch.score(ps)):
        rows = oracle_rows(W, p.tolist())[:-1].astype(np.float64)
        lse = np.log(np.exp(rows - rows.max(-1, keepdims=True)).sum(-1)) + rows.max(-1)
        want = rows[np.arange(len(rows)), p[1:].numpy()] - lse
        assert np.abs(got.logprob.cpu().numpy() - want).max() <= 2 * LOGITS_TOL * np.abs(rows).max()


def test_the_decoders_own_frequencies_by_either_way():
    """rotary given the decoder's frequencies: scores and tokens but for angles that are not rounded to float32 (at positions below
    128 by less than 2^-17, far below a bf16 step of q and k): the logits' errors of two paths."""
    dec = OG.OlmoDecoder(CFG, OG.random_weights(CFG, DEV, seed=13))
    ps = prompts((60, 3, 100), seed=9)
    for a, b in zip(OlmoBatch(dec, pages=30).score(ps), OlmoBatch(dec, pages=30, rotary=(dec.inv_freq, 1.0)).score(ps)):
        # |logit| <= 8, four standard deviations of a normed row times a head row of std 2 / sqrt(hidden)
        assert (a.logprob - b.logprob).abs().max() <= 4 * LOGITS_TOL * 8.0


def test_refusals():
    dec = OG.OlmoDecoder(CFG, OG.random_weights(CFG, DEV, seed=9))
    with pytest.raises(ValueError, match="held in"):
        OlmoBatch(dec, pages=2, cache=torch.float16)
    with pytest.raises(ValueError, match="multiple of 4"):
        OlmoBatch(dec, pages=2, page=6, cache=torch.int8)
    batch = OlmoBatch(dec, pages=2, cache=torch.int8)
    assert batch.k_pages.element_size() == 1 and batch.scales[0]["k_scales"].shape == (2, 1, CFG.heads)
    with pytest.raises(OG.OptimizeError, match="pages"):
        batch.generate(prompts((30,)), max_new_tokens=10)
