"""Several sequences on one decoder: the log probabilities of prompts against the CPU oracle's decode steps, and the tokens of
a batch against the single-sequence loop and against the batch's own scores."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from byteprof_amd.optim import olmo as OG
from byteprof_amd.optim.olmo_batch import OlmoBatch
from oracle import olmo as OO

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
CFG = OG.OlmoConfig(hidden=256, ffn=512, layers=2, heads=4, vocab=500, max_len=128)
# the logits differ from the oracle's by at most two to three bf16 steps of the largest (oracle/olmo.py): 2e-2 of it
LOGITS_TOL = 2e-2


def prompts(lengths, seed=3):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, CFG.vocab, (n,), generator=g) for n in lengths]


def oracle_rows(W, ids):
    cfg = OO.Config(CFG.hidden, CFG.ffn, CFG.layers, CFG.heads, CFG.vocab, CFG.rope_theta, CFG.eps, CFG.max_len)
    kc, vc = OO.new_cache(cfg)
    Wn = {k: v.float().cpu().numpy() for k, v in W.items()}
    return np.stack([OO.decode_step(Wn, cfg, kc, vc, t, p) for p, t in enumerate(ids)])


def test_scores_against_the_oracle():
    W = OG.random_weights(CFG, DEV, seed=7)
    batch = OlmoBatch(OG.OlmoDecoder(CFG, W), pages=16)
    ps = prompts((9, 1, 14, 2))
    for p, got in zip(ps, batch.score(ps, top=3)):
        assert got.logprob.shape == (len(p) - 1,) and got.top_ids.shape == (len(p) - 1, 3)
        if len(p) == 1:
            continue
        rows = oracle_rows(W, p.tolist())[:-1].astype(np.float64)
        # an error of e in every logit moves a log probability by 2 e at most
        tol = 2 * LOGITS_TOL * np.abs(rows).max()
        lse = np.log(np.exp(rows - rows.max(-1, keepdims=True)).sum(-1)) + rows.max(-1)
        lp = rows - lse[:, None]
        want = lp[np.arange(len(rows)), p[1:].numpy()]
        assert np.abs(got.logprob.cpu().numpy() - want).max() <= tol
        ids = got.top_ids.cpu().numpy()
        assert np.abs(got.top_logprobs.cpu().numpy() - np.take_along_axis(lp, ids, 1)).max() <= tol
        assert (np.take_along_axis(lp, ids[:, :1], 1)[:, 0] >= lp.max(-1) - tol).all()


@pytest.mark.parametrize("kind", ["bf16", "int8", "int4"])
def test_generation_follows_its_own_scores_and_the_single_loop(kind):
    dec = OG.OlmoDecoder(CFG, OG.random_weights(CFG, DEV, seed=8), kind)
    batch = OlmoBatch(dec, pages=40, page=8)
    ps = prompts((5, 23, 1, 70), seed=4)
    outs = batch.generate(ps, max_new_tokens=20, top=2)
    assert len(batch.free) == 40
    single = OG.make_generate(dec)
    agree = total = 0
    for p, got in zip(ps, outs):
        assert got.tokens.shape == (20,) and torch.equal(got.tokens, got.top_ids[:, 0])
        whole = torch.cat([p, got.tokens.cpu()])
        again = batch.score([whole], top=2)[0]  # the same tokens through the packed path
        last = slice(len(p) - 1, None)
        # two paths round the attention's probabilities at other places: a few bf16 steps of the logits
        assert (again.logprob[last] - got.logprobs).abs().max() < 0.15
        assert (again.entropy[last] - got.entropy).abs().max() < 0.15
        margin = (got.top_logprobs[:, 0] - got.top_logprobs[:, 1]).cpu()
        want = single(p[None], max_new_tokens=20)[0, len(p):].cpu()
        for t in range(20):  # up to the first choice between two tokens that are nearly alike
            total += 1
            if want[t] != got.tokens[t]:
                assert margin[t] < 0.15, (kind, t, margin[t])
                break
            agree += 1
    assert agree >= total - 4 and total >= 40


def test_an_end_token_ends_its_sequence_alone():
    dec = OG.OlmoDecoder(CFG, OG.random_weights(CFG, DEV, seed=9))
    batch = OlmoBatch(dec, pages=20)
    ps = prompts((6, 11), seed=5)
    free = batch.generate(ps, max_new_tokens=12)
    eos = int(free[0].tokens[3])
    outs = batch.generate(ps, max_new_tokens=12, eos_token_id=eos)
    for a, b in zip(free, outs):
        hits = (a.tokens == eos).nonzero()
        n = int(hits[0]) + 1 if len(hits) else 12
        assert torch.equal(b.tokens, a.tokens[:n])
    assert len(outs[0].tokens) <= 4


def test_refusals():
    dec = OG.OlmoDecoder(CFG, OG.random_weights(CFG, DEV, seed=9))
    batch = OlmoBatch(dec, pages=2)
    with pytest.raises(OG.OptimizeError, match="pages"):
        batch.generate(prompts((30,)), max_new_tokens=10)
    assert len(batch.free) == 2
    with pytest.raises(OG.OptimizeError, match="vocabulary"):
        batch.score([torch.tensor([1, CFG.vocab])])
    with pytest.raises(OG.OptimizeError, match="at least one"):
        batch.generate([], max_new_tokens=1)
    with pytest.raises(OG.OptimizeError, match="new token"):
        batch.generate(prompts((3,)), max_new_tokens=0)
    with pytest.raises(ValueError, match="at least one page"):
        OlmoBatch(dec, pages=0)


def test_every_generated_token_against_the_oracle():
    """The oracle's decode steps over what the batch generated: every token is its best but for the logits' error, every log
    probability and entropy its own. Sequences of all lengths in one batch, through pages of 4."""
    W = OG.random_weights(CFG, DEV, seed=10)
    batch = OlmoBatch(OG.OlmoDecoder(CFG, W), pages=60, page=4)
    ps = prompts((5, 23, 1, 40, 8), seed=6)
    for p, got in zip(ps, batch.generate(ps, max_new_tokens=20, top=2)):
        whole = torch.cat([p, got.tokens.cpu()]).tolist()
        rows = oracle_rows(W, whole[:-1])[len(p) - 1:].astype(np.float64)
        tol = 2 * LOGITS_TOL * np.abs(rows).max()  # an error of e in every logit moves a log probability by 2 e at most
        lp = rows - (np.log(np.exp(rows - rows.max(-1, keepdims=True)).sum(-1, keepdims=True)) + rows.max(-1, keepdims=True))
        mine = lp[np.arange(20), got.tokens.cpu().numpy()]
        assert (mine >= lp.max(-1) - tol).all()
        assert np.abs(got.logprobs.cpu().numpy() - mine).max() <= tol
        assert np.abs(got.top_logprobs.cpu().numpy() - np.take_along_axis(lp, got.top_ids.cpu().numpy(), 1)).max() <= tol
        ent = -(np.exp(lp) * lp).sum(-1)
        # its derivative in a logit is -p (lp + H): errors of e move it by e sum p |lp + H| <= 2 e H at most, and as much again
        assert (np.abs(got.entropy.cpu().numpy() - ent) <= 2 * tol * (1 + ent)).all()


@pytest.mark.parametrize("kind", ["bf16", "int8", "int4"])
def test_the_single_loops_tokens_are_the_batchs_choice(kind):
    """Every token of the single-sequence loop, scored by the batch behind the same tokens: the batch's own choice there but for
    the two paths' errors in the logits."""
    dec = OG.OlmoDecoder(CFG, OG.random_weights(CFG, DEV, seed=8), kind)
    batch = OlmoBatch(dec, pages=1)
    ps = prompts((5, 23, 1, 70), seed=4)
    wholes = [OG.make_generate(dec)(p[None], max_new_tokens=20)[0].cpu() for p in ps]
    for p, got in zip(ps, batch.score(wholes, top=1)):
        new = slice(len(p) - 1, None)
        best = got.top_logprobs[new, 0]
        assert len(best) == 20
        # |logit| <= 8, four standard deviations (a normed row times a head row of std 2 / sqrt(hidden)): an error of e in each of
        # the two paths' logits lets a token be chosen that lies 4 e below the other's best
        assert (got.logprob[new] >= best - 4 * LOGITS_TOL * 8.0).all()
