"""What goes through OlmoBatch over a cache in 8 bits and with frequencies of its own, call by call: the queries and keys that reach the
attention against float64 at their positions, every append's codes against the definition and every step's attention against float64
over what the cache stands for. Each check is also made against a mistake of one step (a position, a scale), which it must see."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from byteprof_amd.optim import attention as A
from byteprof_amd.optim import olmo as OG
from byteprof_amd.optim import olmo_batch as OB
from byteprof_amd.optim.rotary import rotary_frequencies
from oracle import olmo as OO
from tests.test_attention_gpu import reference
from tests.test_cache8_gpu import append_reference, raw
from tests.test_olmo_batch_gpu import CFG, DEV, LOGITS_TOL, oracle_rows, prompts

pytestmark = pytest.mark.gpu
PARTS = dict(scaling="parts", factor=64.0, trained=64, fast=8.0)  # 0.1 ln 64 + 1 = 1.416 on cosine and sine


def turned(x, positions, inv_freq, factor):
    """x [tokens, heads, D] in float64 at its positions, and of every element the sum of its pair's magnitudes."""
    x1, x2 = x.double().cpu().chunk(2, -1)
    a = (positions.double().cpu()[:, None] * inv_freq.double().cpu())[:, None]
    c, s = a.cos() * factor, a.sin() * factor
    return torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], -1), (x1.abs() + x2.abs()).repeat(1, 1, 2) * factor


@pytest.mark.parametrize("way", ["its own", "the kernel", "parts"])
def test_queries_and_keys_that_reach_the_attention(monkeypatch, way):
    """Within half a bf16 step of the definition, and of the pair's magnitudes what the angles are off: in float32, at positions below 128
    and frequencies up to 1, half a step below 128, 2^-18, and some float32 steps for cosine, sine and products: 2^-16 holds them; reduced
    in 64 bits those steps alone, 2^-20."""
    dec = OG.OlmoDecoder(CFG, OG.random_weights(CFG, DEV, seed=21))
    inv, factor = (dec.inv_freq, 1.0) if way != "parts" else rotary_frequencies(CFG.head_dim, CFG.rope_theta, device=DEV, **PARTS)
    batch = OB.OlmoBatch(dec, pages=1, rotary=None if way == "its own" else (inv, factor))
    before, after = [], []
    if way == "its own":
        rope = batch._rope
        monkeypatch.setattr(batch, "_rope", lambda x, cos, sin: (before.append(x.view(-1, CFG.heads, CFG.head_dim).clone()), rope(x, cos, sin))[1])
    else:
        rotate = OB.rotate
        monkeypatch.setattr(OB, "rotate", lambda q, k, *a, **kw: (before.extend((q.clone(), k.clone())), rotate(q, k, *a, **kw))[1])
    flat, positions, cu = batch._pack([p.tolist() for p in prompts((100, 3, 60), seed=22)])
    with torch.no_grad():
        batch._forward(flat, positions, lambda i, q, k, v: (after.extend((q.clone(), k.clone())), A.packed_attention(q, k, v, cu))[1])
    assert len(before) == len(after) == 2 * CFG.layers
    for x, y in zip(before, after):
        want, pair = turned(x, positions, inv, factor)
        bound = want.abs() * 2.0 ** -8 + pair * (2.0 ** -16 if way == "its own" else 2.0 ** -20)
        assert ((y.double().cpu() - want).abs() <= bound).all()
        # the first pair turns by a radian a position: a position on, its columns are 2 sin(1/2) = 0.96 of its radius away, and with a factor
        # 2^-5 greater 2^-5 of their size, where the bound is 2^-8 of it; near a zero of either they may coincide
        first = [0, CFG.head_dim // 2]
        for other in (turned(x, positions + 1, inv, factor)[0], turned(x, positions, inv, factor * (1 + 2.0 ** -5))[0]):
            seen = ((y.double().cpu() - other).abs() > bound)[..., first].double().mean().item()
            assert seen > 0.9, seen


@pytest.mark.parametrize("cache,page", [(torch.float8_e4m3fn, 16), (torch.int8, 16), (torch.int8, 12)])
def test_every_append_and_every_step_of_a_generation(monkeypatch, cache, page):
    """The calls themselves, on the batch's own tensors: codes and scales equal to the definition's, the attention element by element
    within the 16-bit kernels' bound of float64 over paged_read's values. Positions and lengths are those of the tokens."""
    dec = OG.OlmoDecoder(CFG, OG.random_weights(CFG, DEV, seed=23))
    batch = OB.OlmoBatch(dec, pages=30, page=page, cache=cache)
    lens, new = [5, 23, 1, 40], 19
    append, attend, calls = A.paged_append, A.paged_attention, {"append": 0, "attend": 0}

    def check_append(k, v, kp, vp, table, lengths, cu, *, k_scales, v_scales):
        step = calls["append"] // CFG.layers  # 0: the prompts
        assert lengths.tolist() == [n + step for n in lens]
        off = cu.tolist()
        assert off == (np.cumsum([0] + lens).tolist() if step == 0 else list(range(len(lens) + 1)))
        want = [append_reference(x, p, s, table, lengths.tolist(), off, cache, len(x)) for x, p, s in ((k, kp, k_scales), (v, vp, v_scales))]
        append(k, v, kp, vp, table, lengths, cu, k_scales=k_scales, v_scales=v_scales)
        for (pages, scales), p, s in zip(want, (kp, vp), (k_scales, v_scales)):
            assert torch.equal(raw(p), pages) and torch.equal(raw(s), scales), step
        calls["append"] += 1

    def check_attend(q, kp, vp, table, lengths, cu, *, k_scales, v_scales):
        got = attend(q, kp, vp, table, lengths, cu, k_scales=k_scales, v_scales=v_scales)
        n = lengths.tolist()
        every = torch.tensor(np.cumsum([0] + n), dtype=torch.int32, device=DEV)
        k, v = A.paged_read(kp, vp, table, lengths, every, sum(n), k_scales=k_scales, v_scales=v_scales)
        missed = 0
        for b, (lo, hi) in enumerate(zip(every.tolist(), every.tolist()[1:])):
            want, bound = reference(q[b:b + 1], k[lo:hi], v[lo:hi], n[b] - 1, CFG.head_dim ** -0.5)
            out = got[b:b + 1].double().cpu()
            assert ((out - want).abs() <= bound).all(), (calls, b)
            if hi - lo > 2:  # without the last position, with the values one position on, with the last block's scale doubled
                wrong = k[lo:hi], v[lo:hi].clone()
                wrong[1][-((n[b] - 1) % page + 1):] *= 2
                for kk, vv in ((k[lo:hi - 1], v[lo:hi - 1]), (k[lo:hi], v[lo:hi].roll(1, 0)), wrong):
                    other, _ = reference(q[b:b + 1], kk, vv, len(kk) - 1, CFG.head_dim ** -0.5)
                    missed += not ((out - other).abs() > bound).any()
        assert missed == 0
        calls["attend"] += 1
        return got

    monkeypatch.setattr(OB, "paged_append", check_append)
    monkeypatch.setattr(OB, "paged_attention", check_attend)
    outs = batch.generate(prompts(lens, seed=24), max_new_tokens=new)
    assert calls == {"append": new * CFG.layers, "attend": (new - 1) * CFG.layers} and len(batch.free) == 30
    assert all(len(o.tokens) == new for o in outs)


def test_frequencies_by_parts_against_the_oracle(monkeypatch):
    """Scores with frequencies whose cosines and sines have a factor: against the CPU oracle with the same, within the tolerance of the
    scores without (two to three bf16 steps of the largest logit, twice in a log probability); without the factor, or with the decoder's
    own frequencies, the oracle is many times that away."""
    W = OG.random_weights(CFG, DEV, seed=25)
    inv, factor = rotary_frequencies(CFG.head_dim, CFG.rope_theta, device=DEV, **PARTS)
    ps = prompts((30, 14), seed=26)
    scores = OB.OlmoBatch(OG.OlmoDecoder(CFG, W), pages=1, rotary=(inv, factor)).score(ps)

    def logprobs(ids, freq, by):
        def rope(x, pos, cfg):
            a = freq.double().cpu().numpy() * pos
            x1, x2 = np.split(x.astype(np.float64), 2, -1)
            return OO.bf16_round((np.concatenate([x1 * np.cos(a) - x2 * np.sin(a), x2 * np.cos(a) + x1 * np.sin(a)], -1) * by).astype(np.float32))

        monkeypatch.setattr(OO, "rope", rope)
        rows = oracle_rows(W, ids)[:-1].astype(np.float64)
        return rows[np.arange(len(rows)), ids[1:]] - np.log(np.exp(rows - rows.max(-1, keepdims=True)).sum(-1)) - rows.max(-1), np.abs(rows).max()

    own = rotary_frequencies(CFG.head_dim, CFG.rope_theta)[0]
    for p, got in zip(ps, scores):
        ids, got = p.tolist(), got.logprob.cpu().numpy()
        want, largest = logprobs(ids, inv, factor)
        assert np.abs(got - want).max() <= 2 * LOGITS_TOL * largest
        for freq, by in ((inv, 1.0), (own, factor)):
            assert np.abs(got - logprobs(ids, freq, by)[0]).max() > 4 * LOGITS_TOL * largest
