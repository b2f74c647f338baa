"""token_logprobs against log softmax in float64. Ids are equal; probabilities and entropy are float32 sums: a lane adds
vocab / 256 terms at most and the joins a few dozen, each term with a few steps of its own (the difference's rounding, exp2),
so ln z is off by at most (vocab / 256 + 64) 2^-23, and the results by that times their size plus one."""

from __future__ import annotations

import math

import pytest
import torch

from byteprof_amd.optim.logprobs import MAX_TOP, token_logprobs

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def reference(x, targets, top):
    x = x.double().cpu() + 0.0
    x = x - x.amax(-1, keepdim=True)  # next to the lowest value even float64 would lose the logarithm
    lse = torch.logsumexp(x, -1, keepdim=True)
    lp = x - lse
    p = torch.exp(lp)
    ent = -(p * torch.where(p > 0, lp, 0.0)).sum(-1)
    vals, ids = torch.sort(x, dim=-1, descending=True, stable=True)
    return torch.gather(lp, 1, targets.cpu()[:, None])[:, 0], ent, ids[:, :top], vals[:, :top] - lse


def check(x, targets, top):
    out = token_logprobs(x, targets, top=top)
    lp, ent, ids, tlp = reference(x, targets, top)
    assert torch.equal(out.top_ids.cpu(), ids)
    tol = (x.shape[1] / 256 + 64) * 2.0 ** -23
    for got, want in ((out.logprob, lp), (out.entropy, ent), (out.top_logprobs, tlp)):
        got = got.double().cpu()
        same = got == want  # -inf
        assert (same | ((got - want).abs() <= tol * (1 + want.abs()))).all()
    return out


CASES = [(1, 1, 1, "bf16"), (1, 100352, 5, "bf16"), (3, 7, 7, "fp16"), (5, 1000, 0, "fp32"), (2, 2049, 32, "fp32"),
         (70, 5003, 20, "bf16"), (1500, 777, 3, "fp16"), (1, 160001, 32, "fp32"), (33, 50257, 1, "bf16"),
         (1100, 4096, 32, "bf16"), (64, 255, 32, "fp16")]


@pytest.mark.parametrize("rows,vocab,top,dtype", CASES)
@pytest.mark.parametrize("layout", ["plain", "padded", "unaligned"])
def test_rows(rows, vocab, top, dtype, layout):
    print(f"\n[logprobs] {rows} x {vocab} top {top} {dtype} {layout}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(rows + vocab)
    full = torch.randn(rows, vocab + 13, generator=g, device=DEV) * 3.0
    full[:, ::97] += 9.0
    full = full.to(DTYPES[dtype])
    x = full[:, :vocab].contiguous() if layout == "plain" else full[:, :vocab] if layout == "padded" else full[:, 5:5 + vocab]
    targets = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
    check(x, targets, top)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows", [2, 1200])
def test_ties_and_orders(dtype, rows):
    """Equal rows, rising and falling ones (every logit passes the threshold), few distinct values, zeros of both signs."""
    print(f"\n[ties] {dtype} {rows}", flush=True)
    vocab, dt = 6000, DTYPES[dtype]
    i = torch.arange(vocab, device=DEV, dtype=torch.float32)
    g = torch.Generator(device=DEV).manual_seed(1)
    kinds = [torch.zeros_like(i), i / 64, -i / 64, (i % 7) - 3.0, torch.where(i % 2 == 0, 0.0, -0.0),
             torch.randint(0, 3, (vocab,), generator=g, device=DEV).float(), (i / 512).floor()]
    for x in kinds:
        x = x.to(dt).expand(rows, vocab).contiguous()
        check(x, torch.randint(0, vocab, (rows,), generator=g, device=DEV), 32)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_masked_tokens(dtype):
    """-inf and the type's lowest value: rows with one, 31 and no token left; more alternatives asked than tokens left."""
    print(f"\n[masked] {dtype}", flush=True)
    dt, vocab = DTYPES[dtype], 3001
    g = torch.Generator(device=DEV).manual_seed(2)
    base = torch.randn(4, vocab, generator=g, device=DEV).to(dt)
    for low in (-math.inf, torch.finfo(dt).min):
        x = base.clone()
        x[0, torch.arange(vocab, device=DEV) != 2000] = low
        x[1, 31:] = low
        x[2, ::2] = low
        targets = torch.tensor([2000, 30, 1, 5], device=DEV)
        check(x, targets, 32)
        check(x, torch.tensor([0, 2999, 0, 7], device=DEV), 0)  # masked targets: -inf, or far below
    x = torch.full((2, vocab), torch.finfo(dt).min, dtype=dt, device=DEV)
    check(x, torch.tensor([3, 4], device=DEV), 32)  # nothing but the lowest value: all alike
    x[1] = -math.inf
    out = token_logprobs(x, torch.tensor([3, 4], device=DEV), top=4)
    assert out.logprob[1].isnan() and out.entropy[1].isnan() and out.top_logprobs[1].isnan().all()
    assert out.top_ids[1].tolist() == [0, 1, 2, 3] and out.logprob[0].isfinite()


@pytest.mark.parametrize("rows", [1, 1100])
def test_nan_and_inf(rows):
    """A NaN or +inf: NaN probabilities for its row alone; NaN first in the order, then +inf."""
    print(f"\n[nan] {rows}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(rows + 1, 4000, generator=g, device=DEV)
    x[0, 3000], x[0, 17], x[0, 2500] = math.nan, math.inf, -math.nan
    targets = torch.zeros(rows + 1, dtype=torch.int64, device=DEV)
    out = token_logprobs(x[:rows], targets[:rows], top=5)
    assert out.logprob[0].isnan() and out.entropy[0].isnan() and out.top_logprobs[0].isnan().all()
    rest = torch.sort(torch.where(x[0].isnan() | x[0].isinf(), -math.inf, x[0]), descending=True).indices[:2].tolist()
    assert out.top_ids[0].tolist() == [2500, 3000, 17] + rest
    if rows > 1:
        check(x[1:rows], targets[1:rows], 5)
    y = x[rows:].clone()
    y[0, 17] = math.inf
    out = token_logprobs(y, targets[:1], top=2)
    assert out.top_ids[0, 0] == 17 and out.logprob.isnan().all()


def test_targets_outside_and_none():
    x = torch.randn(3, 50, device=DEV)
    out = token_logprobs(x, torch.tensor([-1, 50, 49], device=DEV), top=1)
    assert out.logprob[:2].isnan().all() and out.logprob[2].isfinite() and out.entropy.isfinite().all()
    out = token_logprobs(x, top=50 if MAX_TOP >= 50 else MAX_TOP)
    assert out.logprob is None
    assert torch.equal(out.top_ids, torch.sort(x, descending=True, stable=True).indices[:, :MAX_TOP])
    assert token_logprobs(x[:0], top=3).top_ids.shape == (0, 3)


def test_rows_past_32_bit_offsets():
    x = torch.empty(3, 2 ** 31, dtype=torch.bfloat16, device=DEV)[:, :5000]  # the last row begins past 2^32 elements
    x.copy_(torch.randn(3, 5000, device=DEV))
    check(x, torch.tensor([1, 2, 3], device=DEV), 8)


def test_graph_and_stream():
    g = torch.Generator(device=DEV).manual_seed(4)
    x = torch.randn(4, 9000, generator=g, device=DEV).to(torch.bfloat16)
    t = torch.tensor([1, 2, 3, 4], device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        token_logprobs(x, t, top=6)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = token_logprobs(x, t, top=6)
    for _ in range(3):
        x.copy_(torch.randn(4, 9000, generator=g, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in out]
        want = token_logprobs(x, t, top=6)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_gpu_refusals():
    x = torch.zeros(2, 10, device=DEV)
    with pytest.raises(ValueError, match="all tensors must be on"):
        token_logprobs(x, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="no backward"):
        token_logprobs(x.clone().requires_grad_())


def far_rows(dt, vocab, g):
    """Rows whose greatest logit is far from zero, alone, alike, in ties and next to the nearest number; rows whose masked tokens
    have such a value and leave few others, all in one place."""
    rows = []
    ordinary = torch.randn(vocab, generator=g, device=DEV)
    for far in (1e10, -1e10, 1e30, -1e30, 3e38, -3e38, torch.finfo(dt).max, -1.5e9, 1.2e7, -1.2e7, 1.1e7):
        top = torch.tensor(far, dtype=dt, device=DEV)
        below = torch.nextafter(top, torch.tensor(-math.inf, dtype=dt, device=DEV))
        x = ordinary.to(dt) if far > 0 else torch.full((vocab,), torch.finfo(dt).min, dtype=dt, device=DEV)
        x[vocab // 3] = top
        rows.append(x)
        rows.append(top.expand(vocab).clone())
        y = below.expand(vocab).clone()
        y[torch.tensor([1, vocab // 2, vocab - 1], device=DEV)] = top
        rows.append(y)
    for mask in (-1e9, -1e10, -1e20, -1e30, torch.finfo(dt).min, -math.inf):
        for first in (0, vocab // 2, vocab - 20):
            x = torch.full((vocab,), mask, dtype=dt, device=DEV)
            x[first:first + 20] = ordinary[:20].to(dt)
            rows.append(x)
    rows.append(ordinary.to(dt))
    return torch.stack(rows)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("vocab", [3001, 30011])
@pytest.mark.parametrize("top", [0, 8])
def test_logits_far_from_zero(dtype, vocab, top):
    """Against float64, rounded to float32 (what does not fit becomes -inf there, too). A lane of the pass that takes differences
    first adds vocab / 64 terms."""
    print(f"\n[far] {dtype} {vocab} {top}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(5)
    x = far_rows(DTYPES[dtype], vocab, g)
    targets = x.float().argmax(-1)
    targets[1::2] = torch.randint(0, vocab, (len(targets[1::2]),), generator=g, device=DEV)
    lp, ent, _, _ = reference(x, targets, 0)
    # the order is the logits' own: 1e30 less, float64 would have them all alike
    ids = torch.sort(x.double().cpu() + 0.0, dim=-1, descending=True, stable=True).indices[:, :top]
    tlp = torch.stack([reference(x, ids[:, k], 0)[0] for k in range(top)], 1) if top else torch.empty(len(x), 0).double()
    tol = (vocab / 64 + 64) * 2.0 ** -23

    def alike(got, want):
        got, want = got.double().cpu(), want.float().double()
        return ((got == want) | ((got - want).abs() <= tol * (1 + want.abs()))).all()

    many = x.repeat(20, 1)  # one workgroup a row
    for r in range(len(x) + 2):
        whole = r >= len(x)
        out = token_logprobs(many if r > len(x) else x if whole else x[r:r + 1], targets.repeat(20) if r > len(x) else targets if
                             whole else targets[r:r + 1], top=top)
        of = slice(None) if whole else slice(r, r + 1)
        out = [t[-len(x):] for t in out] if whole else out
        assert torch.equal(out[2].cpu(), ids[of]), r
        assert alike(out[0], lp[of]) and alike(out[1], ent[of]) and alike(out[3], tlp[of]), r
