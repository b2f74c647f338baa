"""Every code at every scale as the value it stands for: what paged_read gives, attention over one position (whose value is the result),
and keys that decide between positions: attention over codes is attention over paged_read's values, whichever kernel takes the launch.

code x scale is exact in float64, and its rounding to the outputs' type (past fp16's range its greatest value) is the definition: values
are equal to it, no tolerance. The scores of the keys are exact in float32, so what is left there is one_hot_reference's bound and the
2^-25 by which an fp16 result below its normal values may be rounded."""

from __future__ import annotations

import math

import pytest
import torch

from byteprof_amd.optim import attention as A
from tests.test_attention_gpu import check as check16
from tests.test_attention_gpu import ints, one_hot_reference, reference
from tests.test_cache8_gpu import BF, DEV, E4M3, E8M0, F32, FP, I8, values_of

pytestmark = pytest.mark.gpu


def every_code(kind):
    """A page of 4 positions of 4 heads of 64 columns that holds every code (NaN codes apart), as uint8."""
    codes = torch.arange(256, dtype=torch.uint8, device=DEV).view(1, 1, 4, 64)
    if kind is E4M3:
        codes = torch.where(codes % 128 == 127, torch.zeros_like(codes), codes)
    return codes.expand(1, 4, 4, 64).contiguous()


def rounded(x, dtype):
    return (x.clamp(-65504.0, 65504.0) if dtype == FP else x).to(dtype)


@pytest.mark.parametrize("kind", [E4M3, I8])
@pytest.mark.parametrize("dtype", [FP, BF, F32])
def test_read_of_every_code_at_every_scale(kind, dtype):
    """bf16's and fp32's own limits: a value past their range is infinite."""
    codes = every_code(kind)
    pages = codes.expand(255, 4, 4, 64).contiguous().view(kind)
    scales = torch.arange(255, dtype=torch.uint8, device=DEV)[:, None, None].expand(255, 1, 4).contiguous().view(E8M0)
    table = torch.arange(255, dtype=torch.int32, device=DEV)[:, None]
    print(f"\n[read every scale] {kind} {dtype}", flush=True)
    k, v = A.paged_read(pages, pages, table, ints([1] * 255), ints(range(256)), 255, k_scales=scales, v_scales=scales, dtype=dtype)
    want = rounded(values_of(codes[:, 0].cpu(), kind) * 2.0 ** (torch.arange(255).double() - 127)[:, None, None], dtype)
    for got in (k, v):
        wrong = (got.cpu() != want).flatten(1).any(1).nonzero().flatten()
        assert not len(wrong), f"scales 2^{(wrong - 127).tolist()}"


@pytest.mark.parametrize("kind", [E4M3, I8])
@pytest.mark.parametrize("rows", [1, 2, 3, 80])
def test_attention_of_every_code_in_fp16(kind, rows):
    """One position and tiles of 16, 32 and 48 rows and the large ones: its value is every row's result."""
    codes = every_code(kind)
    pages = codes.view(kind)
    zero = torch.zeros_like(codes).view(kind)
    hq = {1: 4, 2: 80, 3: 160, 80: 400}[rows]  # 1, 20, 40 and 100 query heads to a key head
    for byte in [0, 60, *range(86, 160), 200, 254]:
        scales = torch.full((1, 1, 4), byte, dtype=torch.uint8, device=DEV).view(E8M0)
        q = torch.ones(1, hq, 64, dtype=FP, device=DEV)
        if byte in (0, 60, 254):
            print(f"\n[attention every code] {kind} {hq} heads, scale 2^{byte - 127}", flush=True)
        got = A.paged_attention(q, zero, pages, ints([[0]]), ints([1]), ints([0, 1]), k_scales=scales, v_scales=scales)
        want = rounded(values_of(codes[0, 0].cpu(), kind) * 2.0 ** (byte - 127), FP).repeat_interleave(hq // 4, 0)
        assert torch.equal(got[0].cpu(), want), byte


@pytest.mark.parametrize("kind", [E4M3, I8])
@pytest.mark.parametrize("e,a,scale", [(12, 1.0, 2.0 ** -12), (23, 1.0, 2.0 ** -12), (-30, 2.0 ** 15, 2.0 ** 12), (-20, 2.0 ** 15, 2.0 ** 4)])
def test_keys_at_the_ends_of_fp16(kind, e, a, scale):
    """Keys of one column that is not 0, past fp16's range or below its normal values: the scores are those of paged_read's keys, in
    launches of one row, of few and of many, but that int8 keys past fp16's range are 2^16 where rows are few (their scale is outside
    the product there). Keys that were not rounded would be far off: at 2^12 the codes 100 and 127 are one value, but apart by 27 in the
    exponent; at 2^-30 by 27 x 2^-30 x 2^15 x 2^12 = 3.4."""
    print(f"\n[keys in fp16] {kind} 2^{e}", flush=True)
    d, n = 64, 32
    big, small = (100.0, 127.0) if kind is I8 else (104.0, 120.0)
    x = torch.zeros(n, 1, d, device=DEV)
    x[:, 0, 5] = torch.tensor([big, small, 1.0, -small], device=DEV).repeat(n // 4)
    pages = x.to(E4M3 if kind is E4M3 else I8).view(2, 16, 1, d)
    v = torch.zeros(n, 1, d, device=DEV)
    v[:, 0] = torch.randint(-8, 9, (n, d), generator=torch.Generator(device=DEV).manual_seed(20), device=DEV).float()
    vpages = v.to(E4M3 if kind is E4M3 else I8).view(2, 16, 1, d)
    ks = torch.full((2, 1, 1), 127 + e, dtype=torch.uint8, device=DEV).view(E8M0)
    vs = torch.full((2, 1, 1), 127, dtype=torch.uint8, device=DEV).view(E8M0)
    where = (ints([[0, 1]]), ints([n]))
    k, _ = A.paged_read(pages, vpages, *where, ints([0, n]), n, k_scales=ks, v_scales=vs, dtype=FP)
    exact = values_of(pages.view(torch.uint8).cpu().view(n, d), kind) * 2.0 ** e
    assert torch.equal(k[:, 0].cpu(), rounded(exact, FP))
    assert (k[:, 0, 5].cpu().double() != exact[:, 5]).any() or e == -20
    for hq in (1, 20, 40, 100):  # tiles of 16, 32 and 48 rows, large ones
        q = torch.zeros(1, hq, d, dtype=FP, device=DEV)
        q[..., 5] = a
        got = A.paged_attention(q, pages, vpages, *where, ints([0, 1]), k_scales=ks, v_scales=vs, scale=scale)
        keys = k.double()
        if kind is I8 and hq < 100:
            keys = torch.where(exact.abs().to(DEV)[:, None] > 65504.0, keys.sign() * 65536.0, keys)
        want, bound = one_hot_reference(q[:, :1], keys, v, n - 1, scale, FP)
        for h in range(hq):
            check16(got[:, h], want, bound + 2.0 ** -25, f"{hq} heads, head {h}")


SHAPES = [
    # lens, chunks, page, block, hq, hk, d: tiles of 16, 32 and 48 rows and large ones, heads in whole tiles and not, divided keys
    ([300, 77], [1, 1], 16, 16, 4, 2, 64),
    ([300, 77], [1, 1], 16, 4, 4, 2, 128),
    ([700, 90], [5, 5], 32, 32, 8, 2, 128),
    ([700, 90], [9, 9], 16, 8, 8, 2, 128),
    ([300, 77], [9, 9], 16, 16, 8, 2, 64),
    ([300, 77], [1, 1], 12, 4, 4, 2, 64),
    ([300, 77], [9, 9], 20, 20, 8, 2, 72),
    ([400, 90], [1, 2], 16, 16, 4, 2, 256),
    ([400, 33], [3, 3], 16, 16, 14, 2, 200),
    ([300, 200], [130, 90], 16, 16, 2, 1, 64),
    ([300, 200], [130, 90], 64, 32, 2, 1, 128),
    ([300, 200], [130, 90], 12, 12, 2, 1, 80),
    ([300, 200], [130, 90], 8, 4, 2, 1, 40),
    ([300, 200], [130, 90], 16, 16, 2, 1, 256),
    ([5000, 17], [1, 1], 16, 16, 4, 1, 128),
    ([3000, 2600], [200, 7], 16, 8, 2, 2, 64),
]
ENDS = [(I8, "v", 90, 106), (I8, "v", 131, 146), (I8, "k", 94, 105), (E4M3, "v", 147, 154), (E4M3, "k", 147, 154)]


@pytest.mark.parametrize("kind,which,low,high", ENDS)
@pytest.mark.parametrize("lens,chunks,page,block,hq,hk,d", SHAPES)
def test_attention_at_the_ends_of_fp16(lens, chunks, page, block, hq, hk, d, kind, which, low, high):
    """Blocks whose scales lie on both sides of where fp16 needs more than a factor, in keys or in values: attention in float64 over what
    paged_read gives. (e4m3: codes below its normal values, half of the values past fp16's range.)"""
    print(f"\n[ends of fp16] {lens} {chunks} page {page} block {block} {hq}/{hk} x {d} {kind} {which}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(21)
    need = [-(-n // page) for n in lens]
    pool = sum(need)
    table = torch.zeros(len(lens), max(need), dtype=torch.int32, device=DEV)
    order = torch.randperm(pool, generator=g, device=DEV).to(torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = order[sum(need[:b]):sum(need[:b]) + n]
    cache = {}
    for name in "kv":
        shape = (pool, page, hk, d)
        if kind is I8:
            codes = torch.randint(-127, 128, shape, generator=g, device=DEV).to(torch.int8).view(torch.uint8)
        else:
            codes = (torch.randint(0, 16, shape, generator=g, device=DEV) + 128 * torch.randint(0, 2, shape, generator=g, device=DEV)).to(torch.uint8)
        ends = (low, high) if name == which else (119, 123)
        scales = torch.randint(*ends, (pool, page // block, hk), generator=g, device=DEV).to(torch.uint8)
        cache[name + "_pages"], cache[name + "_scales"] = codes.view(kind), scales.view(E8M0)
    off = [0]
    for c in chunks:
        off.append(off[-1] + c)
    every = [0]
    for n in lens:
        every.append(every[-1] + n)
    k, v = A.paged_read(table=table, lengths=ints(lens), cu=ints(every), tokens=every[-1], dtype=FP, **cache)
    # scores of a few units, by queries that fp16 holds well
    size = {"v": 1.0, "k": 2.0 ** 10 if kind is I8 else 2.0 ** -8}[which]
    q = (torch.randn(off[-1], hq, d, generator=g, device=DEV) * size).half()
    scale = 2.0 / (size * d ** 0.5 * max(k.float().square().mean().sqrt().item(), 2.0 ** -30))
    got = A.paged_attention(q, table=table, lengths=ints(lens), cu=ints(off), scale=scale, **cache)
    for b, (lo, hi) in enumerate(zip(off, off[1:])):
        want, bound = reference(q[lo:hi], k[every[b]:every[b + 1]], v[every[b]:every[b + 1]], lens[b] - chunks[b], scale)
        check16(got[lo:hi], want, bound + 2.0 ** -25, f"sequence {b}")


@pytest.mark.parametrize("n,rows", [(200, 1), (200, 90), (5000, 1), (5000, 3), (3000, 200)])
def test_values_that_are_all_the_greatest(n, rows):
    """Their mean is no more than that, however the probabilities are rounded: finite, also joined of parts."""
    print(f"\n[all greatest] {n} {rows}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(22)
    pages, d = -(-n // 16), 128
    k = torch.randint(-127, 128, (pages, 16, 1, d), generator=g, device=DEV).to(torch.int8)
    v = torch.full((pages, 16, 1, d), 100, dtype=torch.int8, device=DEV)
    v[..., 1::2] = -100
    ks = torch.full((pages, 1, 1), 121, dtype=torch.uint8, device=DEV).view(E8M0)
    vs = torch.full((pages, 1, 1), 140, dtype=torch.uint8, device=DEV).view(E8M0)
    q = torch.randn(rows, 4, d, generator=g, device=DEV).half()
    table = torch.arange(pages, dtype=torch.int32, device=DEV)[None]
    got = A.paged_attention(q, k, v, table, ints([n]), ints([0, rows]), k_scales=ks, v_scales=vs).double().cpu()
    want = torch.full((d,), 65504.0, dtype=torch.float64)
    want[1::2] = -65504.0
    assert torch.isfinite(got).all()
    # a probability is off by half a step, 2^-11, or, below fp16's normal values, by 2^-25: of a sum of 1 or more (the greatest's part)
    assert ((got - want).abs() <= 65504.0 * (2.0 ** -11 * 1.01 + 2.0 ** -25 * n + 2.0 ** -11)).all()


@pytest.mark.parametrize("n,rows", [(200, 1), (200, 90), (5000, 1), (5000, 9), (3000, 200)])
@pytest.mark.parametrize("kind", [I8, E4M3])
def test_probabilities_that_all_round_up(n, rows, kind):
    """Of 64 keys one is ahead, and the others' probability of its own is 2^-4 (1 + 2^-11 1.02), which becomes 2^-4 (1 + 2^-10): the sum of
    the rounded ones is 63/16 2^-11 over 1 + 63/16, or 2^-11.3, too great, and 65504 times that past where fp16 rounds to infinity
    (2^-12). The result stays the greatest, also joined of parts."""
    print(f"\n[round up] {n} {rows} {kind}", flush=True)
    pages, d = -(-n // 16), 128
    k = torch.zeros(pages * 16, 1, d, device=DEV)
    k[::64, 0, 3] = 1.0
    v = torch.full((pages * 16, 1, d), 100.0, device=DEV)
    v[..., 1::2] = -100.0
    code = lambda x: (x.to(I8) if kind is I8 else x.to(E4M3)).view(pages, 16, 1, d)  # noqa: E731
    ks = torch.full((pages, 1, 1), 127, dtype=torch.uint8, device=DEV).view(E8M0)
    vs = torch.full((pages, 1, 1), 140, dtype=torch.uint8, device=DEV).view(E8M0)
    q = torch.zeros(rows, 4, d, device=DEV).half()
    q[..., 3] = 1.0
    table = torch.arange(pages, dtype=torch.int32, device=DEV)[None]
    got = A.paged_attention(q, code(k), code(v), table, ints([n]), ints([0, rows]), k_scales=ks, v_scales=vs,
                            scale=-math.log(2.0 ** -4 * (1.0 + 2.0 ** -11 * 1.02)))
    want = torch.full((d,), 65504.0, dtype=FP)
    want[1::2] = -65504.0
    assert torch.equal(got.cpu(), want.expand(rows, 4, d))


@pytest.mark.parametrize("n,rows", [(200, 1), (200, 90), (5000, 9), (3000, 200)])
def test_probabilities_that_all_round_up_over_16_bits(n, rows):
    """The same over the cache in 16 bits and over packed sequences; values that are infinite stay so."""
    print(f"\n[round up, 16 bits] {n} {rows}", flush=True)
    pages, d = -(-n // 16), 64
    k = torch.zeros(pages * 16, 1, d, dtype=FP, device=DEV)
    k[::64, 0, 3] = 1.0
    v = torch.full((pages * 16, 1, d), 65504.0, dtype=FP, device=DEV)
    v[..., 1::2] = -65504.0
    v[0, 0, 5] = math.inf  # (none of the probabilities is 0)
    q = torch.zeros(n, 4, d, dtype=FP, device=DEV)
    q[..., 3] = 1.0
    table = torch.arange(pages, dtype=torch.int32, device=DEV)[None]
    scale = -math.log(2.0 ** -4 * (1.0 + 2.0 ** -11 * 1.02))
    want = torch.full((d,), 65504.0, dtype=FP)
    want[1::2] = -65504.0
    want[5] = math.inf
    paged = A.paged_attention(q[:rows], k.view(pages, 16, 1, d), v.view(pages, 16, 1, d), table, ints([n]), ints([0, rows]), scale=scale)
    assert torch.equal(paged.cpu(), want.expand(rows, 4, d))
    packed = A.packed_attention(q, k[:n].contiguous(), v[:n].contiguous(), ints([0, n]), causal=False, scale=scale)
    assert torch.equal(packed.cpu(), want.expand(n, 4, d))
