"""Every code at every scale as the value it stands for: what paged_read gives, attention over one position (whose value is the result),
and keys that decide between positions: attention over codes is attention over paged_read's values, whichever kernel takes the launch.

code x scale is exact in float64, and its rounding to the outputs' type (past fp16's range its greatest value) is the definition: values
are equal to it, no tolerance. The scores of the keys are exact in float32, so what is left there is one_hot_reference's bound and the
2^-25 by which an fp16 result below its normal values may be rounded."""

from __future__ import annotations

import pytest
import torch

from byteprof_amd.optim import attention as A
from tests.test_attention_gpu import check as check16
from tests.test_attention_gpu import ints, one_hot_reference
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
