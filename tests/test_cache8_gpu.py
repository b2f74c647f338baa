"""The paged cache held in 8 bits: paged_append's codes and scales against their definition in float64 (equal, none off), paged_read
against code x scale, and paged_attention over codes against attention in float64 on the values they stand for (element by element,
within the bound of the 16-bit kernels' tests: codes become values exactly, so nothing is added to it but what that bound leaves out,
an fp16 result below its least normal value 2^-14, whose neighbours are 2^-24 apart and which is rounded by up to 2^-25 whatever its
size: int8 codes of 0 at the row's greatest score leave such results)."""

from __future__ import annotations

import math

import pytest
import torch

from byteprof_amd.optim import attention as A
from tests.test_attention_gpu import check as check16
from tests.test_attention_gpu import ints, offsets, one_hot_reference, randn, reference

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
E4M3, I8, E8M0 = torch.float8_e4m3fn, torch.int8, torch.float8_e8m0fnu
GREATEST = {E4M3: 448.0, I8: 127.0}

# the values of the e4m3 codes 0 .. 126: 3 mantissa bits, exponent bias 7, subnormals in steps of 2^-9
TABLE = torch.tensor([(c % 8) * 2.0 ** -9 if c < 8 else (1 + c % 8 / 8) * 2.0 ** (c // 8 - 7) for c in range(127)], dtype=torch.float64)


def check(got, want, bound, what):
    check16(got, want, bound + 2.0 ** -25 if got.dtype == FP else bound, what)


def codes_of(x, kind):
    """x float64 on the CPU to the nearest code (ties to the even one), as uint8 bits."""
    if kind is I8:
        y = torch.round(x.clamp(-127.0, 127.0))
        return torch.where(x.isnan(), 0.0, y).to(torch.int8).view(torch.uint8)
    mid = (TABLE[1:] + TABLE[:-1]) / 2
    a = x.abs().clamp_max(448.0).nan_to_num(0.0)
    code = torch.searchsorted(mid, a)  # the least i with a <= mid[i]: a tie falls to i
    tie = (code < 126) & (a == mid[code.clamp_max(125)])
    code = torch.where(tie & (code % 2 == 1), code + 1, code)
    code = torch.where(x.isnan(), 127, code)
    return (code + 128 * torch.signbit(x)).to(torch.uint8)


def values_of(code, kind):
    """uint8 bits to float64 values, on the CPU."""
    if kind is I8:
        return code.view(torch.int8).double()
    c = code.long()
    return torch.where(c % 128 == 127, math.nan, TABLE[(c % 128).clamp_max(126)]) * torch.where(c >= 128, -1.0, 1.0)


def byte_of(amax, kind):
    """The exponent byte of the least power of two s with amax <= greatest x s."""
    if amax == 0:
        return 0
    m, e = math.frexp(amax / GREATEST[kind])  # amax / greatest = m 2^e, m in [0.5, 1); 448 and 127: the quotient decides m = 0.5
    exact = amax == GREATEST[kind] * 2.0 ** (e - 1)
    return max(0, (e - 1 if exact else e) + 127)


def power(byte):
    return 2.0 ** (byte - 127)


def raw(t):
    return t.view(torch.uint8).cpu()


def empty_cache(pool, page, blocks, hk, d, kind, g):
    """Pages and scales that hold whatever (finite) was there before."""
    pages = torch.randint(0, 100, (2, pool, page, hk, d), generator=g, device=DEV, dtype=torch.uint8)
    scales = torch.randint(100, 150, (2, pool, blocks, hk), generator=g, device=DEV, dtype=torch.uint8)
    return pages[0].view(kind), pages[1].view(kind), scales[0].view(E8M0), scales[1].view(E8M0)


def append_reference(new, pages, scales, table, lens, off, kind, tokens):
    """(pages, scales) as uint8 on the CPU after the append of new [tokens, hk, d], by the definition."""
    pages, scales, table = raw(pages).clone(), raw(scales).clone(), table.tolist()
    pool, page, hk, d = pages.shape
    block = page // scales.shape[1]
    new = new.double().cpu()
    for b, n in enumerate(lens):
        begin, end = max(off[b], 0), min(off[b + 1], tokens)
        start = n - (end - begin)
        for at in range(max(start, 0) // block * block, min(n, page * len(table[b])), block):
            lo, hi = max(at, start), min(at + block, n)
            id = table[b][at // page]
            if hi <= lo or not 0 <= id < pool:
                continue
            x = new[end - n + lo:end - n + hi]
            slot, blk = at % page, at % page // block
            for h in range(hk):
                fine = x[:, h][x[:, h].isfinite()]
                byte = byte_of(fine.abs().max().item() if fine.numel() else 0.0, kind)
                if start > at:
                    had = scales[id, blk, h].item()
                    byte = max(byte, had)
                    old = pages[id, slot:slot + lo - at, h]
                    if byte > had:
                        pages[id, slot:slot + lo - at, h] = codes_of(values_of(old, kind) * 2.0 ** (had - byte), kind)
                pages[id, slot + lo - at:slot + hi - at, h] = codes_of(x[:, h] / power(byte), kind)
                scales[id, blk, h] = byte
    return pages, scales


APPEND = [
    # lens, chunks, page, block, hk, d, cache, dtype
    ([1], [1], 16, 16, 1, 128, E4M3, BF),
    ([155], [1], 16, 16, 16, 128, I8, BF),
    ([9, 30, 3, 12, 2], [1, 30, 5, 0, 2], 4, 4, 3, 24, E4M3, FP),
    ([100, 64, 33, 257], [37, 64, 1, 200], 64, 16, 2, 64, I8, FP),
    ([300, 20], [300, 7], 256, 256, 1, 80, E4M3, BF),  # a unit of more pieces than a wave holds
    ([700], [650], 128, 128, 1, 256, I8, F32),  # than a workgroup holds
    ([50, 51], [20, 51], 12, 6, 5, 7, E4M3, F32),  # rows of no whole pieces, a block that no tile of the attention takes
    ([33, 40], [33, 3], 5, 1, 2, 40, I8, FP),
    ([70 + i for i in range(150)], [i % 5 for i in range(150)], 8, 8, 2, 64, E4M3, BF),  # more sequences than lanes, some without tokens
    ([20] * 70, [1] * 70, 16, 8, 1, 72, I8, BF),
]


@pytest.mark.parametrize("lens,chunks,page,block,hk,d,kind,dtype", APPEND)
def test_append(lens, chunks, page, block, hk, d, kind, dtype):
    """Codes and scales equal the definition's, and nothing else changes; bad pages and rows of no chunk are left out."""
    print(f"\n[append8] {lens[:5]} {chunks[:5]} page {page} block {block} {hk} x {d} {kind} {dtype}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(1)
    need = [-(-n // page) + 1 for n in lens]
    pool = sum(need) + 2
    kp, vp, ks, vs = empty_cache(pool, page, page // block, hk, d, kind, g)
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32, device=DEV)
    order = torch.randperm(pool, generator=g, device=DEV).to(torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = order[sum(need[:b]):sum(need[:b]) + n]
    if len(lens) > 3:
        table[1, 0], table[2, (lens[2] - 1) // page] = -1, pool
    off = [1 + x for x in offsets(chunks)]  # token 0 and the last two belong to no chunk
    tokens = off[-1] + 2
    make = lambda: (torch.randn(tokens, hk, d, generator=g, device=DEV)  # noqa: E731
                    * torch.exp2(torch.randint(-6, 9, (tokens, hk, 1), generator=g, device=DEV).float())).to(dtype)
    k, v = make(), make()
    v[tokens // 2] = 0.0
    want = [append_reference(x, p, s, table, lens, off, kind, tokens) for x, p, s in ((k, kp, ks), (v, vp, vs))]
    A.paged_append(k, v, kp, vp, table, ints(lens), ints(off), k_scales=ks, v_scales=vs)
    for (pages, scales), p, s in zip(want, (kp, vp), (ks, vs)):
        assert torch.equal(raw(s), scales)
        assert torch.equal(raw(p), pages)


@pytest.mark.parametrize("kind", [E4M3, I8])
def test_append_token_by_token(kind):
    """A block that fills up one token at a time, each greater than those before it: rounded again at every growth, and equal to the
    definition after every call."""
    print(f"\n[append8] one by one {kind}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(2)
    kp, vp, ks, vs = empty_cache(3, 16, 2, 2, 32, kind, g)
    table = ints([[2, 0]])
    for n in range(1, 30):
        k, v = (torch.randn(1, 2, 32, generator=g, device=DEV) * 1.7 ** (n % 9) for _ in range(2))
        want = [append_reference(x, p, s, table, [n], [0, 1], kind, 1) for x, p, s in ((k, kp, ks), (v, vp, vs))]
        A.paged_append(k, v, kp, vp, table, ints([n]), ints([0, 1]), k_scales=ks, v_scales=vs)
        assert torch.equal(raw(ks), want[0][1]) and torch.equal(raw(vs), want[1][1]), n
        assert torch.equal(raw(kp), want[0][0]) and torch.equal(raw(vp), want[1][0]), n


@pytest.mark.parametrize("kind", [E4M3, I8])
@pytest.mark.parametrize("dtype", [BF, FP, F32])
def test_append_borders(kind, dtype):
    """Greatest values on either side of a power of two times the greatest code, ties, zeros of both signs, the type's least and
    greatest values, infinities and NaN; a block of nothing but those."""
    print(f"\n[append8] borders {kind} {dtype}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(3)
    info, q = torch.finfo(dtype), GREATEST[kind]
    up = lambda x: x * (1 + 2 * info.eps)  # noqa: E731
    rows = [[q, 1.5, 2.5, -0.5], [up(q), q, 3.5, -1.5], [q / 64, up(q / 128), 0.0, -0.0], [0.0, -0.0, 0.0, 0.0],
            [info.max, info.tiny, -info.max, 1.0], [info.tiny, -info.tiny, info.tiny / 4, 0.0], [math.inf, 1.0, -math.inf, math.nan],
            [math.nan, math.inf, -math.inf, math.nan], [q * 0.5, up(q * 0.5), -q * 0.25, q / 1024], [17.0, 18.0, 19.0, 21.0]]
    x = torch.tensor(rows, dtype=F32, device=DEV).repeat_interleave(2, 1).to(dtype)[:, None, :].contiguous()  # [10, 1, 8]
    y = x.flip(0).contiguous()
    kp, vp, ks, vs = empty_cache(len(rows) + 1, 4, 1, 1, 8, kind, g)
    table = torch.arange(len(rows), dtype=torch.int32, device=DEV)[:, None]
    cu, lens = list(range(len(rows) + 1)), [1] * len(rows)
    want = [append_reference(a, p, s, table, lens, cu, kind, len(rows)) for a, p, s in ((x, kp, ks), (y, vp, vs))]
    A.paged_append(x, y, kp, vp, table, ints(lens), ints(cu), k_scales=ks, v_scales=vs)
    for (pages, scales), p, s in zip(want, (kp, vp), (ks, vs)):
        assert torch.equal(raw(s), scales)
        got = raw(p)
        if kind is E4M3:  # the sign of a NaN says nothing
            got, pages = (torch.where(t % 128 == 127, torch.tensor(127, dtype=torch.uint8), t) for t in (got, pages))
        assert torch.equal(got, pages)


def test_append_strides_and_slices():
    """k and v as slices of one projection, keys and values in one pool of any strides: the same as from tensors of their own."""
    g = torch.Generator(device=DEV).manual_seed(4)
    page, hk, d, lens, chunks = 16, 2, 64, [100, 37], [60, 1]
    kp, vp, ks, vs = empty_cache(12, page, 2, hk, d, E4M3, g)
    table = ints([[0, 1, 2, 3, 4, 5, 6], [8, 10, 9, -1, -1, -1, -1]])
    qkv = randn(g, 61, 3 * hk, d, dtype=BF)
    k, v = qkv[:, hk:2 * hk], qkv[:, 2 * hk:]
    both = torch.stack([raw(kp), raw(vp)], 1).to(DEV).transpose(2, 3).contiguous()  # [pool, 2, hk, page, d]
    kq, vq = both[:, 0].transpose(1, 2).view(E4M3), both[:, 1].transpose(1, 2).view(E4M3)
    st = torch.stack([raw(ks), raw(vs)], 0).to(DEV).permute(0, 3, 2, 1).contiguous()  # [2, hk, blocks, pool]
    kt, vt = st[0].permute(2, 1, 0).view(E8M0), st[1].permute(2, 1, 0).view(E8M0)
    args = (table, ints(lens), ints(offsets(chunks)))
    A.paged_append(k, v, kq, vq, *args, k_scales=kt, v_scales=vt)
    A.paged_append(k.contiguous(), v.contiguous(), kp, vp, *args, k_scales=ks, v_scales=vs)
    for a, b in ((kq, kp), (vq, vp), (kt, ks), (vt, vs)):
        assert torch.equal(raw(a.contiguous()), raw(b))
    got = A.paged_read(kq, vq, *args, 61, k_scales=kt, v_scales=vt)
    for a, b in zip(got, A.paged_read(kp, vp, *args, 61, k_scales=ks, v_scales=vs)):
        assert torch.equal(a, b)
    q = randn(g, 61, 4, d, dtype=BF)
    want = A.paged_attention(q, kp, vp, *args, k_scales=ks, v_scales=vs)
    assert torch.isfinite(want).all()
    assert torch.equal(A.paged_attention(q, kq, vq, *args, k_scales=kt, v_scales=vt), want)


def cache_state(lens, page, block, hk, d, kind, g, spare=3, spread=2, finite=True):
    """A pool whose unused places hold NaN (int8: 127 at a huge scale), a table whose unused entries are far out of range, and the
    sequences' values in float64 on the GPU. finite: without the NaN codes of the few values past 448."""
    need = [-(-n // page) for n in lens]
    pool = sum(need) + spare
    order = torch.randperm(pool, generator=g, device=DEV)[:sum(need)].to(torch.int32)
    table = torch.full((len(lens), max(need) + 1), 2 ** 31 - 1, dtype=torch.int32, device=DEV)
    outs, rows = [], []
    for _ in range(2):
        codes = torch.full((pool, page, hk, d), 127, dtype=torch.uint8, device=DEV)
        scales = torch.full((pool, page // block, hk), 255, dtype=torch.uint8, device=DEV)
        used, vals = 0, []
        for b, n in enumerate(lens):
            ids = order[used:used + need[b]].long()
            table[b, :need[b]] = ids.to(torch.int32)
            used += need[b]
            x = torch.randn(need[b] * page, hk, d, generator=g, device=DEV)
            x = x.clamp(-4.48, 4.48) if finite else x
            c = (x * 100).to(E4M3).view(torch.uint8) if kind is E4M3 else (x * 32).round().clamp(-127, 127).to(I8).view(torch.uint8)
            unit = 120 if kind is E4M3 else 122
            s = torch.randint(unit - spread, unit + spread + 1, (need[b], page // block, hk), generator=g, device=DEV).to(torch.uint8)
            at = torch.arange(n, device=DEV)
            codes[ids[at // page], at % page] = c[:n]
            scales[ids] = s
            val = values_of(c[:n].cpu(), kind).to(DEV)
            vals.append(val * torch.exp2(s.view(-1, hk)[at // block].double() - 127)[..., None])
        outs.append((codes.view(kind), scales.view(E8M0)))
        rows.append(vals)
    return outs[0][0], outs[1][0], outs[0][1], outs[1][1], table, rows[0], rows[1]


READ = [
    ([1], [1], 16, 16, 1, 128, E4M3, BF),
    ([161, 40, 0, 300], [161, 3, 0, 299], 16, 4, 3, 40, I8, FP),
    ([129, 77], [100, 77], 7, 7, 2, 72, E4M3, F32),
    ([500] * 70, [i % 9 for i in range(70)], 64, 32, 1, 64, I8, BF),
    ([600, 20], [600, 20], 256, 64, 2, 256, E4M3, FP),
    ([90, 3], [80, 3], 32, 8, 1, 8, I8, F32),
    ([1500, 0, 700], [1500, 0, 690], 16, 16, 1, 8, I8, BF),  # a piece a token
    ([40, 3], [2, 3], 16, 16, 40, 256, E4M3, BF),  # a token of more pieces than a workgroup has
]


@pytest.mark.parametrize("lens,chunks,page,block,hk,d,kind,dtype", READ)
def test_read(lens, chunks, page, block, hk, d, kind, dtype):
    """Values equal code x scale (NaN codes among them); rows of no sequence are zeros."""
    print(f"\n[read] {lens[:5]} {chunks[:5]} page {page} block {block} {hk} x {d} {kind} {dtype}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(5)
    kp, vp, ks, vs, table, kv, vv = cache_state(lens, page, block, hk, d, kind, g, finite=False)
    off = [2 + x for x in offsets(chunks)]
    got = A.paged_read(kp, vp, table, ints(lens), ints(off), off[-1] + 3, k_scales=ks, v_scales=vs, dtype=dtype)
    for out, vals in zip(got, (kv, vv)):
        assert out.dtype == dtype and out.shape == (off[-1] + 3, hk, d)
        for b, (a, z) in enumerate(zip(off, off[1:])):
            assert torch.allclose(out[a:z].double(), vals[b][lens[b] - chunks[b]:], rtol=0.0, atol=0.0, equal_nan=True)
        assert not out[:2].any() and not out[off[-1]:].any()


def test_read_of_a_16_bit_cache_and_what_it_does_not_have():
    g = torch.Generator(device=DEV).manual_seed(6)
    kp, vp = randn(g, 9, 16, 2, 64, dtype=FP), randn(g, 9, 16, 2, 64, dtype=FP)
    table, lens, cu = ints([[3, 8], [-1, 4]]), ints([20, 40]), ints([0, 22, 62])  # 2 before the first position, 8 past the table
    k, v = A.paged_read(kp, vp, table, lens, cu, 70)
    for out, pool in ((k, kp), (v, vp)):
        assert not out[:2].any() and torch.equal(out[2:22], torch.cat([pool[3], pool[8, :4]]))
        assert out[22:38].isnan().all() and torch.equal(out[38:54], pool[4]) and not out[54:].any()
    assert A.paged_read(kp, vp, table, lens, cu, 0)[0].shape == (0, 2, 64)
    k, v = A.paged_read(kp, vp, table[:0], lens[:0], cu[:1], 5)
    assert not k.any() and not v.any()


ATTEND = [
    # lens, chunks, page, block, hq, hk, d, cache, dtype
    ([1], [1], 16, 16, 1, 1, 128, E4M3, BF),
    ([161], [1], 16, 16, 16, 16, 128, I8, BF),
    ([5, 300, 64, 33], [1, 1, 1, 1], 8, 4, 8, 2, 64, E4M3, FP),
    ([900, 130, 77, 9], [9, 9, 9, 9], 64, 32, 16, 4, 128, I8, FP),
    ([400, 90, 700], [129, 90, 3], 32, 32, 4, 1, 96, E4M3, BF),
    ([129, 40, 260], [40, 0, 200], 12, 12, 6, 2, 80, I8, FP),  # blocks of no power of two
    ([50, 257, 31], [1, 33, 31], 4, 4, 5, 1, 40, E4M3, BF),  # rows of 40 bytes: 8 codes at a time
    ([600, 300], [5, 80], 128, 64, 4, 2, 256, E4M3, BF),
    ([333, 1024], [1, 1], 256, 256, 8, 1, 256, I8, FP),
    ([300, 77, 700], [70, 70, 65], 20, 20, 4, 2, 256, I8, BF),
    ([5000, 17], [1, 1], 16, 16, 4, 1, 128, E4M3, BF),  # divided
    ([3000, 2600], [200, 7], 16, 8, 2, 2, 64, I8, BF),
    ([2049], [2], 16, 16, 1, 1, 256, E4M3, FP),
    ([4, 0, 2], [4, 0, 2], 16, 16, 2, 1, 64, I8, BF),
    ([40 + i for i in range(130)], [1 + i % 3 for i in range(130)], 16, 16, 2, 1, 64, E4M3, FP),
    ([600 + i for i in range(70)], [1 + 40 * (i % 2) for i in range(70)], 16, 16, 2, 1, 64, I8, FP),  # more sequences than lanes
    ([260, 900], [3, 40], 24, 8, 160, 1, 64, E4M3, FP),  # more query heads to a key head than a tile has rows
    ([4000, 3900, 10], [1, 1, 1], 12, 4, 4, 1, 72, E4M3, BF),
    ([6000], [150], 16, 16, 1, 1, 64, I8, FP),  # large tiles of many parts
    ([1300, 2000], [400, 129], 48, 48, 3, 3, 96, I8, BF),
    ([700, 900], [1, 2], 32, 16, 20, 1, 128, I8, BF),
    ([700, 1500, 3], [1, 1, 1], 32, 16, 16, 1, 96, E4M3, FP),
    ([20, 40], [20, 33], 8, 8, 2, 1, 8, I8, FP),
]


@pytest.mark.parametrize("lens,chunks,page,block,hq,hk,d,kind,dtype", ATTEND)
def test_attention(lens, chunks, page, block, hq, hk, d, kind, dtype):
    print(f"\n[attention8] {lens[:5]} {chunks[:5]} page {page} block {block} {hq}/{hk} x {d} {kind} {dtype}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(7)
    kp, vp, ks, vs, table, kv, vv = cache_state(lens, page, block, hk, d, kind, g)
    off = offsets(chunks)
    q = randn(g, off[-1] + 2, hq, d, dtype=dtype)
    got = A.paged_attention(q, kp, vp, table, ints(lens), ints(off), k_scales=ks, v_scales=vs)
    for b, (a, z) in enumerate(zip(off, off[1:])):
        want, bound = reference(q[a:z], kv[b], vv[b], lens[b] - chunks[b], d ** -0.5)
        check(got[a:z], want, bound, f"sequence {b}")
    assert not got[off[-1]:].any()


@pytest.mark.parametrize("kind", [E4M3, I8])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_attention_of_every_code(kind, dtype):
    """Every code at every column, keys and values, at scales far from 1 (fp16: past its range, where its greatest value stands for
    them): one position, whose value is the result."""
    g = torch.Generator(device=DEV).manual_seed(8)
    hk, d = 4, 64
    codes = torch.arange(256, dtype=torch.uint8, device=DEV).view(1, 1, hk, d)
    if kind is E4M3:
        codes = torch.where(codes % 128 == 127, torch.zeros_like(codes), codes)
    codes = codes.expand(1, 4, hk, d).contiguous()
    for byte in (127, 110, 135) if dtype == FP else (127, 90, 160):
        scales = torch.full((1, 1, hk), byte, dtype=torch.uint8, device=DEV)
        want = values_of(codes.cpu(), kind)[0, :1] * power(byte)
        want = (want.clamp(-65504.0, 65504.0) if dtype == FP else want).to(dtype)
        where = (ints([[0]]), ints([1]), ints([0, 1]))
        got = A.paged_attention(randn(g, 1, hk, d, dtype=dtype), torch.zeros_like(codes).view(kind), codes.view(kind), *where,
                                k_scales=scales.view(E8M0), v_scales=scales.view(E8M0))
        assert torch.equal(got.cpu(), want), byte
        back = A.paged_read(codes.view(kind), codes.view(kind), *where, 1, k_scales=scales.view(E8M0), v_scales=scales.view(E8M0),
                            dtype=dtype)
        assert torch.equal(back[0].cpu(), want) and torch.equal(back[1].cpu(), want)


def test_rows_that_see_nothing_and_lengths_past_the_table():
    g = torch.Generator(device=DEV).manual_seed(9)
    kp, vp, ks, vs, table, kv, vv = cache_state([3, 300, 64], 16, 16, 1, 64, E4M3, g)
    scales = {"k_scales": ks, "v_scales": vs}
    q = randn(g, 312, 2, 64, dtype=BF)
    got = A.paged_attention(q, kp, vp, table[:2], ints([3, 0]), ints([0, 8, 12]), **scales)
    assert not got[:5].any() and not got[8:].any()
    want, bound = reference(q[5:8], kv[0], vv[0], 0, 64 ** -0.5)
    check(got[5:8], want, bound, "the rows with keys")
    got = A.paged_attention(q, kp, vp, table[:2], ints([-5, 100]), ints([0, 12, 312]), **scales)  # 300 rows, 100 positions
    assert not got[:212].any()
    want, bound = reference(q[212:], kv[1][:100], vv[1][:100], 0, 64 ** -0.5)
    check(got[212:], want, bound, "the last 100")
    got = A.paged_attention(q[:6], kp, vp, table[2:, :4], ints([1000]), ints([-1, 900]), **scales)
    want, bound = reference(q[:6], kv[2], vv[2], 58, 64 ** -0.5)
    check(got, want, bound, "offsets and a length that are cut")
    assert not A.paged_attention(q, kp, vp, table[:0], ints([]), ints([0]), **scales).any()
    assert A.paged_attention(q[:0], kp, vp, table, ints([1, 1, 1]), ints([0, 0, 0, 0]), **scales).shape == (0, 2, 64)


@pytest.mark.parametrize("n,chunk", [(100, 1), (100, 90), (3000, 1), (3000, 90)])
def test_bad_pages_and_nan_codes_give_nan_rows(n, chunk):
    """Ids outside the pool and NaN codes and scales below a sequence's length (its own rows become NaN); others are untouched."""
    print(f"\n[attention8 bad pages] {n} {chunk}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(10)
    lens, chunks = [n, 200, n, n, n], [chunk, 3, chunk, chunk, chunk]
    kp, vp, ks, vs, table, kv, vv = cache_state(lens, 16, 16, 1, 64, E4M3, g)
    vp.view(torch.uint8)[table[3, 1], 5, 0, :] = 0x7f
    ks.view(torch.uint8)[table[4, (n - 1) // 16], 0, 0] = 255
    table[0, 2], table[2, (n - 1) // 16] = -1, kp.shape[0]
    off = offsets(chunks)
    q = randn(g, off[-1], 1, 64, dtype=BF)
    got = A.paged_attention(q, kp, vp, table, ints(lens), ints(off), k_scales=ks, v_scales=vs)
    for b in (0, 2, 3, 4):
        assert got[off[b]:off[b + 1]][-1].isnan().all(), b
    want, bound = reference(q[off[1]:off[2]], kv[1], vv[1], 197, 64 ** -0.5)
    check(got[off[1]:off[2]], want, bound, "the good sequence")


@pytest.mark.parametrize("kind", [E4M3, I8])
@pytest.mark.parametrize("dtype,byte,a", [(BF, 127 + 60, 2.0 ** 40), (BF, 127 + 8, 2.0 ** 13), (FP, 127 + 6, 2.0 ** 14)])
def test_scores_far_from_zero(kind, dtype, byte, a):
    """Finite scores of any size, positive and negative, tied, beside rows of zeros."""
    print(f"\n[attention8 far] {kind} {dtype} {byte}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(11)
    d = 64
    for n, rows, hq in ((5000, 1, 1), (900, 9, 4), (33, 2, 1), (700, 100, 2)):
        pages = -(-n // 16)
        c = torch.zeros(pages * 16, 1, d, device=DEV)
        c[:, 0, 5] = torch.randint(64, 128, (len(c),), generator=g, device=DEV) // 8 * 8.0  # 8 values, exact in either code
        codes = (c.to(E4M3) if kind is E4M3 else c.to(I8)).view(pages, 16, 1, d)
        q = torch.zeros(rows, hq, d, device=DEV)
        q[..., 5] = torch.tensor([a, -a, 0.0], device=DEV)[torch.randint(0, 3, (rows, hq), generator=g, device=DEV)]
        v = torch.randint(-8, 9, (pages * 16, 1, d), generator=g, device=DEV).float()
        vcodes = (v.to(E4M3) if kind is E4M3 else v.to(I8)).view(pages, 16, 1, d)
        ks = torch.full((pages, 2, 1), byte, dtype=torch.uint8, device=DEV).view(E8M0)
        vs = torch.full((pages, 2, 1), 127, dtype=torch.uint8, device=DEV).view(E8M0)
        q = q.to(dtype)
        table = torch.arange(pages, dtype=torch.int32, device=DEV)[None]
        got = A.paged_attention(q, codes, vcodes, table, ints([n]), ints([0, rows]), k_scales=ks, v_scales=vs, scale=1.0)
        for h in range(hq):
            want, bound = one_hot_reference(q[:, h:h + 1], c[:n].double() * power(byte), v[:n], n - rows, 1.0, dtype)
            check(got[:, h], want, bound, f"{n} keys, {rows} rows, head {h}")


def test_far_pages():
    """Pages whose byte offset passes 2^32: appended to, read, attended."""
    page, hk, d, n = 16, 8, 128, 50
    pool = (2 ** 32 + 2 ** 28) // (page * hk * d)
    g = torch.Generator(device=DEV).manual_seed(12)
    kp, vp = (torch.empty(pool, page, hk, d, dtype=E4M3, device=DEV) for _ in range(2))
    ks, vs = (torch.empty(pool, 1, hk, dtype=E8M0, device=DEV) for _ in range(2))
    where = (ints([[pool - 1, 5, pool - 3, pool // 2 + 1]]), ints([n]))
    k, v = randn(g, n, hk, d, dtype=BF), randn(g, n, hk, d, dtype=BF)
    near = [torch.zeros(4, page, hk, d, dtype=E4M3, device=DEV) for _ in range(2)] + [
        torch.zeros(4, 1, hk, dtype=E8M0, device=DEV) for _ in range(2)]
    there = (torch.arange(4, dtype=torch.int32, device=DEV)[None], ints([n]))
    q = randn(g, 2, hk, d, dtype=BF)
    outs = []
    for (a, b, c, e), (table, lens) in (((kp, vp, ks, vs), where), (near, there)):
        A.paged_append(k, v, a, b, table, lens, ints([0, n]), k_scales=c, v_scales=e)
        outs.append((*A.paged_read(a, b, table, lens, ints([0, n]), n, k_scales=c, v_scales=e),
                     A.paged_attention(q, a, b, table, lens, ints([0, 2]), k_scales=c, v_scales=e)))
    for x, y in zip(*outs):
        assert torch.equal(x, y)
    assert ((outs[0][0].float() - k.float()).abs().amax() <= 2.0 ** -4 * k.float().abs().amax()).item()


def test_graph_replays_follow_the_lengths():
    """Append, attention and read captured once; at every replay the lengths, the offsets and the inputs are others."""
    g = torch.Generator(device=DEV).manual_seed(13)
    page, hk, hq, d, tokens = 16, 2, 4, 64, 100
    kp, vp, ks, vs, table, _, _ = cache_state([1200, 900], page, 8, hk, d, I8, g)
    ks.view(torch.uint8)[ks.view(torch.uint8) == 255] = 120
    vs.view(torch.uint8)[vs.view(torch.uint8) == 255] = 120
    table.clamp_max_(kp.shape[0] - 1)
    q, k, v = randn(g, tokens, hq, d, dtype=BF), randn(g, tokens, hk, d, dtype=BF), randn(g, tokens, hk, d, dtype=BF)
    lengths, cu = ints([1200, 900]), ints([0, 90, 100])
    out = torch.empty(tokens, hq, d, dtype=BF, device=DEV)
    scales = {"k_scales": ks, "v_scales": vs}

    def step():
        A.paged_append(k, v, kp, vp, table, lengths, cu, **scales)
        A.paged_attention(q, kp, vp, table, lengths, cu, out=out, **scales)
        return A.paged_read(kp, vp, table, lengths, cu, tokens, **scales)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        back = step()
    for lens, off in (([1200, 900], [0, 90, 100]), ([33, 70], [0, 33, 99]), ([1, 850], [0, 1, 2]), ([500, 0], [0, 100, 100])):
        q.copy_(randn(g, tokens, hq, d, dtype=BF))
        k.copy_(randn(g, tokens, hk, d, dtype=BF))
        lengths.copy_(ints(lens))
        cu.copy_(ints(off))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (out, *back)]
        again = step()
        torch.cuda.synchronize()
        for x, y in zip(got, (out, *again)):
            assert torch.equal(x, y)


def test_in_place_another_stream_and_two_calls_alike():
    g = torch.Generator(device=DEV).manual_seed(14)
    kp, vp, ks, vs, table, _, _ = cache_state([3000, 500], 16, 16, 2, 128, E4M3, g)
    args = (kp, vp, table, ints([3000, 500]), ints([0, 100, 103]))
    scales = {"k_scales": ks, "v_scales": vs}
    q = randn(g, 103, 4, 128, dtype=BF)
    want = A.paged_attention(q, *args, **scales)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = A.paged_attention(q, *args, **scales)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want) and torch.equal(A.paged_attention(q, *args, **scales), want)
    assert A.paged_attention(q, *args, out=q, **scales) is q and torch.equal(q, want)


def test_a_run_of_them_together():
    """Prompts appended, then steps of one token and of several: the attention over the 8-bit cache equals attention in float64 on
    what paged_read gives back."""
    g = torch.Generator(device=DEV).manual_seed(15)
    page, block, hk, hq, d = 16, 16, 2, 8, 128
    for kind in (E4M3, I8):
        kp, vp, ks, vs = empty_cache(40, page, page // block, hk, d, kind, g)
        table = torch.randperm(40, generator=g, device=DEV)[:39].to(torch.int32).view(3, 13)
        lens, scales = [0, 0, 0], {"k_scales": ks, "v_scales": vs}
        for chunks in ([100, 37, 64], [1, 1, 1], [1, 1, 1], [5, 0, 9], [1, 1, 1], [60, 1, 30]):
            lens = [n + c for n, c in zip(lens, chunks)]
            off, every = offsets(chunks), offsets(lens)
            k, v, q = (randn(g, off[-1], n, d, dtype=BF) for n in (hk, hk, hq))
            A.paged_append(k, v, kp, vp, table, ints(lens), ints(off), **scales)
            got = A.paged_attention(q, kp, vp, table, ints(lens), ints(off), **scales)
            kr, vr = A.paged_read(kp, vp, table, ints(lens), ints(every), every[-1], **scales)
            for b, (a, z) in enumerate(zip(off, off[1:])):
                want, bound = reference(q[a:z], kr[every[b]:every[b + 1]], vr[every[b]:every[b + 1]], lens[b] - chunks[b], d ** -0.5)
                check(got[a:z], want, bound, f"sequence {b}")


def test_written_tensors_count_as_changed_and_gradients_are_refused():
    g = torch.Generator(device=DEV).manual_seed(16)
    q = randn(g, 4, 1, 64, dtype=BF)
    kp, vp, ks, vs = empty_cache(1, 16, 1, 1, 64, I8, g)
    args, scales = (ints([[0]]), ints([4]), ints([0, 4])), {"k_scales": ks, "v_scales": vs}
    before = [t._version for t in (kp, vp, ks, vs)]
    A.paged_append(q, q, kp, vp, *args, **scales)
    assert all(t._version > n for t, n in zip((kp, vp, ks, vs), before))
    out = torch.zeros_like(q)
    n = out._version
    A.paged_attention(q, kp, vp, *args, out=out, **scales)
    assert out._version > n
    w = q.clone().requires_grad_()
    with pytest.raises(ValueError, match="no backward"):
        A.paged_attention(w, kp, vp, *args, **scales)
    with pytest.raises(ValueError, match="no backward"):
        A.paged_append(q, w, kp, vp, *args, **scales)
    with pytest.raises(ValueError, match="all tensors must be on"):
        A.paged_attention(q, kp, vp, *args, k_scales=ks, v_scales=vs.cpu())
    with pytest.raises(ValueError, match="overlap"):
        flat = kp.view(-1)[:512].view(BF).view(4, 1, 64)
        A.paged_attention(q, kp, vp, *args, out=flat, **scales)
    from torch.autograd import forward_ad
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(q, q)
        for call in (lambda: A.paged_attention(dual, kp, vp, *args, **scales), lambda: A.paged_append(dual, q, kp, vp, *args, **scales)):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
