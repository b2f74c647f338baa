"""packed_attention, paged_append and paged_attention against attention in float64, element by element.

The bound of an element, with h half a step of the output's type (relative), A = sum_j p_j |v_j| and d the head dimension: the
result is rounded once (h |o|) and the probabilities once each (h A); a score is a float32 sum of d products (its error at
most d 2^-24 sum |q k| scale, which moves a probability and the total by as much, relatively); exp2, the sums and the joins of
parts add a few float32 steps (2^-18 A in all). fp16 probabilities below 2^-14 of the row's greatest are rounded to multiples
of 2^-24: 2^-25 each, times |v|."""

from __future__ import annotations

import math

import pytest
import torch

from byteprof_amd.optim import attention as A

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, FP = torch.bfloat16, torch.float16


def reference(q, k, v, first, scale):
    """q [n, Hq, D] at positions first + i (None: sees all) over k, v [m, Hk, D]: (out, bound) in float64 on the CPU."""
    h = torch.finfo(q.dtype).eps / 2
    tiny = 2.0 ** -25 if q.dtype == FP else 0.0
    n, hq, d = q.shape
    m, hk = k.shape[:2]
    q, k, v = (t.double().cpu() for t in (q, k, v))
    out, bound = torch.zeros(n, hq, d, dtype=torch.float64), torch.zeros(n, hq, d, dtype=torch.float64)
    if m == 0:
        return out, bound
    for head in range(hq):
        qh, kh, vh = q[:, head], k[:, head * hk // hq], v[:, head * hk // hq]
        s = qh @ kh.T * scale
        off = (d + 4) * 2.0 ** -24 * (qh.abs() @ kh.abs().T).amax(-1, keepdim=True) * scale
        seen = torch.ones(n, m, dtype=torch.bool)
        if first is not None:
            seen = torch.arange(m)[None, :] <= first + torch.arange(n)[:, None]
        s = torch.where(seen, s, -math.inf)
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
        z = p.sum(-1, keepdim=True)
        p = torch.where(z > 0, p / z, 0.0)
        o, a = p @ vh, p @ vh.abs()
        out[:, head] = o
        bound[:, head] = h * o.abs() * 1.01 + (h * 1.01 + 2 * off + 2.0 ** -18) * a + tiny * (seen.double() @ vh.abs())
    return out, bound


def check(got, want, bound, what):
    got = got.double().cpu()
    assert torch.isfinite(got).all(), what
    worst = ((got - want).abs() / bound.clamp_min(1e-30)).max().item() if got.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst} of the bound"


def ints(xs):
    return torch.tensor(xs, dtype=torch.int32, device=DEV)


def offsets(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def randn(g, *shape, dtype):
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


PACKED = [
    # lens, hq, hk, d, dtype, causal, pad, fused
    ([1], 1, 1, 128, BF, True, 0, False),
    ([17, 1, 0, 64, 160], 4, 4, 128, BF, True, 0, True),
    ([31, 32, 33, 63, 65], 8, 2, 64, FP, True, 5, False),
    ([127, 128, 129], 6, 2, 96, BF, True, 3, True),
    ([300, 2, 77], 5, 1, 40, FP, False, 1, False),
    ([129, 500], 3, 3, 80, BF, False, 130, True),
    ([200, 33, 70], 7, 1, 256, BF, True, 9, False),
    ([200, 33], 4, 2, 256, FP, False, 0, True),
    ([65, 66], 28, 4, 200, BF, True, 0, False),
    ([20, 40], 2, 1, 8, FP, True, 2, False),
    ([1500, 900], 2, 1, 128, BF, True, 0, False),  # long, few heads: the keys of a tile are divided
    ([1500], 1, 1, 256, FP, False, 0, False),
    ([700] * 3 + [0] * 70 + [5] * 70, 1, 1, 64, BF, True, 0, False),  # more sequences than a wave's lanes
    ([3, 40, 1], 200, 1, 64, BF, True, 2, False),  # more query heads to a key head than a tile has rows
    ([9, 30], 129, 3, 72, FP, False, 0, False),
]


@pytest.mark.parametrize("lens,hq,hk,d,dtype,causal,pad,fused", PACKED)
def test_packed(lens, hq, hk, d, dtype, causal, pad, fused):
    print(f"\n[packed] {lens[:6]} {hq}/{hk} x {d} {dtype} causal={causal} pad={pad} fused={fused}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(1)
    off = offsets(lens)
    total = off[-1] + pad
    if fused:
        qkv = randn(g, total, (hq + 2 * hk) * d, dtype=dtype).view(total, hq + 2 * hk, d)
        q, k, v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
    else:
        q, k, v = (randn(g, total, n, d, dtype=dtype) for n in (hq, hk, hk))
    q = q * 2.0 if not fused else q
    if pad:
        k[off[-1]:], v[off[-1]:] = math.nan, math.inf  # rows of no sequence are read by none
    out = torch.full((total, hq, d), math.nan, dtype=dtype, device=DEV)
    got = A.packed_attention(q, k, v, ints(off), causal=causal, out=out)
    assert got is out
    for a, b in zip(off, off[1:]):
        want, bound = reference(q[a:b], k[a:b], v[a:b], 0 if causal else None, d ** -0.5)
        check(got[a:b], want, bound, f"sequence at {a}")
    assert not got[off[-1]:].any()


@pytest.mark.parametrize("causal", [True, False])
def test_packed_many_tiles_in_order(causal):
    """More tiles than the card holds at once, of 2 to 64 sequences: they run longest first, whatever sequence they are of."""
    g = torch.Generator(device=DEV).manual_seed(20)
    lens = [(37 * i * i + 11) % 620 for i in range(64)]
    off = offsets(lens)
    q, k, v = (randn(g, off[-1] + 3, n, 64, dtype=BF) for n in (6, 3, 3))
    print(f"\n[order] packed {off[-1]} causal={causal}", flush=True)
    got = A.packed_attention(q, k, v, ints(off), causal=causal)
    for a, b in zip(off, off[1:]):
        want, bound = reference(q[a:b], k[a:b], v[a:b], 0 if causal else None, 64 ** -0.5)
        check(got[a:b], want, bound, f"sequence at {a}")
    assert not got[off[-1]:].any()


def test_paged_many_tiles_in_order():
    g = torch.Generator(device=DEV).manual_seed(21)
    lens = [(53 * i * i + 7) % 700 for i in range(50)]
    chunks = [min(n, (29 * i) % 300 if i % 3 else 1) for i, n in enumerate(lens)]
    lens[7], chunks[7] = 20, 250  # the first 230 rows see nothing
    print("\n[order] paged", flush=True)
    kp, vp, table, ks, vs = paged_state(lens, 16, 4, 64, FP, g)
    off = offsets(chunks)
    q = randn(g, off[-1], 8, 64, dtype=FP)
    got = A.paged_attention(q, kp, vp, table, ints(lens), ints(off))
    for b, (a, z) in enumerate(zip(off, off[1:])):
        want, bound = reference(q[a:z], ks[b], vs[b], lens[b] - chunks[b], 64 ** -0.5)
        check(got[a:z], want, bound, f"sequence {b}")


def test_packed_rows_before_the_first_sequence_and_a_scale():
    g = torch.Generator(device=DEV).manual_seed(2)
    q, k, v = randn(g, 90, 4, 64, dtype=BF), randn(g, 90, 2, 64, dtype=BF), randn(g, 90, 2, 64, dtype=BF)
    got = A.packed_attention(q, k, v, ints([7, 50, 81]), scale=0.31)
    for a, b in ((7, 50), (50, 81)):
        want, bound = reference(q[a:b], k[a:b], v[a:b], 0, 0.31)
        check(got[a:b], want, bound, f"sequence at {a}")
    assert not got[:7].any() and not got[81:].any()
    assert not A.packed_attention(q, k, v, ints([0])).any()  # no sequence at all
    assert A.packed_attention(q[:0], k[:0], v[:0], ints([0, 0])).shape == (0, 4, 64)


def test_packed_layouts_that_need_a_copy():
    """A transposed and an unaligned operand give what their contiguous copies give."""
    g = torch.Generator(device=DEV).manual_seed(3)
    q, k, v = randn(g, 100, 4, 64, dtype=FP), randn(g, 100, 4, 64, dtype=FP), randn(g, 100, 4, 64, dtype=FP)
    cu = ints([0, 37, 100])
    want = A.packed_attention(q, k, v, cu)
    qt = q.transpose(1, 2).contiguous().transpose(1, 2)
    flat = torch.empty(k.numel() + 1, dtype=FP, device=DEV)
    ku = flat[1:].view(k.shape)
    ku.copy_(k)
    vh = v.transpose(0, 1).contiguous().transpose(0, 1)  # [heads, tokens, d] seen as [tokens, heads, d]: taken as it lies
    assert torch.equal(A.packed_attention(qt, ku, vh, cu), want)


def test_packed_large_scores():
    """Scores of some hundreds: one key takes all, in the first tile, in the last and past a divided range."""
    n, d = 700, 64
    g = torch.Generator(device=DEV).manual_seed(4)
    q = torch.ones(n, 1, d, dtype=BF, device=DEV)
    k = randn(g, n, 1, d, dtype=BF) * 0.125
    v = randn(g, n, 1, d, dtype=BF)
    for at, value in ((0, 30.0), (333, 40.0), (699, 90.0)):
        k[at] = value
    got = A.packed_attention(q, k, v, ints([0, n]))
    want, bound = reference(q, k, v, 0, d ** -0.5)
    check(got, want, bound, "large scores")


PAGED = [
    # lens, chunks, page, hq, hk, d, dtype
    ([1], [1], 16, 1, 1, 128, BF),
    ([161], [1], 16, 16, 16, 128, BF),
    ([5, 300, 64, 33], [1, 1, 1, 1], 8, 8, 2, 64, FP),
    ([900, 130, 77, 9], [9, 9, 9, 9], 64, 16, 4, 128, BF),
    ([400, 90, 700], [129, 90, 3], 32, 4, 1, 96, BF),
    ([129, 40, 260], [40, 0, 200], 7, 6, 2, 80, FP),
    ([50, 257, 31], [1, 33, 31], 1, 5, 1, 40, BF),
    ([600, 300], [5, 80], 128, 4, 2, 256, BF),
    ([333, 1024], [1, 1], 256, 8, 1, 256, FP),
    ([5000, 17], [1, 1], 16, 4, 1, 128, BF),  # divided
    ([3000, 2600], [200, 7], 16, 2, 2, 64, BF),
    ([2049], [2], 16, 1, 1, 256, FP),
    ([4, 0, 2], [4, 0, 2], 16, 2, 1, 64, BF),
    ([40 + i for i in range(130)], [1 + i % 3 for i in range(130)], 16, 2, 1, 64, FP),
    ([600 + i for i in range(70)], [1 + 40 * (i % 2) for i in range(70)], 16, 2, 1, 64, BF),  # divided, more than 64 sequences
    ([300, 77, 129], [1, 70, 129], 2, 3, 1, 128, BF),  # pages smaller than a load instruction's rows, and than a block's share
    ([300, 77, 700], [1, 70, 65], 5, 4, 2, 256, BF),
    ([260, 900], [3, 40], 3, 160, 1, 64, FP),
    ([4000, 3900, 10], [1, 1, 1], 12, 4, 1, 72, BF),
    ([6000], [150], 16, 1, 1, 64, BF),  # large tiles of many parts
]


def paged_state(lens, page, hk, d, dtype, g, spare=3, pool=None):
    """A pool whose unused places hold NaN, a table whose unused entries are far out of range, and the sequences' rows."""
    need = [-(-n // page) for n in lens]
    pool = pool or sum(need) + spare
    order = torch.randperm(pool, generator=g, device=DEV)[:sum(need)].to(torch.int32)
    table = torch.full((len(lens), max(need) + 1), 2 ** 31 - 1, dtype=torch.int32, device=DEV)
    kp = torch.full((pool, page, hk, d), math.nan, dtype=dtype, device=DEV)
    vp = torch.full((pool, page, hk, d), math.nan, dtype=dtype, device=DEV)
    ks, vs, used = [], [], 0
    for b, n in enumerate(lens):
        ids = order[used:used + need[b]]
        used += need[b]
        table[b, :need[b]] = ids
        ks.append(randn(g, n, hk, d, dtype=dtype))
        vs.append(randn(g, n, hk, d, dtype=dtype))
        at = torch.arange(n, device=DEV)
        where = (ids.long()[at // page], at % page)
        kp[where], vp[where] = ks[-1], vs[-1]
    return kp, vp, table, ks, vs


@pytest.mark.parametrize("lens,chunks,page,hq,hk,d,dtype", PAGED)
def test_paged(lens, chunks, page, hq, hk, d, dtype):
    print(f"\n[paged] {lens[:6]} {chunks[:6]} page {page} {hq}/{hk} x {d} {dtype}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(5)
    kp, vp, table, ks, vs = paged_state(lens, page, hk, d, dtype, g)
    off = offsets(chunks)
    q = randn(g, off[-1] + 2, hq, d, dtype=dtype) * 1.5
    got = A.paged_attention(q, kp, vp, table, ints(lens), ints(off))
    for b, (a, z) in enumerate(zip(off, off[1:])):
        want, bound = reference(q[a:z], ks[b], vs[b], lens[b] - chunks[b], d ** -0.5)
        check(got[a:z], want, bound, f"sequence {b}")
    assert not got[off[-1]:].any()


def test_paged_rows_that_see_nothing():
    """A length below the chunk's leaves the first rows without a key; a length of 0 all of them: zeros."""
    g = torch.Generator(device=DEV).manual_seed(6)
    kp, vp, table, ks, vs = paged_state([3, 300], 16, 1, 64, BF, g)
    q = randn(g, 8 + 4 + 300, 2, 64, dtype=BF)
    got = A.paged_attention(q, kp, vp, table, ints([3, 0]), ints([0, 8, 12]))
    assert not got[:5].any() and not got[8:].any()
    want, bound = reference(q[5:8], ks[0], vs[0], 0, 64 ** -0.5)
    check(got[5:8], want, bound, "the rows with keys")
    got = A.paged_attention(q, kp, vp, table, ints([-5, 100]), ints([0, 12, 312]))  # 300 rows, 100 positions
    assert not got[:212].any()
    want, bound = reference(q[212:], ks[1][:100], vs[1][:100], 0, 64 ** -0.5)
    check(got[212:], want, bound, "the last 100")


@pytest.mark.parametrize("n,chunk", [(100, 1), (100, 90), (3000, 1), (3000, 90)])
def test_paged_bad_pages_give_nan_rows(n, chunk):
    """Ids outside the pool below a sequence's length (its own rows become NaN); the other sequences are not touched."""
    print(f"\n[bad pages] {n} {chunk}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(7)
    lens, chunks = [n, 200, n], [chunk, 3, chunk]
    kp, vp, table, ks, vs = paged_state(lens, 16, 1, 64, BF, g)
    table[0, 2], table[2, (n - 1) // 16] = -1, kp.shape[0]
    off = offsets(chunks)
    q = randn(g, off[-1], 1, 64, dtype=BF)
    got = A.paged_attention(q, kp, vp, table, ints(lens), ints(off))
    # every row that sees the bad page; a row that stops before it may be NaN with its tile
    assert got[:chunk][-1].isnan().all() and got[off[2]:][-1].isnan().all()
    want, bound = reference(q[off[1]:off[2]], ks[1], vs[1], 197, 64 ** -0.5)
    check(got[off[1]:off[2]], want, bound, "the good sequence")


def test_lengths_past_the_table_and_offsets_past_the_tokens_are_cut():
    g = torch.Generator(device=DEV).manual_seed(8)
    kp, vp, table, ks, vs = paged_state([64, 64], 16, 1, 64, BF, g)
    table = table[:, :4].contiguous()
    q = randn(g, 6, 1, 64, dtype=BF)
    got = A.paged_attention(q, kp, vp, table, ints([1000, 64]), ints([0, 3, 900]))
    for b, a in ((0, 0), (1, 3)):
        want, bound = reference(q[a:a + 3], ks[b], vs[b], 61, 64 ** -0.5)
        check(got[a:a + 3], want, bound, f"sequence {b}")


def test_pages_past_32_bit_offsets():
    """Pages whose element offset passes 2^32 (a pool of 4.4e9 elements), read and appended to."""
    page, hk, d, n = 16, 8, 128, 50
    pool = (2 ** 32 + 2 ** 27) // (page * hk * d)
    g = torch.Generator(device=DEV).manual_seed(9)
    kp = torch.empty(pool, page, hk, d, dtype=BF, device=DEV)
    vp = torch.empty(pool, page, hk, d, dtype=BF, device=DEV)
    table = ints([[pool - 1, 5, pool - 3, pool // 2 + 1]])
    k, v = randn(g, n, hk, d, dtype=BF), randn(g, n, hk, d, dtype=BF)
    A.paged_append(k, v, kp, vp, table, ints([n]), ints([0, n]))
    at = torch.arange(n, device=DEV)
    where = (table[0].long()[at // page], at % page)
    assert torch.equal(kp[where], k) and torch.equal(vp[where], v)
    q = randn(g, 2, hk, d, dtype=BF)
    got = A.paged_attention(q, kp, vp, table, ints([n]), ints([0, 2]))
    want, bound = reference(q, k, v, n - 2, d ** -0.5)
    check(got, want, bound, "far pages")


def test_cache_strides():
    """Keys and values in one pool [pages, 2, heads, positions, d]: any strides between pages, positions and heads."""
    g = torch.Generator(device=DEV).manual_seed(10)
    lens, chunks, page, hk, d = [300, 20], [70, 1], 16, 2, 64
    kp, vp, table, ks, vs = paged_state(lens, page, hk, d, BF, g)
    both = torch.stack([kp, vp], 1).transpose(2, 3).contiguous()  # [pool, 2, hk, page, d]
    kq, vq = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    q = randn(g, 71, 4, d, dtype=BF)
    args = (table, ints(lens), ints(offsets(chunks)))
    assert torch.equal(A.paged_attention(q, kq, vq, *args), A.paged_attention(q, kp, vp, *args))
    k, v = randn(g, 71, hk, d, dtype=BF), randn(g, 71, hk, d, dtype=BF)
    A.paged_append(k, v, kq, vq, *args)
    A.paged_append(k, v, kp, vp, *args)
    assert torch.equal(kq.nan_to_num(7.0), kp.nan_to_num(7.0)) and torch.equal(vq.nan_to_num(7.0), vp.nan_to_num(7.0))


@pytest.mark.parametrize("dtype,d", [(BF, 128), (torch.float32, 20), (torch.int8, 24), (torch.uint8, 32), (FP, 7)])
def test_append(dtype, d):
    """Chunks to the last positions, nothing else changed; bad pages, positions past the table and rows of no chunk are left
    out. Rows of whole 16 bytes and others."""
    print(f"\n[append] {dtype} {d}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(11)
    page, hk, pool = 4, 3, 40
    lens, chunks = [9, 30, 3, 12, 2], [1, 30, 5, 0, 2]
    off = [1 + x for x in offsets(chunks)]  # token 0 and the last two belong to no chunk
    make = lambda *s: (torch.randn(*s, generator=g, device=DEV) * 30).to(dtype)  # noqa: E731
    k, v = make(off[-1] + 2, hk, d), make(off[-1] + 2, hk, d)
    kp, vp = make(pool, page, hk, d), make(pool, page, hk, d)
    table = torch.randperm(pool, generator=g, device=DEV)[:5 * 7].view(5, 7).to(torch.int32)
    table[1, 2], table[4, 0] = -1, pool
    want = [kp.clone(), vp.clone()]
    host = table.tolist()
    for b, n in enumerate(lens):
        for i in range(chunks[b]):
            pos = n - chunks[b] + i
            if 0 <= pos < 7 * page and 0 <= host[b][pos // page] < pool:
                want[0][host[b][pos // page], pos % page] = k[off[b] + i]
                want[1][host[b][pos // page], pos % page] = v[off[b] + i]
    A.paged_append(k, v, kp, vp, table, ints(lens), ints(off))
    assert torch.equal(kp, want[0]) and torch.equal(vp, want[1])


def test_append_of_slices():
    """k and v as slices of one projection."""
    g = torch.Generator(device=DEV).manual_seed(12)
    qkv = randn(g, 20, 6, 64, dtype=BF)
    kp, vp = torch.zeros(4, 16, 1, 64, dtype=BF, device=DEV), torch.zeros(4, 16, 1, 64, dtype=BF, device=DEV)
    A.paged_append(qkv[:, 4:5], qkv[:, 5:], kp, vp, ints([[2, 0]]), ints([20]), ints([0, 20]))
    assert torch.equal(kp[2], qkv[:16, 4:5]) and torch.equal(vp[0, :4], qkv[16:, 5:]) and not kp[0, 4:].any()


def test_graph_replays_follow_the_lengths():
    """Append and attention captured once; at every replay the lengths, the offsets, the table and the inputs are others."""
    g = torch.Generator(device=DEV).manual_seed(13)
    page, hk, hq, d = 16, 2, 4, 64
    kp, vp, table, _, _ = paged_state([1200, 900], page, hk, d, BF, g)
    kp.nan_to_num_(0.0), vp.nan_to_num_(0.0)
    tokens = 100
    q, k, v = randn(g, tokens, hq, d, dtype=BF), randn(g, tokens, hk, d, dtype=BF), randn(g, tokens, hk, d, dtype=BF)
    lengths, cu = ints([1200, 900]), ints([0, 90, 100])
    out = torch.empty(tokens, hq, d, dtype=BF, device=DEV)

    def step():
        A.paged_append(k, v, kp, vp, table, lengths, cu)
        A.paged_attention(q, kp, vp, table, lengths, cu, out=out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for lens, off in (([1200, 900], [0, 90, 100]), ([33, 70], [0, 33, 99]), ([1, 850], [0, 1, 2]), ([500, 0], [0, 100, 100])):
        q.copy_(randn(g, tokens, hq, d, dtype=BF))
        k.copy_(randn(g, tokens, hk, d, dtype=BF))
        lengths.copy_(ints(lens))
        cu.copy_(ints(off))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        step()
        torch.cuda.synchronize()
        assert torch.equal(got, out)


def test_another_stream_and_two_calls_alike():
    g = torch.Generator(device=DEV).manual_seed(14)
    q, k, v = (randn(g, 1500, 2, 128, dtype=BF) for _ in range(3))
    cu = ints([0, 1000, 1500])
    want = A.packed_attention(q, k, v, cu)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = A.packed_attention(q, k, v, cu)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    assert torch.equal(A.packed_attention(q, k, v, cu), want)


def test_gpu_refusals():
    q, kp = torch.zeros(4, 2, 64, dtype=BF, device=DEV), torch.zeros(3, 16, 1, 64, dtype=BF, device=DEV)
    table, lens, cu = ints([[0, 1]]), ints([4]), ints([0, 4])
    with pytest.raises(ValueError, match="all tensors must be on"):
        A.paged_attention(q, kp, kp, table, lens.cpu(), cu)
    with pytest.raises(ValueError, match="no backward"):
        A.packed_attention(q.clone().requires_grad_(), q, q, cu)
    with torch.no_grad():
        A.packed_attention(q.clone().requires_grad_(), q, q, cu)
    with pytest.raises(ValueError, match="16-byte aligned"):
        odd = torch.zeros(3 * 16 * 64 + 1, dtype=BF, device=DEV)[1:].view(3, 16, 1, 64)
        A.paged_attention(q, odd, kp, table, lens, cu)
    with pytest.raises(ValueError, match="out must be"):
        A.packed_attention(q, q, q, cu, out=torch.zeros(4, 2, 64, dtype=FP, device=DEV))


@pytest.mark.parametrize("counts,lens,hq,hk,d,dtype", [
    ([100, 1000], None, 200, 1, 64, BF),
    ([0, 700, 3], None, 160, 1, 96, FP),
    ([30, 500], None, 387, 3, 256, BF),
    ([0, 40, 500], [0, 900, 500], 400, 2, 64, BF),
    ([3, 600, 2], [3, 600, 200], 129, 1, 128, FP),
])
def test_more_query_heads_than_a_tile_has_rows_in_order(counts, lens, hq, hk, d, dtype):
    """More than 128 query heads to a key head and more tiles than the card holds at once, the long sequence not the first."""
    print(f"\n[heads] {counts} {lens} {hq}/{hk} x {d} {dtype}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(30)
    off = offsets(counts)
    q = randn(g, off[-1], hq, d, dtype=dtype)
    out = torch.full_like(q, math.nan)
    if lens is None:
        k, v = randn(g, off[-1], hk, d, dtype=dtype), randn(g, off[-1], hk, d, dtype=dtype)
        A.packed_attention(q, k, v, ints(off), out=out)
        ks, vs, firsts = [k[a:z] for a, z in zip(off, off[1:])], [v[a:z] for a, z in zip(off, off[1:])], [0] * len(counts)
    else:
        kp, vp, table, ks, vs = paged_state(lens, 16, hk, d, dtype, g)
        A.paged_attention(q, kp, vp, table, ints(lens), ints(off), out=out)
        firsts = [n - c for n, c in zip(lens, counts)]
    for b, (a, z) in enumerate(zip(off, off[1:])):
        want, bound = reference(q[a:z], ks[b], vs[b], firsts[b], d ** -0.5)
        check(out[a:z], want, bound, f"sequence {b}")


def one_hot_reference(q, k, v, first, scale, dtype):
    """(out, bound) in float64 where every score and every difference of scores is exact in float32 and each row's probabilities
    are 0 or shares of 1 (or ordinary scores of a few units): what is left is the rounding of the probabilities and of the
    result, and a few float32 steps."""
    h = torch.finfo(dtype).eps / 2
    s = q[:, 0].double().cpu() @ k[:, 0].double().cpu().T * scale
    seen = torch.arange(len(k))[None, :] <= first + torch.arange(len(q))[:, None]
    s = torch.where(seen, s, -math.inf)
    p = torch.softmax(s, -1)
    v = v[:, 0].double().cpu()
    o, a = p @ v, p @ v.abs()
    tiny = 2.0 ** -25 if dtype == FP else 0.0
    return o, h * o.abs() * 1.01 + (h * 1.01 + 2.0 ** -18) * a + tiny * (seen.double() @ v.abs())


FAR = [(BF, 2.0 ** 12, 2.0 ** 12, 1.0), (BF, 2.0 ** 15, 2.0 ** 15, 1.0), (BF, 2.0 ** 16, 2.0 ** 16, None), (BF, 2.0 ** 17, 2.0 ** 17, 0.75),
       (BF, 2.0 ** 50, 2.0 ** 50, 1.0), (BF, 2.0 ** 63, 2.0 ** 63, 1.5), (BF, 2.0 ** 63, 2.0 ** 63, 16.0),
       (FP, 2.0 ** 13, 2.0 ** 13, 1.0), (FP, 2.0 ** 14, 2.0 ** 14, 1.0), (FP, 2.0 ** 15, 2.0 ** 15, 1.0), (FP, 2.0 ** 15, 2.0 ** 15, 4.0),
       (FP, 2.0 ** 15, 2.0 ** 14, 64.0)]


@pytest.mark.parametrize("dtype,a,b,scale", FAR)
def test_scores_far_from_zero(dtype, a, b, scale):
    """Finite scores from 2^24 up to float32's range and past it with the scale, positive and negative, tied, beside rows of
    ordinary scores: large tiles, whole and divided, and small ones."""
    print(f"\n[far] {dtype} {a} {b} {scale}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(40)
    d = 64
    for n, rows, hq in ((160, 160, 1), (1500, 1500, 1), (5000, 1, 1), (900, 9, 4), (33, 2, 1)):
        k = torch.zeros(n, 1, d, device=DEV)
        k[:, 0, 5] = b * (1.0 + torch.randint(0, 128, (n,), generator=g, device=DEV) / 128.0)
        q = torch.zeros(rows, hq, d, device=DEV)
        kind = torch.randint(0, 4, (rows, hq), generator=g, device=DEV)
        q[..., 5] = torch.tensor([a, -a, 2.0 / b, 0.0], device=DEV)[kind]  # the third: ordinary scores of 2 scale to 4 scale
        if dtype == FP:
            q[..., 5] = torch.where(kind == 2, 0.0, q[..., 5])
        v = torch.randn(n, 1, d, generator=g, device=DEV)
        q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)
        s = d ** -0.5 if scale is None else scale
        if rows == n:
            got = A.packed_attention(q, k, v, ints([0, n]), scale=scale)
        else:
            order = torch.randperm(-(-n // 16) + 2, generator=g, device=DEV)[:-(-n // 16)].to(torch.int32)
            kp, vp = (torch.zeros(len(order) + 2, 16, 1, d, dtype=dtype, device=DEV) for _ in range(2))
            at = torch.arange(n, device=DEV)
            kp[order.long()[at // 16], at % 16], vp[order.long()[at // 16], at % 16] = k, v
            got = A.paged_attention(q, kp, vp, order[None], ints([n]), ints([0, rows]), scale=scale)
        for h in range(hq):
            want, bound = one_hot_reference(q[:, h:h + 1], k, v, n - rows, s, dtype)
            check(got[:, h], want, bound, f"{n} keys, {rows} rows, head {h}")


def test_append_and_attention_agree_on_offsets_past_the_tokens():
    """Offsets before the first token and past the last: both take the tokens that there are, at the same positions."""
    g = torch.Generator(device=DEV).manual_seed(41)
    tokens, page, d = 6, 16, 64
    table, lengths, cu = ints([[3, 0], [1, 4]]), ints([20, 30]), ints([-2, 3, 900])
    k, v, q = (randn(g, tokens, 1, d, dtype=BF) for _ in range(3))
    old = [randn(g, 30, 1, d, dtype=BF) for _ in range(4)]  # keys, values of either sequence
    kp, vp = (torch.zeros(5, page, 1, d, dtype=BF, device=DEV) for _ in range(2))
    for b, n in enumerate((17, 27)):
        at = torch.arange(n, device=DEV)
        where = (table[b].long()[at // page], at % page)
        kp[where], vp[where] = old[2 * b][:n], old[2 * b + 1][:n]
    A.paged_append(k, v, kp, vp, table, lengths, cu)
    got = A.paged_attention(q, kp, vp, table, lengths, cu)
    for b, (n, a) in enumerate(((17, 0), (27, 3))):
        ks, vs = torch.cat([old[2 * b][:n], k[a:a + 3]]), torch.cat([old[2 * b + 1][:n], v[a:a + 3]])
        want, bound = reference(q[a:a + 3], ks, vs, n, d ** -0.5)
        check(got[a:a + 3], want, bound, f"sequence {b}")


def test_strides_of_dimensions_of_one_entry_do_not_count():
    """One token or one head in a wider buffer whose rows are no multiple of 8: the same as from a tensor of its own."""
    g = torch.Generator(device=DEV).manual_seed(42)
    wide = randn(g, 1, 1, 67, dtype=BF)
    q, k, v = wide[..., :64], randn(g, 1, 1, 65, dtype=BF)[..., :64], randn(g, 1, 1, 71, dtype=BF)[..., :64]
    assert q.stride()[0] % 8 and q.is_contiguous()
    own = [t.clone(memory_format=torch.contiguous_format).view(1, 1, 64) for t in (q, k, v)]
    assert torch.equal(A.packed_attention(q, k, v, ints([0, 1])), A.packed_attention(*own, ints([0, 1])))
    q3, k3 = randn(g, 3, 1, 64, dtype=BF), randn(g, 3, 1, 64, dtype=BF)  # many tokens, one head with any stride
    odd = lambda t: t.as_strided(t.shape, (64, 13, 1))  # noqa: E731
    assert torch.equal(A.packed_attention(odd(q3), odd(k3), odd(k3), ints([0, 3])), A.packed_attention(q3, k3, k3, ints([0, 3])))

    pool = randn(g, 16, 64, dtype=BF)  # one page of 16 positions, one head; then 16 pages of one position
    table, lengths, cu = ints([[0]]), ints([11]), ints([0, 1])
    plain = pool.view(1, 16, 1, 64)
    page = pool.as_strided((1, 16, 1, 64), (17, 64, 3, 1))
    want = A.paged_attention(q, plain, plain, table, lengths, cu)
    assert torch.equal(A.paged_attention(q, page, page, table, lengths, cu), want)
    single = pool.as_strided((16, 1, 1, 64), (64, 5, 3, 1))
    table = torch.arange(16, dtype=torch.int32, device=DEV)[None]
    assert torch.equal(A.paged_attention(q, single, single, table, lengths, cu), want)
    with pytest.raises(ValueError, match="multiples of 8"):
        two = randn(g, 40, 64, dtype=BF).as_strided((2, 16, 1, 64), (65 * 16 + 1, 64, 64, 1))
        A.paged_attention(q, two, two, ints([[0]]), lengths, cu)


def test_tangents_are_refused():
    """A dual tensor of forward-mode differentiation, whose tangent a launch would drop; its primal and other tensors run."""
    from torch.autograd import forward_ad

    from byteprof_amd.optim.logprobs import token_logprobs

    g = torch.Generator(device=DEV).manual_seed(43)
    q, t = randn(g, 4, 1, 64, dtype=BF), randn(g, 4, 1, 64, dtype=BF)
    pages, table, lens, cu = torch.zeros(1, 16, 1, 64, dtype=BF, device=DEV), ints([[0]]), ints([4]), ints([0, 4])
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(q, t)
        for call in (lambda x: A.packed_attention(x, q, q, cu), lambda x: A.packed_attention(q, q, x, cu),
                     lambda x: A.paged_attention(x, pages, pages, table, lens, cu),
                     lambda x: A.paged_append(q, x, pages, pages, table, lens, cu), lambda x: token_logprobs(x[:, 0])):
            with pytest.raises(ValueError, match="forward-mode"):
                call(dual)
            with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
                call(dual)
            call(q)
            call(forward_ad.unpack_dual(dual).primal)


def test_written_tensors_count_as_changed():
    """The caches of an append and the output of an attention, saved by another graph before: its backward pass refuses."""
    g = torch.Generator(device=DEV).manual_seed(44)
    q = randn(g, 4, 1, 64, dtype=BF)
    kp, vp = torch.zeros(1, 16, 1, 64, dtype=BF, device=DEV), torch.zeros(1, 16, 1, 64, dtype=BF, device=DEV)
    out, w = torch.zeros_like(q), torch.ones(1, device=DEV, requires_grad=True)
    table, lens, cu = ints([[0]]), ints([4]), ints([0, 4])
    for saved, call in ((kp, lambda: A.paged_append(q, q, kp, vp, table, lens, cu)), (vp, lambda: A.paged_append(q, q, kp, vp, table, lens, cu)),
                        (out, lambda: A.packed_attention(q, q, q, cu, out=out)),
                        (out, lambda: A.paged_attention(q, kp, vp, table, lens, cu, out=out))):
        loss = (saved * w).sum()
        call()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    with torch.inference_mode():
        pages = torch.zeros(1, 16, 1, 64, dtype=BF, device=DEV)  # has no version
        A.paged_append(q, q, pages, pages.clone(), table, lens, cu)
        A.packed_attention(q, q, q, cu, out=torch.empty_like(q))


def test_in_place():
    """out = q, in whole and divided tiles, small and large, with rows of no sequence."""
    g = torch.Generator(device=DEV).manual_seed(45)
    q, k, v = randn(g, 1600, 4, 64, dtype=BF), randn(g, 1600, 1, 64, dtype=BF), randn(g, 1600, 1, 64, dtype=BF)
    for cu in ([0, 1500], [0, 10, 13, 333, 1400], [3, 14]):
        x = q.clone()
        want = A.packed_attention(x, k, v, ints(cu))
        assert A.packed_attention(x, k, v, ints(cu), out=x) is x and torch.equal(x, want)
    with pytest.raises(ValueError, match="overlap"):
        A.packed_attention(k, k, v, ints([0, 1600]), out=v)
