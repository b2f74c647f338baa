"""rotary against the rotation in float64 (angles in float64: position x frequency up to 2^62 is exact to 2^-52 of itself).

The bound of an element, with h half a step of the output's type (relative) and A = |factor| (|x1| + |x2|): the result is rounded
once (h |y|); the angle, reduced in 64 bits, is rounded to float32 in half turns (at most 1, so 2^-24 of it, times pi), sine and
cosine to a few steps, factor, products and sum once each: 2^-21 A in all. fp16 results below its least normal value are rounded to
multiples of 2^-24. A position past 2^20 adds what 64 bits lose: position x frequency x 2^-51."""

from __future__ import annotations

import math

import pytest
import torch

from byteprof_amd.optim.rotary import rotary, rotary_frequencies

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def reference(x, positions, inv_freq, interleaved, factor):
    """(result, bound) in float64 on the CPU."""
    h = torch.finfo(x.dtype).eps / 2
    tiny = {BF: 2.0 ** -134, FP: 2.0 ** -25, F32: 2.0 ** -150}[x.dtype]
    x, pos, f = x.double().cpu(), positions.double().cpu(), inv_freq.double().cpu()
    rot = 2 * len(f)
    angle = (pos[:, None] * f)[:, None]
    c, s = angle.cos() * factor, angle.sin() * factor
    out, bound = x.clone(), torch.zeros_like(x)
    a, b = (x[..., :rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    y1, y2 = a * c - b * s, b * c + a * s
    big = abs(factor) * (a.abs() + b.abs()) * (2.0 ** -21 + angle.abs() * 2.0 ** -51)
    for y, at in ((y1, 0), (y2, 1)):
        where = slice(at, rot, 2) if interleaved else slice(at * rot // 2, (at + 1) * rot // 2)
        out[..., where] = y
        bound[..., where] = h * 1.01 * (y.abs() + big) + big + tiny
    return out, bound


def check(got, want, bound, what):
    worst = ((got.double().cpu() - want).abs() - bound).max().item() if got.numel() else 0.0
    assert worst <= 0.0, f"{what}: {worst} past the bound"


CASES = [
    # tokens, hq, hk, d, rot, interleaved, dtype, far, fused
    (1, 16, 16, 128, 128, False, BF, 4000, True),
    (1, 1, 0, 64, 64, True, FP, 10, False),
    (777, 8, 2, 128, 128, False, BF, 1 << 20, True),
    (300, 12, 4, 80, 32, True, FP, 1 << 24, True),
    (5000, 4, 1, 64, 64, False, FP, 1 << 17, False),
    (257, 5, 1, 40, 40, False, BF, 5000, True),  # halves of 20: no whole vectors
    (100, 3, 3, 96, 2, True, F32, 1 << 30, True),
    (64, 2, 1, 72, 24, False, F32, 100000, False),
    (33, 7, 1, 256, 256, True, BF, 300, True),
    (10, 2, 2, 1024, 1024, False, BF, 300, False),
    (2000, 1, 1, 8, 8, True, BF, 1 << 40, True),
    (50, 2, 1, 7, 6, False, FP, 99, True),  # odd heads
    (9, 4, 2, 64, 0, False, BF, 99, True),  # nothing turns
]


@pytest.mark.parametrize("tokens,hq,hk,d,rot,interleaved,dtype,far,fused", CASES)
def test_rotary(tokens, hq, hk, d, rot, interleaved, dtype, far, fused):
    print(f"\n[rotary] {tokens} {hq}/{hk} x {d} rot {rot} {interleaved} {dtype}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(1)
    if fused:
        qkv = torch.randn(tokens, hq + 2 * hk, d, generator=g, device=DEV).to(dtype)
        q, k = qkv[:, :hq], qkv[:, hq:hq + hk]
    else:
        q, k = (torch.randn(tokens, n, d, generator=g, device=DEV).to(dtype) for n in (hq, hk))
    k = k if hk else None
    positions = torch.randint(0, far, (tokens,), generator=g, device=DEV)
    positions[0] = -7
    inv_freq = rotary_frequencies(rot, device=DEV)[0] if rot else torch.zeros(0, device=DEV)
    keep = q.clone()
    outs = rotary(q, k, positions, inv_freq, interleaved=interleaved, factor=1.25)
    assert torch.equal(q, keep) and (outs[1] is None) == (k is None)
    for x, y in zip((q, k), outs):
        if x is not None:
            assert y.shape == x.shape and y.dtype == dtype and y.is_contiguous()
            want, bound = reference(x, positions, inv_freq, interleaved, 1.25)
            check(y, want, bound, "q or k")
            assert torch.equal(y[..., rot:], x[..., rot:])
    # in place, in a projection whose other columns and rows stay
    if fused:
        rest = qkv[:, hq + hk:].clone()
        got = rotary(q, k, positions, inv_freq, interleaved=interleaved, factor=1.25, out=(q, k))
        assert got[0] is q and got[1] is k
        assert torch.equal(q, outs[0]) and (k is None or torch.equal(k, outs[1])) and torch.equal(qkv[:, hq + hk:], rest)


def test_layouts():
    """int32 positions, a head-major input, an output with strides, positions and frequencies with strides: the same bits."""
    g = torch.Generator(device=DEV).manual_seed(2)
    q, k = torch.randn(60, 4, 64, generator=g, device=DEV).to(BF), torch.randn(60, 2, 64, generator=g, device=DEV).to(BF)
    positions, (inv, _) = torch.randint(0, 9999, (60,), generator=g, device=DEV), rotary_frequencies(64, device=DEV)
    want = rotary(q, k, positions, inv)
    qh = q.transpose(0, 1).contiguous().transpose(0, 1)
    out = (torch.empty(4, 60, 64, dtype=BF, device=DEV).transpose(0, 1), torch.empty(60, 3, 80, dtype=BF, device=DEV)[:, :2, :64])
    got = rotary(qh, k, positions.to(torch.int32), inv, out=out)
    assert got[0] is out[0] and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    wide = positions.repeat_interleave(2)[::2]
    assert torch.equal(rotary(q, k, wide, inv.repeat_interleave(3)[::3])[0], want[0])
    odd = torch.empty(60 * 4 * 64 + 1, dtype=BF, device=DEV)[1:].view(60, 4, 64)
    odd.copy_(q)
    assert torch.equal(rotary(odd, k, positions, inv)[0], want[0])
    assert rotary(q[:0], k[:0], positions[:0], inv)[0].shape == (0, 4, 64)
    one = torch.randn(1, 1, 67, generator=g, device=DEV).to(BF)[..., :64]  # strides of dimensions of one entry do not count
    alone = rotary(one.contiguous().clone(), None, positions[:1], inv)[0]
    assert torch.equal(rotary(one, None, positions[:1], inv, out=(one, None))[0], alone)


def test_turned_back():
    """The angle of the opposite position undoes the rotation, to the roundings of two results (fp32)."""
    g = torch.Generator(device=DEV).manual_seed(3)
    q = torch.randn(500, 3, 128, generator=g, device=DEV)
    positions = torch.randint(0, 1 << 22, (500,), generator=g, device=DEV)
    inv, _ = rotary_frequencies(128, device=DEV)
    there, _ = rotary(q, None, positions, inv)
    back, _ = rotary(there, None, -positions, inv)
    big = q[..., :64].abs() + q[..., 64:].abs()
    assert ((back - q).abs() <= 2.0 ** -20 * 2 * torch.cat([big, big], -1)).all()


def test_far_tensor_and_other_streams():
    """A tensor whose element offsets pass 2^31, on another stream; a captured graph follows its positions."""
    g = torch.Generator(device=DEV).manual_seed(4)
    big = torch.empty(1 << 16, 2, (1 << 14) + 8, dtype=BF, device=DEV)[..., :128]
    some = torch.tensor([0, 1, 40000, (1 << 16) - 1], device=DEV)
    big[some] = torch.randn(4, 2, 128, generator=g, device=DEV).to(BF)
    keep = big[some].clone()
    positions = torch.arange(1 << 16, device=DEV)
    inv, _ = rotary_frequencies(128, device=DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        rotary(big, None, positions, inv, out=(big, None))
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(big[some], rotary(keep, None, some, inv)[0])
    del big
    q, k, pos = keep[:3].clone(), keep[1:].clone(), torch.tensor([5, 6, 7], device=DEV)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = rotary(q, k, pos, inv)
    for n in range(3):
        pos.add_(n * 1000)
        q.copy_(torch.randn(3, 2, 128, generator=g, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(outs, rotary(q, k, pos, inv)):
            assert torch.equal(x, y)


def test_what_it_refuses_on_the_gpu():
    q, k = torch.zeros(4, 2, 64, device=DEV), torch.zeros(4, 1, 64, device=DEV)
    pos, (inv, _) = torch.arange(4, device=DEV), rotary_frequencies(64, device=DEV)
    with pytest.raises(ValueError, match="no backward"):
        rotary(q.clone().requires_grad_(), k, pos, inv)
    with torch.no_grad():
        rotary(q.clone().requires_grad_(), k, pos, inv)
    with pytest.raises(ValueError, match="all tensors must be on"):
        rotary(q, k, pos.cpu(), inv)
    with pytest.raises(ValueError, match="apart from everything"):
        rotary(q, k, pos, inv, out=(torch.zeros_like(q), q[:, 1:]))
    both = torch.zeros(8, 2, 64, device=DEV)
    with pytest.raises(ValueError, match="apart from everything"):
        rotary(both[:4], k, pos, inv, out=(both[2:6], torch.zeros_like(k)))
    n = q._version
    rotary(q, k, pos, inv, out=(q, k))
    assert q._version > n
    from torch.autograd import forward_ad
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="forward-mode"):
            rotary(q, forward_ad.make_dual(k, k), pos, inv)
