"""What the operators of the 8-bit cache and rotary refuse, at their Python names and at their C entries, and the frequencies of
rotary_frequencies. CPU only: every call here returns or raises before anything is enqueued."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from byteprof_amd.optim import attention as A
from byteprof_amd.optim import rotary as R
from byteprof_amd.optim.rotary import rotary, rotary_frequencies

BF, FP = torch.bfloat16, torch.float16
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
CU = torch.tensor([0, 4], dtype=torch.int32)


def z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


@pytest.fixture(scope="module")
def L():
    from byteprof_amd import _lib

    return _lib.lib()


def cache(**kw):
    args = {"k_pages": z(3, 16, 1, 64, dtype=E4M3), "v_pages": z(3, 16, 1, 64, dtype=E4M3),
            "table": torch.zeros(1, 2, dtype=torch.int32), "lengths": torch.tensor([4], dtype=torch.int32), "cu": CU,
            "k_scales": z(3, 2, 1, dtype=E8M0), "v_scales": z(3, 2, 1, dtype=E8M0)}
    args.update(kw)
    return args


BAD_CACHE = [
    ({"k_scales": None}, "8 bits"),
    ({"v_scales": None}, "8 bits"),
    ({"k_pages": z(3, 16, 1, 64), "v_pages": z(3, 16, 1, 64)}, "8 bits"),
    ({"v_pages": z(3, 16, 1, 64, dtype=torch.int8)}, "8 bits"),
    ({"k_pages": z(3, 16, 1, 64, dtype=torch.uint8), "v_pages": z(3, 16, 1, 64, dtype=torch.uint8)}, "8 bits"),
    ({"k_scales": z(3, 2, 1, dtype=torch.float32)}, "scales must be"),
    ({"k_scales": z(3, 2, 1, dtype=torch.uint8)}, "scales must be"),
    ({"v_scales": z(3, 4, 1, dtype=E8M0)}, "scales must be"),
    ({"k_scales": z(3, 3, 1, dtype=E8M0), "v_scales": z(3, 3, 1, dtype=E8M0)}, "scales must be"),
    ({"k_scales": z(3, 0, 1, dtype=E8M0), "v_scales": z(3, 0, 1, dtype=E8M0)}, "scales must be"),
    ({"k_scales": z(2, 2, 1, dtype=E8M0), "v_scales": z(2, 2, 1, dtype=E8M0)}, "scales must be"),
    ({"k_scales": z(3, 2, dtype=E8M0), "v_scales": z(3, 2, dtype=E8M0)}, "scales must be"),
    ({"table": torch.zeros(1, 2, dtype=torch.int64)}, "int32"),
    ({"table": torch.zeros(2, 2, dtype=torch.int32)}, "disagree"),
    ({}, "on a GPU"),
]


@pytest.mark.parametrize("change,match", BAD_CACHE + [
    ({"q": z(4, 64)}, "q must be"),
    ({"q": z(4, 2, 64, dtype=torch.float32)}, "bfloat16 or float16"),
    ({"q": z(4, 2, 128)}, "head_dim"),
    ({"k_scales": z(3, 8, 1, dtype=E8M0), "v_scales": z(3, 8, 1, dtype=E8M0)}, "multiple of 4"),
    ({"k_pages": z(3, 16, 1, 72, dtype=E4M3).as_strided((3, 16, 1, 64), (16 * 72, 72, 68, 1), 4)}, "8-byte aligned"),
    ({"k_pages": z(3, 16, 2, 64, dtype=E4M3).as_strided((3, 16, 1, 64), (2000, 68, 64, 1))}, "8-byte aligned"),
])
def test_attention_refusals(change, match):
    with pytest.raises(ValueError, match=match):
        A.paged_attention(**{"q": z(4, 2, 64), **cache(**change)})


@pytest.mark.parametrize("change,match", BAD_CACHE + [
    ({"k": z(4, 64)}, "k and v must be"),
    ({"v": z(5, 1, 64)}, "k and v must be"),
    ({"k": z(4, 2, 64), "v": z(4, 2, 64)}, "the caches hold"),
    ({"v": z(4, 1, 64, dtype=FP)}, "share one dtype"),
    ({"k": z(4, 1, 64, dtype=E4M3), "v": z(4, 1, 64, dtype=E4M3)}, "share one dtype"),
    ({"k": z(4, 1, 128)[..., ::2]}, "contiguous in the head"),
])
def test_append_refusals(change, match):
    with pytest.raises(ValueError, match=match):
        A.paged_append(**{"k": z(4, 1, 64), "v": z(4, 1, 64), **cache(**change)})


@pytest.mark.parametrize("change,match", BAD_CACHE + [
    ({"dtype": E4M3}, "dtype must be"),
    ({"tokens": -1}, "must not be negative"),
    ({"k_pages": z(3, 16, 1, 60, dtype=E4M3), "v_pages": z(3, 16, 1, 60, dtype=E4M3)}, "multiple"),
    ({"k_pages": z(3, 16, 1, 64, dtype=E4M3)[..., :60], "v_pages": z(3, 16, 1, 64, dtype=E4M3)[..., :60]}, "head_dim must be"),
    ({"k_scales": None, "v_scales": None}, "without scales"),
    ({"k_scales": None, "v_scales": None, "k_pages": z(3, 16, 1, 64), "v_pages": z(3, 16, 1, 64), "dtype": FP}, "own dtype"),
    ({"k_scales": None, "v_scales": None, "k_pages": z(3, 16, 1, 64), "v_pages": z(3, 16, 1, 64, dtype=FP)}, "without scales"),
])
def test_read_refusals(change, match):
    with pytest.raises(ValueError, match=match):
        A.paged_read(**{"tokens": 4, **cache(**change)})


POS, INV = torch.arange(4), torch.ones(32)


@pytest.mark.parametrize("change,match", [
    ({"q": z(4, 64)}, "q must be"),
    ({"k": z(5, 1, 64)}, "q must be"),
    ({"k": z(4, 1, 72)}, "q must be"),
    ({"k": z(4, 1, 64, dtype=FP)}, "share one dtype"),
    ({"q": z(4, 2, 64, dtype=torch.float64), "k": None}, "share one dtype"),
    ({"q": z(4, 1, 1032), "k": None}, "1024 columns"),
    ({"positions": POS.float()}, "positions must be"),
    ({"positions": POS[:3]}, "positions must be"),
    ({"inv_freq": INV.double()}, "inv_freq must be"),
    ({"inv_freq": torch.ones(33)}, "inv_freq must be"),
    ({"inv_freq": INV[None]}, "inv_freq must be"),
    ({"factor": math.inf}, "factor must be"),
    ({"factor": math.nan}, "factor must be"),
    ({"q": z(4, 2, 128)[..., ::2]}, "contiguous in the head"),
    ({"out": (z(4, 2, 64),)}, "out must be"),
    ({"out": (z(4, 2, 64), None)}, "out must be"),
    ({}, "on a GPU"),
])
def test_rotary_refusals(change, match):
    args = {"q": z(4, 2, 64), "k": z(4, 1, 64), "positions": POS, "inv_freq": INV}
    args.update(change)
    with pytest.raises(ValueError, match=match):
        rotary(**args)


def test_outputs_of_rotary_that_are_apart():
    from byteprof_amd.optim.rotary import _disjoint, _writable

    x = torch.zeros(6, 5, 8)
    assert _disjoint(x[:, :2], x[:, 2:]) and _disjoint(x[:, 2:], x[:, :2]) and _disjoint(x[:3], x[3:])
    assert not _disjoint(x[:, :3], x[:, 2:]) and not _disjoint(x[:4], x[3:]) and not _disjoint(x, x)
    assert _disjoint(x[..., :4], x[..., 4:]) is False  # columns of every head: not looked into
    assert not _disjoint(x[1:, :2], x[:5, 1:3]) and _disjoint(x[1:, :2], x[:5, 2:4])
    assert _writable(x) and _writable(x.transpose(0, 1)) and _writable(x[:, :2]) and _writable(x[:1])
    assert not _writable(torch.zeros(6, 1, 8).expand(6, 5, 8)) and not _writable(torch.zeros(1, 5, 8).expand(6, 5, 8))
    assert not _writable(x.view(-1).as_strided((6, 2, 8), (10, 8, 1)))


def test_rotary_frequencies():
    inv, by = rotary_frequencies(8, 10000.0)
    assert torch.allclose(inv.double(), torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=2.0 ** -23) and by == 1.0
    assert torch.equal(rotary_frequencies(8, scaling="linear", factor=4.0)[0], inv / 4)
    base, by = rotary_frequencies(8, scaling="base", factor=4.0)
    assert base[0] == 1.0 and abs(base[-1].item() / (0.001 / 4) - 1) < 1e-6 and by == 1.0
    # 10000 positions: 1591.5, 159.2, 15.9 and 1.59 turns
    parts, by = rotary_frequencies(8, scaling="parts", factor=8.0, trained=10000, slow=2.0, fast=100.0)
    ramp = (10000 * 0.01 / (2 * math.pi) - 2) / 98
    want = [1.0, 0.1, 0.01 * ramp + 0.01 / 8 * (1 - ramp), 0.001 / 8]
    assert torch.allclose(parts.double(), torch.tensor(want, dtype=torch.float64), rtol=2.0 ** -22)
    assert by == 0.1 * math.log(8.0) + 1.0
    assert torch.equal(rotary_frequencies(64, scaling="parts", factor=1.0, trained=100)[0], rotary_frequencies(64)[0])
    for bad in ({"dim": 7}, {"dim": 0}, {"dim": 8, "theta": 0.0}, {"dim": 8, "factor": 0.5}, {"dim": 8, "scaling": "other"},
                {"dim": 8, "scaling": "parts", "factor": 2.0}, {"dim": 2, "scaling": "base", "factor": 2.0},
                {"dim": 8, "scaling": "parts", "factor": 2.0, "trained": 100, "slow": 3.0, "fast": 3.0}):
        with pytest.raises(ValueError, match="rotary_frequencies"):
            rotary_frequencies(**bad)


class Cache(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("k_pages", "v_pages", "k_scales", "v_scales", "table", "lengths")] + [
        ("table_stride", ctypes.c_int64)] + [(n, ctypes.c_int64 * 3) for n in ("kp", "vp", "ks", "vs")] + [
        (n, ctypes.c_int32) for n in ("dtype", "seqs", "pool", "page", "block", "max_pages", "hk", "head_dim")]


def described(**kw):
    """A cache whose addresses are never dereferenced."""
    c = Cache(64, 64, 64, 64, 64, 64, 4, (1024, 64, 64), (1024, 64, 64), (1, 1, 1), (1, 1, 1), 4, 1, 4, 16, 16, 4, 1, 64)
    for name, value in kw.items():
        setattr(c, name, (ctypes.c_int64 * 3)(*value) if isinstance(value, tuple) else value)
    return ctypes.byref(c)


def test_the_description_is_the_headers():
    assert ctypes.sizeof(Cache) == A._DESCRIPTION.size == 6 * 8 + 13 * 8 + 8 * 4
    packed = A._DESCRIPTION.pack(*range(1, 28))
    c = Cache.from_buffer_copy(packed)
    assert (c.k_pages, c.lengths, c.table_stride, list(c.kp), list(c.vs), c.dtype, c.head_dim) == (1, 6, 7, [8, 9, 10], [17, 18, 19], 20, 27)


def test_attention_entry_refuses_before_any_launch(L):
    p = ctypes.c_void_p(64)

    def attn(dtype=0, q=p, out=ctypes.c_void_p(1 << 20), cu=p, tokens=4, hq=2, scale=0.1, ws=None, n=0, cache=None, **kw):
        return L.bp_attn_paged8(described(**kw), dtype, q, out, cu, tokens, hq, 128, 64, scale, ws, n, None)

    assert attn(tokens=0) == 0
    assert L.bp_attn_paged8(None, 0, p, p, p, 4, 2, 128, 64, 0.1, None, 0, None) == -1
    for kw in ({"dtype": 2}, {"head_dim": 60}, {"head_dim": 264}, {"tokens": 1 << 29}):
        assert attn(**kw) == -2, kw
    for kind in (0, 2):
        assert L.bp_attn_paged8(described(dtype=kind), 0, p, ctypes.c_void_p(1 << 20), p, 4, 2, 128, 64, 0.1, None, 0, None) == -2
    for kw in ({"q": None}, {"cu": None}, {"k_pages": None}, {"k_scales": None}, {"table": None}, {"lengths": None}, {"pool": 0},
               {"pool": -1}, {"seqs": -1}, {"max_pages": -1}, {"page": 0}, {"block": 0}, {"block": 2}, {"block": 12},
               {"page": 18, "block": 6}, {"k_pages": 68}, {"kp": (1024, 68, 64)}, {"hq": 3, "hk": 2}, {"hk": 0}, {"scale": 0.0},
               {"page": 1 << 20, "max_pages": 1 << 12}, {"out": p}):
        assert attn(**kw) == -1, kw
    assert attn(page=64, block=64, max_pages=100) == -3  # 6400 positions may be divided: no workspace
    need = L.bp_attn_paged8_workspace_bytes(4, 1, 2, 1, 64, 6400)
    assert need > 0 and attn(page=64, block=64, max_pages=100, ws=p, n=need - 1) == -3
    assert L.bp_attn_paged8_workspace_bytes(4, 1, 2, 1, 64, 256) == 0 and L.bp_attn_paged8_workspace_bytes(4, 1, 3, 2, 64, 6400) == 0


def test_append_and_read_entries_refuse_before_any_launch(L):
    p, odd = ctypes.c_void_p(64), ctypes.c_void_p(68)

    def append(dtype=0, k=p, tokens=4, cu=p, **kw):
        return L.bp_paged_append8(described(**kw), dtype, k, p, cu, tokens, 64, 64, 64, 64, None)

    assert append(page=4096, block=4096, head_dim=8, hk=1 << 23) == -2  # threads past 32 bits
    assert append(dtype=3) == -2 and append(hk=1 << 29) == -2 and append(page=1 << 16, block=1 << 16, head_dim=1 << 15) == -2
    assert L.bp_paged_append8(described(dtype=0), 0, p, p, p, 4, 64, 64, 64, 64, None) == -2
    assert L.bp_paged_append8(None, 0, p, p, p, 4, 64, 64, 64, 64, None) == -1
    for kw in ({"k": None}, {"k_scales": None}, {"table": None}, {"cu": None}, {"tokens": -1}, {"page": 0}, {"block": 0}, {"block": 5},
               {"page": 1 << 20, "max_pages": 1 << 10}, {"seqs": -1}):
        assert append(**kw) == -1, kw
    for kw in ({"tokens": 0}, {"seqs": 0}, {"pool": 0}, {"max_pages": 0}, {"head_dim": 0}, {"hk": 0}):
        assert append(**kw) == 0, kw

    far = ctypes.c_void_p(1 << 40)

    def read(dtype=0, k=ctypes.c_void_p(1 << 30), v=far, cu=p, tokens=4, **kw):
        return L.bp_paged_read(described(**kw), dtype, k, v, cu, tokens, None)

    assert read(dtype=3) == -2 and read(head_dim=60) == -2 and read(tokens=1 << 28, hk=8) == -2
    assert L.bp_paged_read(described(dtype=0), 1, p, p, p, 4, None) == -2 and L.bp_paged_read(described(dtype=2), 2, p, p, p, 4, None) == -2
    assert L.bp_paged_read(None, 0, p, p, p, 4, None) == -1
    for kw in ({"k_pages": None}, {"k_scales": None}, {"k": None}, {"table": None}, {"cu": None}, {"block": 5}, {"block": 0}, {"page": 0},
               {"tokens": -1}, {"k": odd}, {"k_pages": 68}, {"kp": (1024, 68, 64)}):
        assert read(**kw) == -1, kw
    assert read(tokens=0) == 0 and read(hk=0) == 0
    # k and v apart from each other and from the cache: codes of 4 pages of 1024 bytes from 1 << 35, 19 bytes of scales from 1 << 36
    apart = dict(k_pages=1 << 35, v_pages=1 << 35, k_scales=1 << 36, v_scales=1 << 36, ks=(6, 3, 1), vs=(6, 3, 1))
    for at in ((1 << 40) + 496, (1 << 40) - 496, (1 << 35) - 496, (1 << 35) + 4080, (1 << 36) - 496, (1 << 36) + 16):
        assert read(k=ctypes.c_void_p(at), **apart) == -1 and read(k=far, v=ctypes.c_void_p(at), **apart) == -1, at


def test_rotary_entry_refuses_before_any_launch(L):
    q, k, pos, inv = (ctypes.c_void_p(n << 20) for n in (1, 2, 3, 4))

    def rot(dtype=0, q=q, qo=ctypes.c_void_p(5 << 20), k=k, ko=ctypes.c_void_p(6 << 20), pos=pos, size=8, inv=inv, tokens=4, hq=2, hk=1,
            d=64, r=64, factor=1.0, q_t=128, qo_t=128, qo_h=64):
        at = lambda p: (p.value if p is not None else 0) or 0  # noqa: E731
        return L.bp_rotary(R._DESCRIPTION.pack(at(q), at(k), at(qo), at(ko), at(pos), at(inv), tokens, q_t, 64, 64, 64, qo_t, qo_h, 64, 64,
                                               dtype, size, hq, hk, d, r, 0, factor), None)

    assert L.bp_rotary(None, None) == -1 and R._DESCRIPTION.size == 6 * 8 + 9 * 8 + 8 * 4
    assert rot(tokens=0) == 0 and rot(d=0, r=0) == 0 and rot(hq=0, hk=0) == 0
    assert rot(dtype=3) == -2 and rot(d=1032) == -2
    far = dict(zip(("q", "k", "qo", "ko"), (ctypes.c_void_p(1 << n) for n in (40, 41, 42, 43))))
    assert rot(**far, tokens=1, hq=1 << 30, hk=1 << 30, d=8, r=8) == -2  # heads past 32 bits
    assert rot(**far, tokens=1 << 24, hq=1, hk=0, d=1024, r=1024, q_t=1024, qo_t=1024) == -2  # threads past 32 bits
    assert rot(r=63) == -1 and rot(r=66) == -1 and rot(r=-2) == -1 and rot(size=2) == -1 and rot(factor=math.nan) == -1
    assert rot(tokens=-1) == -1 and rot(hq=-1) == -1 and rot(q=None) == -1 and rot(ko=None) == -1 and rot(pos=None) == -1
    assert rot(inv=None) == -1 and rot(qo_t=100) == -1 and rot(qo_h=32) == -1
    assert rot(qo=ctypes.c_void_p((1 << 20) + 64)) == -1  # shifted within its own input
    assert rot(qo=k) == -1 and rot(qo=ctypes.c_void_p(6 << 20)) == -1 and rot(qo=pos) == -1 and rot(qo=inv) == -1
    assert rot(q_t=256, qo=q) == -1  # its own input's place, but not its strides


def test_read_entry_needs_a_table_wherever_it_looks_one_up(L):
    """Also with no page in the pool: every position of the table is looked up before its page is found to be outside."""
    p = ctypes.c_void_p(64)

    def read(**kw):
        return L.bp_paged_read(described(**kw), 0, ctypes.c_void_p(1 << 30), ctypes.c_void_p(1 << 40), p, 4, None)

    assert read(pool=0, table=None) == -1 and read(pool=0, lengths=None) == -1
    assert L.bp_paged_read(described(dtype=0, pool=0, table=None), 0, ctypes.c_void_p(1 << 30), ctypes.c_void_p(1 << 40), p, 4, None) == -1


@pytest.mark.parametrize("name", ["k_scales", "v_scales"])
def test_scales_that_require_a_gradient_are_refused(monkeypatch, name):
    """As the codes are: scales made of something that does are part of its graph."""
    monkeypatch.setattr(A, "_same_device", lambda *args: 0)
    scales = torch.ones(3, 2, 1, requires_grad=True).to(E8M0)
    assert scales.requires_grad
    for call in (lambda c: A.paged_attention(q=z(4, 2, 64), **c), lambda c: A.paged_append(k=z(4, 1, 64), v=z(4, 1, 64), **c),
                 lambda c: A.paged_read(tokens=4, **c)):
        with pytest.raises(ValueError, match="no backward"):
            call(cache(**{name: scales}))


def test_append_refuses_keys_and_values_in_one_place(monkeypatch, L):
    """One tensor for both scales (or both caches) would hold whichever was written last."""
    monkeypatch.setattr(A, "_same_device", lambda *args: 0)
    c, k = cache(), z(4, 1, 64)
    for same in ({"v_scales": c["k_scales"]}, {"v_pages": c["k_pages"]}, {"v_scales": c["k_scales"].view(torch.uint8).view(E8M0)}):
        with pytest.raises(ValueError, match="memory of their own"):
            A.paged_append(k=k, v=k, **{**c, **same})
    p = ctypes.c_void_p(64)
    apart = dict(k_pages=1 << 20, v_pages=2 << 20, k_scales=3 << 20, v_scales=4 << 20)
    for same in ({"v_scales": 3 << 20}, {"v_pages": 1 << 20}):
        assert L.bp_paged_append8(described(**{**apart, **same}), 0, p, p, p, 4, 64, 64, 64, 64, None) == -1, same


def test_a_batch_refuses_frequencies_that_are_not_its_heads():
    """Fewer pairs would turn a part of each head only, and tensors elsewhere would be found out in the middle of a pass."""
    from types import SimpleNamespace

    from byteprof_amd.optim.olmo import OlmoConfig
    from byteprof_amd.optim.olmo_batch import OlmoBatch

    cfg = OlmoConfig(hidden=128, ffn=64, layers=1, heads=2, vocab=20)
    dec = SimpleNamespace(cfg=cfg, device=torch.device("cpu"), inv_freq=torch.ones(32))
    assert OlmoBatch(dec, pages=2, rotary=(torch.ones(32), 1.25)).rotary[1] == 1.25
    for bad in ((torch.ones(16), 1.0), (torch.ones(64), 1.0), (torch.ones(32, dtype=torch.float64), 1.0), (torch.ones(1, 32), 1.0),
                (torch.ones(32, device="meta"), 1.0), (torch.ones(32), math.inf), (torch.ones(32), math.nan), (torch.ones(32),),
                torch.ones(32)):
        with pytest.raises(ValueError, match="rotary must be"):
            OlmoBatch(dec, pages=2, rotary=bad)
