"""What packed_attention, paged_attention, paged_append and token_logprobs refuse, at their Python names and at their C
entries. CPU only: every call here returns or raises before anything is enqueued."""

from __future__ import annotations

import ctypes
import re
from pathlib import Path

import pytest
import torch

from byteprof_amd.optim import attention as A
from byteprof_amd.optim.logprobs import token_logprobs

BF, FP = torch.bfloat16, torch.float16
CU = torch.tensor([0, 4], dtype=torch.int32)


def z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


@pytest.fixture(scope="module")
def L():
    from byteprof_amd import _lib

    return _lib.lib()


@pytest.mark.parametrize("q,k,v,cu,match", [
    (z(4, 64), z(4, 1, 64), z(4, 1, 64), CU, "q must be"),
    (z(4, 2, 64), z(5, 1, 64), z(5, 1, 64), CU, "q must be"),
    (z(4, 2, 64), z(4, 1, 64), z(4, 2, 64), CU, "q must be"),
    (z(4, 3, 64), z(4, 2, 64), z(4, 2, 64), CU, "no multiple"),
    (z(4, 2, 64), z(4, 0, 64), z(4, 0, 64), CU, "no multiple"),
    (z(4, 2, 60), z(4, 2, 60), z(4, 2, 60), CU, "multiple of 8"),
    (z(4, 2, 264), z(4, 2, 264), z(4, 2, 264), CU, "multiple of 8"),
    (z(4, 2, 64), z(4, 2, 72), z(4, 2, 72), CU, "head_dim"),
    (z(4, 2, 64, dtype=torch.float32),) + (z(4, 2, 64, dtype=torch.float32),) * 2 + (CU, "bfloat16 or float16"),
    (z(4, 2, 64), z(4, 2, 64), z(4, 2, 64, dtype=FP), CU, "share one dtype"),
    (z(4, 2, 64), z(4, 2, 64), z(4, 2, 64), CU.long(), "int32"),
    (z(4, 2, 64), z(4, 2, 64), z(4, 2, 64), CU[:0], "at least one"),
    (z(4, 2, 64), z(4, 2, 64), z(4, 2, 64), CU[None], "int32"),
    (z(4, 2, 64), z(4, 2, 64), z(4, 2, 64), CU, "on a GPU"),
])
def test_packed_refusals(q, k, v, cu, match):
    with pytest.raises(ValueError, match=match):
        A.packed_attention(q, k, v, cu)


def paged(**kw):
    args = {"q": z(4, 2, 64), "k_pages": z(3, 16, 1, 64), "v_pages": z(3, 16, 1, 64),
            "table": torch.zeros(1, 2, dtype=torch.int32), "lengths": torch.tensor([4], dtype=torch.int32), "cu": CU}
    args.update(kw)
    return args


@pytest.mark.parametrize("change,match", [
    ({"q": z(4, 64)}, "q must be"),
    ({"k_pages": z(3, 16, 64)}, "caches must be"),
    ({"v_pages": z(3, 8, 1, 64)}, "caches must be"),
    ({"k_pages": z(3, 0, 1, 64), "v_pages": z(3, 0, 1, 64)}, "caches must be"),
    ({"k_pages": z(3, 16, 1, 128)[..., ::2]}, "contiguous in the head dimension"),
    ({"table": torch.zeros(1, 2, dtype=torch.int64)}, "int32"),
    ({"table": torch.zeros(2, 2, dtype=torch.int32)}, "disagree"),
    ({"lengths": torch.zeros(2, dtype=torch.int32)}, "disagree"),
    ({"table": torch.zeros(2, 1, dtype=torch.int32).T.expand(1, 2)[:, :1].expand(1, 1 << 26)}, "int32"),
    ({"k_pages": z(3, 16, 1, 64, dtype=FP)}, "share one dtype"),
    ({}, "on a GPU"),
])
def test_paged_refusals(change, match):
    with pytest.raises(ValueError, match=match):
        A.paged_attention(**paged(**change))


def test_a_scale_has_to_be_positive():
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="scale must be"):
            A._scale("x", scale, 64)
    assert A._scale("x", None, 64) == 0.125


@pytest.mark.parametrize("change,match", [
    ({"k": z(4, 64)}, "k and v must be"),
    ({"v": z(5, 1, 64)}, "k and v must be"),
    ({"k": z(4, 2, 64), "v": z(4, 2, 64)}, "the caches hold"),
    ({"v": z(4, 1, 64, dtype=FP)}, "share one dtype"),
    ({"k": z(4, 1, 128)[..., ::2]}, "contiguous in the head"),
    ({"cu": CU[:1]}, "disagree"),
    ({}, "on a GPU"),
])
def test_append_refusals(change, match):
    args = paged()
    del args["q"]
    args.update({"k": z(4, 1, 64), "v": z(4, 1, 64)})
    args.update(change)
    with pytest.raises(ValueError, match=match):
        A.paged_append(**args)


@pytest.mark.parametrize("logits,targets,top,match", [
    (z(10), None, 0, "logits must be"),
    (z(10, 2).T, None, 0, "logits must be"),
    (torch.zeros(2, 10, dtype=torch.float64), None, 0, "bfloat16, float16 or float32"),
    (z(2, 10), None, 11, "top must be"),
    (z(2, 100), None, 33, "top must be"),
    (z(2, 100), None, -1, "top must be"),
    (z(2, 0), None, 0, "vocabulary"),
    (z(2, 10), torch.zeros(2, dtype=torch.int32), 0, "targets"),
    (z(2, 10), torch.zeros(3, dtype=torch.int64), 0, "targets"),
    (z(2, 10), None, 2, "on a GPU"),
])
def test_logprobs_refusals(logits, targets, top, match):
    with pytest.raises(ValueError, match=match):
        token_logprobs(logits, targets, top=top)


def test_attention_entries_refuse_before_any_launch(L):
    p, odd = ctypes.c_void_p(64), ctypes.c_void_p(72)  # never dereferenced

    def packed(dtype=0, q=p, k=p, out=p, cu=p, tokens=4, seqs=1, hq=2, hk=1, d=64, q_t=128, scale=0.1, ws=None, n=0):
        return L.bp_attn_packed(dtype, q, k, p, out, cu, tokens, seqs, hq, hk, d, q_t, 64, 64, 64, 64, 64, 1, scale, ws, n, None)

    assert packed(tokens=0) == 0
    assert packed(dtype=2) == -2 and packed(d=60) == -2 and packed(d=264) == -2 and packed(d=0) == -2
    assert packed(q=None) == -1 and packed(k=None) == -1 and packed(out=None) == -1 and packed(cu=None) == -1
    assert packed(q=odd) == -1 and packed(out=odd) == -1 and packed(q_t=100) == -1
    assert packed(hq=3, hk=2) == -1 and packed(hk=0) == -1 and packed(tokens=-1) == -1 and packed(seqs=-1) == -1
    assert packed(scale=0.0) == -1 and packed(scale=float("nan")) == -1
    assert packed(tokens=1 << 29, hq=2) == -2  # rows past 32 bits
    need = L.bp_attn_workspace_bytes(1000, 1, 2, 1, 64, 1000)
    assert need > 0
    assert packed(tokens=1000) == -3 and packed(tokens=1000, ws=p, n=need - 1) == -3 and packed(tokens=1000, ws=odd, n=need) == -3

    def paged(table=p, lengths=p, pool=4, page=16, pages=4, seqs=1, k=p):
        return L.bp_attn_paged(0, p, k, p, p, table, 4, lengths, p, 4, seqs, pool, page, pages, 2, 1, 64, 128, 64, 1024, 64, 64,
                               1024, 64, 64, 0.1, None, 0, None)

    assert paged(table=None) == -1 and paged(lengths=None) == -1 and paged(k=None) == -1
    assert paged(page=0) == -1 and paged(pool=-1) == -1 and paged(pool=0) == -1 and paged(pages=-1) == -1
    assert paged(page=1 << 20, pages=1 << 12) == -1
    assert paged(page=64, pages=100) == -3  # 6400 positions may be divided: no workspace


def test_append_entry_refuses_before_any_launch(L):
    p = ctypes.c_void_p(64)

    def append(size=2, k=p, table=p, tokens=4, seqs=1, pool=4, page=16, pages=4, hk=1, d=64):
        return L.bp_paged_append(size, k, p, p, p, table, 4, p, p, tokens, seqs, pool, page, pages, hk, d, *([64] * 10), None)

    assert append(size=3) == -1 and append(k=None) == -1 and append(table=None) == -1 and append(tokens=-1) == -1
    assert append(page=0) == -1 and append(page=1 << 20, pages=1 << 10) == -1
    assert append(tokens=0) == 0 and append(seqs=0) == 0 and append(pool=0) == 0 and append(pages=0) == 0 and append(d=0) == 0
    assert append(hk=1 << 16, d=1 << 15) == -2


def test_logprobs_entry_refuses_before_any_launch(L):
    p = ctypes.c_void_p(64)

    def lp(dtype=0, x=p, targets=p, logprob=p, entropy=p, ids=p, tl=p, rows=2000, vocab=100, top=5, ws=None, n=0, stride=100):
        return L.bp_logprobs(dtype, x, stride, targets, logprob, entropy, ids, tl, rows, vocab, top, ws, n, None)

    assert lp(rows=0) == 0
    assert lp(dtype=3) == -2 and lp(top=33) == -2 and lp(vocab=1 << 30) == -2 and lp(rows=1 << 24) == -2
    assert lp(x=None) == -1 and lp(entropy=None) == -1 and lp(ids=None) == -1 and lp(tl=None) == -1 and lp(logprob=None) == -1
    assert lp(rows=-1) == -1 and lp(vocab=-1) == -1 and lp(top=-1) == -1 and lp(stride=-1) == -1 and lp(vocab=0) == -1
    assert lp(vocab=4) == -1 and lp(x=ctypes.c_void_p(65)) == -1
    assert lp(rows=1, vocab=100000) == -3
    assert L.bp_logprobs_workspace_bytes(0, 2000, 100, 5) == 0 and L.bp_logprobs_workspace_bytes(0, 1, 100000, 5) > 0


def test_workspace_of_attention(L):
    """None where no sequence can have more keys than a split; within a bound of the target elsewhere."""
    text = (Path(__file__).resolve().parent.parent / "include" / "byteprof_amd.h").read_text()
    assert int(re.search(r"#define BP_ATTN_UNDIVIDED_KEYS (\d+)", text).group(1)) == A.UNDIVIDED_KEYS
    assert L.bp_attn_workspace_bytes(64, 64, 32, 8, 128, A.UNDIVIDED_KEYS) == 0
    assert L.bp_attn_workspace_bytes(64, 64, 32, 8, 128, A.UNDIVIDED_KEYS + 1) > 0
    assert L.bp_attn_workspace_bytes(0, 1, 8, 8, 128, 10000) == 0
    small = L.bp_attn_workspace_bytes(1, 1, 16, 16, 128, 512)  # 16 heads, 2 parts, 32 rows
    assert small == 16 * 2 * 32 * (128 + 2) * 4
    assert L.bp_attn_workspace_bytes(1 << 14, 64, 32, 8, 128, 1 << 20) <= 1400 * 128 * 130 * 4


def test_a_scale_that_leaves_the_range_of_float32_is_refused(L):
    for scale in (1e39, 3e38, 1e-60):
        with pytest.raises(ValueError, match="scale must be"):
            A._scale("x", scale, 64)
    assert A._scale("x", 2e38, 64) == 2e38 and A._scale("x", 1e-37, 64) == 1e-37
    p = ctypes.c_void_p(64)  # never dereferenced

    def packed(scale):
        return L.bp_attn_packed(0, p, p, p, p, p, 1000, 1, 2, 1, 64, 128, 64, 64, 64, 64, 64, 1, scale, None, 0, None)

    assert packed(3e38) == -1 and packed(float("inf")) == -1 and packed(2e38) == -3  # the last: no workspace


def test_attention_entries_refuse_an_output_that_overlaps_what_they_read(L):
    """out over k or v, or over another part of q; nothing is dereferenced, the places are numbers."""
    kb = 4 * 64 * 2  # bytes of 4 tokens of one head of 64

    def packed(out, q=1 << 20, k=2 << 20, v=3 << 20, q_t=128, k_t=64):
        ptr = ctypes.c_void_p
        return L.bp_attn_packed(0, ptr(q), ptr(k), ptr(v), ptr(out), ptr(64), 4, 1, 2, 1, 64, q_t, 64, k_t, 64, k_t, 64, 1, 0.1,
                                None, 0, None)

    assert packed(2 << 20) == -1 and packed(3 << 20) == -1 and packed((2 << 20) + kb - 16) == -1
    assert packed((3 << 20) - 2 * kb + 16) == -1 and packed((1 << 20) + 128) == -1 and packed(1 << 20, q_t=256) == -1
    assert packed((2 << 20) + 3 * 1024 * 2, k_t=1024) == -1  # the last of k's rows

    def paged(out, pool=3, page=16):
        ptr = ctypes.c_void_p
        return L.bp_attn_paged(0, ptr(1 << 20), ptr(2 << 20), ptr(3 << 20), ptr(out), ptr(64), 4, ptr(64), ptr(64), 4, 1, pool,
                               page, 4, 2, 1, 64, 128, 64, 1024, 64, 64, 1024, 64, 64, 0.1, None, 0, None)

    assert paged(2 << 20) == -1 and paged((3 << 20) + 2 * (3 * 16 * 64) - 16) == -1 and paged((1 << 20) + 16) == -1


def test_out_has_to_be_apart():
    q, k, v = z(4, 2, 64), z(4, 2, 64), z(4, 2, 64)
    both = z(2, 4, 2, 64)
    assert A._output("x", q, q, k, v) is q and A._output("x", both[0], both[1], k, v) is not None
    for out, read in ((k, (k, v)), (v, (k, v)), (both[0], (both[1], both)), (both[1], (both.transpose(0, 1)[:, 1], v))):
        with pytest.raises(ValueError, match="overlap"):
            A._output("x", q, out, *read)
    wide = z(5, 2, 64)
    with pytest.raises(ValueError, match="overlap"):
        A._output("x", wide[1:], wide[:4], k, v)


def test_a_batch_refuses_its_arguments_before_any_pass(monkeypatch):
    from types import SimpleNamespace

    from byteprof_amd.optim.olmo import OlmoConfig
    from byteprof_amd.optim.olmo_batch import OlmoBatch

    dec = SimpleNamespace(cfg=OlmoConfig(hidden=64, ffn=64, layers=1, heads=1, vocab=20), device=torch.device("cpu"))
    batch = OlmoBatch(dec, pages=4)
    monkeypatch.setattr(batch, "_forward", lambda *a, **k: pytest.fail("a pass ran"))
    ids = [torch.tensor([1, 2, 3])]
    for top in (33, 21, -1):
        with pytest.raises(ValueError, match="top must be"):
            batch.generate(ids, max_new_tokens=2, top=top)
        with pytest.raises(ValueError, match="top must be"):
            batch.score(ids, top=top)
    assert len(batch.free) == 4
