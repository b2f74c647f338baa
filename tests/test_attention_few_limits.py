"""From how many positions on launches of few rows a sequence are divided: below, neither a workspace nor a launch of the merge. CPU only."""

from __future__ import annotations

import pytest

from tests.test_attention_few_plan import plan  # noqa: F401  (a fixture)


@pytest.fixture(scope="module")
def workspace():
    from byteprof_amd import _lib

    return _lib.lib().bp_attn_paged8_workspace_bytes


@pytest.mark.parametrize("tokens,seqs,hq,hk,d", [(1, 1, 16, 16, 128), (64, 64, 32, 8, 128), (3, 3, 16, 16, 64), (54, 6, 16, 4, 128), (5, 1, 4, 1, 256)])
def test_no_workspace_where_nothing_is_divided(workspace, tokens, seqs, hq, hk, d):
    """A part has 512 keys at least, and a sequence is divided from one and a half times that on."""
    for most in (257, 272, 512, 767):
        assert workspace(tokens, seqs, hq, hk, d, most) == 0, most
    rows = next(r for r in (16, 32, 48) if tokens * hq // hk <= r * seqs)
    for most in (768, 1024, 1536, 8192):
        parts = -(-most // 512)
        need = workspace(tokens, seqs, hq, hk, d, most)
        assert 0 < need <= (tokens * hq // hk // rows + seqs) * hk * parts * rows * ((d if d != 72 else 96) + 2) * 4, most


@pytest.mark.parametrize("rb", [1, 2, 3])
def test_plans_about_the_limit(plan, rb):  # noqa: F811
    """Every part of every tile once, its slot inside the workspace, at lengths and capacities on either side."""
    cases = []
    for n in (511, 512, 767, 768, 769, 1279, 1280, 1281):
        for most in sorted({n, max(n, 767), max(n, 768), n + 300}):
            for seqs in (1, 3, 70):
                for hk in (1, 8):
                    cases.append((rb, [1] * seqs, [n] * (seqs - 1) + [max(1, n - 300)], 4 * hk, hk, 128, 0, most))
    for case, answer in zip(cases, plan(cases)):
        assert answer.endswith("divided 0") == (max(case[2]) < 768 or case[7] < 768), (case, answer)
