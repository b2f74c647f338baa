"""The plan of an attention launch on the CPU: csrc/attention_plan.h compiled for the host with a wave of 64 fibers
(tests/host), every workgroup's tile found as on the GPU. Every part of every tile comes out once, with keys that are whole and
apart and a slot of its own inside the workspace, and every row of a divided tile in one unit of the merge."""

from __future__ import annotations

import random
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    exe = tmp_path_factory.mktemp("plan") / "attention_plan"
    subprocess.run(["g++", "-std=c++17", "-O2", "-U_FORTIFY_SOURCE", f"-I{ROOT / 'tests/host'}",
                    f"-I{ROOT / 'byteprof_amd/csrc'}", f"-I{ROOT / 'include'}", str(ROOT / "tests/host/attention_plan.cpp"),
                    "-o", str(exe)], check=True)

    def run(cases):
        out = subprocess.run([str(exe)], input="\n".join(map(line, cases)) + "\n", capture_output=True, text=True, timeout=100)
        answers = out.stdout.splitlines()
        assert len(answers) == len(cases), (out.returncode, cases[len(answers)])
        wrong = [(c, a) for c, a in zip(cases, answers) if not a.startswith("ok")]
        assert not wrong, wrong[0]
        return answers

    return run


def line(case) -> str:
    counts, lengths, hq, hk, d, causal, pad, most = case
    cu = [0]
    for n in counts:
        cu.append(cu[-1] + n)
    tokens = cu[-1] + pad
    words = [tokens, len(counts), hq, hk, d, int(causal), tokens if lengths is None else most, *cu]
    return " ".join(map(str, words + ([] if lengths is None else ["paged", *lengths])))


def packed(counts, hq, hk, d=64, causal=True, pad=0):
    return counts, None, hq, hk, d, causal, pad, 0


def paged(counts, lengths, hq, hk, d=64, most=None):
    return counts, lengths, hq, hk, d, True, 0, most or max(lengths)


def log(rng, lo, hi):
    return round(lo * (hi / lo) ** rng.random())


def draw(rng, groups):
    """A plan of a few hundred to a few thousand tiles: one key head in the order of the tiles counts as many."""
    group, hk = rng.choice(groups), rng.choice((1, 2, 3, 8, 32))
    seqs = rng.choice((1, 2, 2, 3, 5, 20, 63, 64, 65, 130))
    rows = log(rng, 200, 100000)
    counts = [max(0, round(rows / group / seqs * rng.choice((0, 0.02, 0.5, 1, 2)))) for _ in range(seqs)]
    d = rng.choice((64, 96, 128, 256))
    if rng.random() < 0.5:
        return packed(counts, hk * group, hk, d, rng.random() < 0.7, rng.choice((0, 5)))
    lengths = [rng.choice((n, n, n + log(rng, 1, 50000), max(0, n - 7), 0)) for n in counts]
    return paged(counts, lengths, hk * group, hk, d, max(lengths) + rng.choice((1, 300)))


def test_every_part_once(plan):
    rng = random.Random(1)
    answers = plan([draw(rng, (1, 1, 2, 3, 4, 5, 7, 8, 16, 28, 40, 64, 100, 127, 128)) for _ in range(80)])
    assert sum("ordered 1" in a for a in answers) >= 15 and sum(not a.endswith("divided 0") for a in answers) >= 15


def test_more_query_heads_than_a_tile_has_rows(plan):
    """A token's rows are more than one tile: long sequences behind short ones and behind empty ones, in the order of the tiles."""
    cases = [packed([10, 4000], 160, 1), packed([0, 3000], 200, 1), packed([100, 1000], 200, 1), packed([5, 300], 256, 1),
             packed([30, 900], 192, 1, 128), paged([0, 40, 700], [0, 9000, 700], 400, 2, 256), packed([4, 0, 900, 3], 512, 1),
             paged([3, 600, 2], [3, 600, 2], 129, 1)]
    assert all("ordered 1" in a for a in plan(cases))
    rng = random.Random(2)
    plan([draw(rng, (129, 160, 192, 200, 255, 256, 300, 512)) for _ in range(40)])
