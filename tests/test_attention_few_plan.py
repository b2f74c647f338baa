"""The plan of an attention launch of few rows a sequence on the CPU (csrc/attention_plan.h, FewTiles; tests/host): every part of every
tile comes out once, with keys that are whole and apart and a slot of its own inside the workspace, and every row of a divided tile
in one unit of the merge, whatever the offsets hold: also sequences of far more rows than the host expects."""

from __future__ import annotations

import random
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    exe = tmp_path_factory.mktemp("plan") / "attention_few_plan"
    subprocess.run(["g++", "-std=c++17", "-O2", "-U_FORTIFY_SOURCE", f"-I{ROOT / 'tests/host'}",
                    f"-I{ROOT / 'byteprof_amd/csrc'}", f"-I{ROOT / 'include'}", str(ROOT / "tests/host/attention_few_plan.cpp"),
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
    rb, counts, lengths, hq, hk, d, pad, most = case
    cu = [0]
    for n in counts:
        cu.append(cu[-1] + n)
    return " ".join(map(str, [rb, cu[-1] + pad, len(counts), hq, hk, d, most, *cu, *lengths]))


def draw(rng, rb):
    group, hk = rng.choice((1, 2, 3, 4, 7, 8, 16, 16 * rb)), rng.choice((1, 2, 3, 8, 16))
    seqs = rng.choice((1, 2, 3, 5, 20, 63, 64, 65, 130))
    most = max(1, 16 * rb // group)
    counts = [rng.choice((0, 1, 1, rng.randint(1, most))) for _ in range(seqs)]
    if rng.random() < 0.3:  # not what the host expects: all tokens are one sequence's
        counts = [0] * (seqs - 1) + [sum(counts) + 1]
    long = rng.choice((100, 5000, 100000))
    lengths = [rng.choice((n, n + rng.randint(0, long), rng.randint(0, 300), max(0, n - 3))) for n in counts]
    return rb, counts, lengths, hk * group, hk, rng.choice((64, 96, 128, 256 if rb < 3 else 128)), rng.choice((0, 0, 5)), max(lengths) + rng.choice((1, 300))


@pytest.mark.parametrize("rb", [1, 2, 3])
def test_every_part_once(plan, rb):
    rng = random.Random(rb)
    answers = plan([draw(rng, rb) for _ in range(60)])
    assert sum("ordered 1" in a for a in answers) >= 5 and sum(not a.endswith("divided 0") for a in answers) >= 10
