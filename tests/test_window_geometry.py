"""The window prefill's tile lists, on the CPU: every key that a row sees lies in exactly one
tile that the row's wave computes, whatever the sizes, sides, sinks, key groups and
splits (tests/window_check.hip replays the kernels' own header)."""

import os
import random
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
OPEN = 1 << 30


@pytest.fixture(scope="module")
def checker(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("window") / "window_check")
    r = subprocess.run(["hipcc", "-x", "hip", "--offload-arch=gfx950", "-O1", "-std=c++17", "-w",
                        os.path.join(HERE, "window_check.hip"), "-o", exe], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-3000:]
    return exe


def run(exe, lines):
    text = "\n".join(" ".join(map(str, x)) for x in lines)
    out = subprocess.run([exe], input=text, capture_output=True, text=True, timeout=600, check=True).stdout.split("\n")
    bad = [(x, o) for x, o in zip(lines, out) if o != "ok"]
    assert len(out) > len(lines) and not bad, bad[:5]


# the kernels' block shapes: rows, keys per tile, key groups, splits
SHAPES = [(128, 64, 1, 1), (128, 64, 2, 1), (128, 64, 1, 3), (128, 32, 1, 1), (32, 128, 1, 1)]


@pytest.mark.parametrize("bm,bn,kg,splits", SHAPES)
def test_tile_lists(checker, bm, bn, kg, splits):
    lines = []
    for L, S in ((1, 1), (1, 500), (64, 64), (129, 129), (300, 300), (130, 700), (500, 130), (257, 256)):
        for left, right in ((0, 0), (1, 0), (31, 0), (63, 5), (64, 200), (200, OPEN), (OPEN, 3), (500, 0)):
            for sinks in (0, 1, 64, 65, 130, min(S, 400)):
                lines.append((L, S, left, right, min(sinks, S), bm, bn, kg, splits))
    rng = random.Random(bm + bn + kg + splits)
    for _ in range(400):
        S = rng.randint(1, 700)
        L = rng.choice((S, rng.randint(1, 700)))
        lines.append((L, S, rng.choice((OPEN, rng.randint(0, 300))), rng.choice((0, 0, OPEN, rng.randint(0, 300))),
                      min(S, rng.choice((0, 1, 4, rng.randint(0, 300)))), bm, bn, kg, rng.choice((splits, rng.randint(1, 7)))))
    run(checker, lines)
