"""Where a sequence of the position bias stands, in whole numbers, without a GPU."""
import os
import subprocess

import numpy as np

from conftest import REPO


def test_positions_do_not_wrap(tmp_path):
    exe = str(tmp_path / "corner_check")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-Wno-unknown-pragmas", "-fsanitize=undefined", "-fno-sanitize-recover",
                    os.path.join(REPO, "tests", "corner_check.cc"), "-o", exe], check=True)
    rng = np.random.default_rng(1)
    ask = []
    for _ in range(5000):
        rel0, own, step = (int(rng.integers(-(1 << 20), 1 << 20)) for _ in range(3))
        rel0 += int(rng.choice([0, (1 << 61) - (1 << 20), -(1 << 61) + (1 << 20), 1 << 30, -(1 << 30)]))
        own += int(rng.choice([0, rel0, (1 << 63) - (1 << 20), -(1 << 63) + (1 << 20), 1 << 62, -(1 << 62), 1 << 30, -(1 << 30), 1 << 61]))
        ask.append((rel0, max(-(1 << 63), min((1 << 63) - 1, own)), step))
    ask += [(r, o, s) for r in (0, 1 << 61, -(1 << 61)) for o in ((1 << 63) - 1, -(1 << 63)) for s in (0, 1 << 31, -(1 << 31))]
    got = subprocess.run([exe], input="\n".join("%d %d %d" % x for x in ask), capture_output=True, text=True, check=True).stdout.split()
    most = (1 << 30) + 65536
    assert [int(x) for x in got] == [max(-most, min(most, r - o + s)) for r, o, s in ask]
