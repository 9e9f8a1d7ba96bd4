"""CPU check of the first key of a shared prefix that a window leaves a row, over the whole
range of lengths: prefix and own tokens together may pass 31 bits."""
import os
import random
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BIG = 2 ** 31 - 1


def test_first_key_that_a_window_leaves(tmp_path):
    exe = tmp_path / "prefix_window_test"
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", os.path.join(ROOT, "genie-ai-runtime_amd", "csrc"),
                    os.path.join(ROOT, "tests", "cxx", "prefix_window_test.cpp"), "-o", str(exe)], check=True)
    cases = [(5003, 300, 4096), (5003, 0, 5003), (5003, 0, 5004), (5003, 4096, 4096), (5003, 4097, 4096), (0, 0, 1),
             (0, 7, 3), (7, 0, BIG), (BIG, 0, 1), (BIG, 0, BIG), (BIG, 1, BIG), (BIG, 64, 64), (BIG, 63, 64),
             (BIG, BIG, 1), (BIG, BIG, BIG), (BIG, BIG - 1, BIG), (1 << 30, 1 << 30, 1), (1 << 30, 1 << 30, 100),
             (1500000000, 1200000000, 100), (1, BIG, BIG), (1, BIG, 1)]
    r = random.Random(7)
    cases += [tuple(int((BIG + 1) ** r.random()) - d for d in (1, 1, 0)) for _ in range(2000)]
    cases = [(a, b, min(max(w, 1), BIG)) for a, b, w in cases]
    got = subprocess.run([str(exe)], input="".join("%d %d %d\n" % c for c in cases), capture_output=True, text=True, check=True)
    want = [min(max(a + b - w, 0), a) for a, b, w in cases]
    assert [int(x) for x in got.stdout.split()] == want

