"""CPU check that the sizes the GPU tests of the product of 8-bit codes run reach every form
of it, as the table of costs stands: a change of that table that takes a form its tests away
fails here."""
import os
import subprocess

import pytest

import jllm
import test_gemm_i8_rounding_gpu as rounding
import test_layer_i8_gpu as layer

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FEW = ["", "few", "few, many channels", "few, long K"]
TILES = ["256 x 256", "128 x 256", "128 x 128", "64 x 64", "32 x 64"]


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    exe = tmp_path_factory.mktemp("plan") / "gemm_plan_test"
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", os.path.join(ROOT, "genie-ai-runtime_amd", "csrc"),
                    os.path.join(ROOT, "tests", "cxx", "gemm_plan_test.cpp"), "-o", str(exe)], check=True)

    def of(sizes):
        got = subprocess.run([str(exe)], input="".join("%d %d %d\n" % s for s in sizes), capture_output=True, text=True, check=True)
        out = []
        for line in got.stdout.splitlines():
            few, tile, splits, whole = map(int, line.split())
            out.append((FEW[few] if few else "rounds" if whole else TILES[tile], splits))
        return out

    return of


def test_every_form_is_tested(plans):
    got = plans(rounding.FORMS)
    assert {f for f, _ in got} == set(FEW[1:] + TILES + ["rounds"])
    assert sum(s > 1 for _, s in got) >= 3
    assert {f for f, _ in plans(layer.FORMS)} >= set(TILES + ["rounds"])


def test_every_tile_has_whole_and_odd_rows(plans):
    """fp16 rows of whole 16-byte pieces (M a multiple of 8) and others, each with a last tile
    that M cuts, uncut in K: they leave the tile in different ways."""
    wide = {"rounds": 256, "256 x 256": 256, "128 x 256": 128, "128 x 128": 128, "64 x 64": 64, "32 x 64": 32}
    seen = {(f, M % 8 == 0) for (M, N, K), (f, s) in zip(rounding.FORMS, plans(rounding.FORMS)) if s == 1 and M % wide.get(f, M + 1)}
    assert seen >= {(f, whole) for f in wide for whole in (False, True)}


def test_workspace_is_the_plans(plans):
    sizes = layer.FORMS + rounding.FORMS + layer.GEMM
    for (M, N, K), (_, s) in zip(sizes, plans(sizes)):
        need = 4 * s * M * N if s > 1 else 0
        assert jllm.lib().jllm_hip_gemm_i8_workspace(M, N, K) == (need + 15) // 16 * 16
