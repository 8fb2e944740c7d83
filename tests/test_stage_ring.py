"""CPU check of the tile kernels' producers (csrc/stage_ring.cuh) on a model of their barriers.

A producer leaves its ring only when every stage that it filled is free again: the MMAs' arrivals
are asynchronous, reach both CTAs of a pair, and may not land in a CTA that has ended."""

from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

HERE = Path(__file__).resolve().parent
CSRC = HERE.parent / "cuda_force_b200" / "csrc"


@pytest.fixture(scope="module")
def check(tmp_path_factory):
    path = tmp_path_factory.mktemp("stage_ring")
    shutil.copy(CSRC / "stage_ring.cuh", path)
    (path / "ptx.cuh").write_text("")  # in the place of the device's: the model is its own
    exe = path / "check_stage_ring"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-Wno-unknown-pragmas",
                    f"-I{path}", str(HERE / "native" / "check_stage_ring.cpp"), "-o", str(exe)],
                   check=True)
    return lambda *args: subprocess.run([str(exe), *args], capture_output=True, text=True,
                                        timeout=60)


def test_a_producer_leaves_nothing_under_way(check):
    out = check()
    assert out.returncode == 0, out.stdout
    assert out.stdout.splitlines()[-1] == "0 left under way"


def test_the_model_sees_a_producer_that_leaves_early(check):
    assert check("drop_wait").returncode == 1


def test_the_tile_kernels_end_their_producers_that_way():
    for name in ("fp8_linear.cu", "gated_linear.cu"):
        source = (CSRC / name).read_text()
        assert source.count("StageRing<C::kStages> ring;") == 1, name
        assert source.count("ring.wait_all_free(empty)") == 1, name
