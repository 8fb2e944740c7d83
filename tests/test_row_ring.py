"""CPU check of the row ring's bookkeeping (csrc/row_ring.cuh) on a model of its barriers.

On a GPU a wait that gives up is a protocol failure that no test provokes; here each wait of the
row loop gives up in turn, and the copies that are in flight then have to be waited for before
the CTA's shared memory goes away."""

from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

HERE = Path(__file__).resolve().parent
CSRC = HERE.parent / "cuda_force_b200" / "csrc"


def test_no_copy_is_left_in_flight(tmp_path):
    # Beside the ring, empty headers in the place of the device's: the model is its own.
    shutil.copy(CSRC / "row_ring.cuh", tmp_path)
    for name in ("cf_common.cuh", "ptx.cuh"):
        (tmp_path / name).write_text("")
    exe = tmp_path / "check_row_ring"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror",
                    "-Wno-unknown-pragmas", f"-I{tmp_path}",
                    str(HERE / "native" / "check_row_ring.cpp"), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0, out.stdout
    assert out.stdout.splitlines()[-1].endswith(" 0 copies left in flight")
