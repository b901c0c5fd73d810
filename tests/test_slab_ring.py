"""The host-compilable order of the slabs through which the dense layers' results leave, compiled and walked on the CPU."""

import re
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent
CSRC = ROOT.parent / "bionemo_inference_runtime_b200/csrc"


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_no_slab_is_written_before_its_store_has_read_it(tmp_path):
    program = tmp_path / "check"
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{CSRC}", str(ROOT / "slab_ring_check.cpp"), "-o", str(program)], check=True)
    done = subprocess.run([str(program)], capture_output=True, text=True)
    assert done.returncode == 0 and done.stdout == "ok\n", done.stdout


def test_the_products_pass_every_result_through_the_ring():
    """Slots and groups are counted in one place: the kernel itself commits nothing and advances nothing."""
    text = re.sub(r"//[^\n]*", "", (CSRC / "matmul.cuh").read_text())
    assert text.count(".pass(") == 1 and text.count("tma_store_commit()") == 1 and "++slot" not in text
