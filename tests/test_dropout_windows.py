"""The windows of dropout's odd rows, compiled for the host and walked for rows longer than any test's tensor."""

import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent
CSRC = ROOT.parent / "bionemo_inference_runtime_b200" / "csrc"


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_windows_of_long_rows(tmp_path):
    program = tmp_path / "check"
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{CSRC}", str(ROOT / "dropout_windows_check.cpp"), "-o", str(program)], check=True)
    done = subprocess.run([str(program)], capture_output=True, text=True)
    assert done.returncode == 0 and done.stdout == "ok\n", done.stdout


def test_the_kernel_takes_its_windows_there():
    kernel = (CSRC / "dropout.cu").read_text().split("dropout_rows_kernel(const DropoutParams p")[1].split("\n}\n")[0]
    assert "dropout_window(blockIdx.x" in kernel and "% unsigned(windows)" not in kernel
