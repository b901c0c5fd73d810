"""The host's question whether rows of two tensors have memory in common, compiled and compared with marks on every byte."""

import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_rows_in_common(tmp_path):
    program = tmp_path / "check"
    subprocess.run(["g++", "-std=c++17", "-O2", f"-I{ROOT.parent / 'bionemo_inference_runtime_b200/csrc'}",
                    str(ROOT / "rows_overlap_check.cpp"), "-o", str(program)], check=True)
    done = subprocess.run([str(program)], capture_output=True, text=True)
    assert done.returncode == 0 and done.stdout == "ok\n", done.stdout
