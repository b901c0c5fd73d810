"""The host's questions about an index of adapters, compiled and asked on the CPU."""

import os
import re
import shutil
import subprocess
from pathlib import Path

import pytest

from bionemo_inference_runtime_b200.csrc import build

ROOT = Path(__file__).resolve().parent


@pytest.mark.skipif(not (shutil.which("nvcc") or os.path.exists("/usr/local/cuda/bin/nvcc")), reason="needs nvcc")
def test_entries_and_tiles(tmp_path):
    program = tmp_path / "check"
    subprocess.run([build._nvcc(), *build.NVCC_FLAGS, f"-I{build.CSRC}", str(ROOT / "adapter_index_check.cu"), "-o", str(program)], check=True)
    done = subprocess.run([str(program)], capture_output=True, text=True)
    assert done.returncode == 0 and done.stdout == "ok\n", done.stdout


def test_pairs_of_blocks_are_charged_the_adapters_of_their_rows():
    text = (build.CSRC / "dense.cu").read_text()
    assert re.search(r"more_pair = double\(adapters_of_tile\(.*, 2 \* matmul::kBM\)", text)
    assert "m.kblocks + m.more_pair" in text.split("consider(n, 1, 0")[1].split("\n")[0]
