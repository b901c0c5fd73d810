"""Registers of the few rows' kernel, whose blocks on a multiprocessor they decide."""

import os
import re
import shutil
import subprocess

import pytest

from bionemo_inference_runtime_b200.csrc import build


@pytest.mark.skipif(not (shutil.which("nvcc") or os.path.exists("/usr/local/cuda/bin/nvcc")), reason="needs nvcc")
def test_adapters_take_no_registers_from_layers_without_them(tmp_path):
    """With 256 threads to a block: five, four and three blocks of 65536 registers, those of the widest layers that have weights to read."""
    done = subprocess.run([build._nvcc(), *build.NVCC_FLAGS, "-Xptxas", "-v", "-c", str(build.CSRC / "dense.cu"), "-o", str(tmp_path / "dense.o")],
                          capture_output=True, text=True)
    assert done.returncode == 0, done.stderr
    used = {}
    for name, rest in re.findall(r"Compiling entry function '(\w*few_rows_kernel\w*)'(.*?registers)", done.stderr, re.S):
        two, eights, vec, adapt = map(int, re.search(r"Lb(\d)ELi(\d)ELb(\d)ELb(\d)", name).groups())
        if vec and not adapt:
            used.setdefault((two, eights), set()).add(int(re.search(r"Used (\d+) registers", rest).group(1)))
    assert used.keys() == {(0, 1), (0, 2), (1, 1), (1, 2)}
    for form, most in (((0, 1), 48), ((0, 2), 64), ((1, 1), 80), ((1, 2), 96)):  # 65536 / 256 threads, in steps of 8: 5, 4, 3 and 2 blocks
        assert max(used[form]) <= most, form
