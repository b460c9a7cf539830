"""Host check: the matrix-product engine keeps a health flag in each source file that
instantiates it, so the function that reads the flag has to be each file's own too.  Two
files compiled without inlining, where a shared definition shows as a weak symbol."""
import re
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
NVCC = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"


@pytest.mark.skipif(not Path(NVCC).exists() or shutil.which("nm") is None, reason="no nvcc")
def test_each_file_reads_its_own_flag(tmp_path):
    src = tmp_path / "one.cu"
    src.write_text('#include "fms_gemm_tc.cuh"\nint read_one(int r) { return fms::gemm::read_error(r); }\n')
    subprocess.check_call([NVCC, "-gencode", "arch=compute_100a,code=sm_100a", "-O0", "-std=c++17", "-Xcompiler",
                           "-O0,-fno-inline", "-I", str(ROOT / "include"), "-I",
                           str(ROOT / "flashmaxsim.jl_b200" / "csrc"), "-c", str(src), "-o", str(tmp_path / "one.o")])
    table = subprocess.check_output(["nm", "-C", str(tmp_path / "one.o")], text=True)
    kinds = re.findall(r"^\S*\s+(\w) fms::gemm::read_error\(int\)", table, re.M)
    assert kinds == ["t"], table
