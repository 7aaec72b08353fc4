"""The prefill kernel's registers, as its compiler reports them: forms with an epilogue must not cost the plain store any."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")


@pytest.mark.skipif(not os.path.exists(NVCC), reason="needs nvcc")
def test_the_plain_store_spills_no_more_than_it_must(tmp_path):
    (tmp_path / "t.cu").write_text('#include "prefill.cuh"\n')
    report = subprocess.run([NVCC, "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", "-Xptxas", "-v", "-I", os.path.join(ROOT, "include"),
                             "-I", os.path.join(ROOT, "w4a16-gemm_b200", "csrc"), "-cubin", str(tmp_path / "t.cu"), "-o", str(tmp_path / "t.cubin")],
                            capture_output=True, text=True, check=True).stderr
    # prefill_kernel<G, TOK, OUT_F32, EPI>: fp16 stores of the plain form; 832 threads leave 78 registers each
    found = {}
    for g, tok, stores, loads in re.findall(r"Compiling entry function '\S*prefill_kernelILi(\d+)ELi(\d+)ELb0ELi0E\S*'.*?"
                                            r"(\d+) bytes spill stores, (\d+) bytes spill loads", report, re.S):
        found[int(g), int(tok)] = max(int(stores), int(loads))
    assert sorted(found) == [(g, t) for g in (64, 128) for t in (32, 64, 128, 256)]
    assert max(found.values()) <= 12, found
