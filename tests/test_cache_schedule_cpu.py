"""The order of the cache prompt kernel's tensor-core products, checked on the host: see
cache_schedule_check.cpp, which compiles the header that the kernel is built from."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "w4a16-gemm_b200", "csrc")


def build_and_run(tmp_path, csrc):
    exe = tmp_path / "schedule_check"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-I", str(csrc),
                    os.path.join(HERE, "cache_schedule_check.cpp"), "-o", str(exe)], check=True)
    return subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_products_wait_for_what_they_overwrite(tmp_path):
    r = build_and_run(tmp_path, CSRC)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.startswith("ok ")


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
@pytest.mark.parametrize("line,left", [
    # next scores over the weights of an unfinished product
    ("!op.wait_o(h, w.step_of(e) - 1)", "false"),
    # a stage handed back after the first half's product
    ("if (w.ends_tile(e)) op.commit_k(st);", "if (!w.ends_tile(e) || w.shift() == 0) op.commit_k(st);"),
    # a product that does not wait for the weights
    ("|| !op.wait_p(h, step)", ""),
])
def test_the_check_notices_what_is_left_out(tmp_path, line, left):
    with open(os.path.join(CSRC, "cache_schedule.h")) as f:
        text = f.read()
    assert text.count(line) == 1
    (tmp_path / "cache_schedule.h").write_text(text.replace(line, left))
    r = build_and_run(tmp_path, tmp_path)
    assert r.returncode == 1 and "FAIL" in r.stdout
