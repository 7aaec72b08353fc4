"""How the cache's attention cuts its work, checked on the host: see cache_partition_check.cpp, which compiles the
headers that the kernels and their launches are built from."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "w4a16-gemm_b200", "csrc")

pytestmark = pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")


def build_and_run(tmp_path, csrc=None):
    exe = tmp_path / "partition_check"
    first = ["-I", str(csrc)] if csrc else []
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Werror", *first, "-I", CSRC,
                    os.path.join(HERE, "cache_partition_check.cpp"), "-o", str(exe)], check=True)
    return subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)


def test_work_is_cut_as_the_kernels_expect(tmp_path):
    r = build_and_run(tmp_path)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.startswith("ok ")


@pytest.mark.parametrize("line,instead", [
    ("u += kCdSegmentCost;\n        seg0 = u;", "seg0 = u;"),                       # a start that is not passed over
    ("(seg0 >= u0 ? 1 : 0)", "(seg0 > u0 ? 1 : 0)"),                                # a part's slot
    ("(unsigned long long)ctas - 1ull;", "(unsigned long long)ctas;"),               # the last CTA of a segment
    ("(ends_segment() ? kCdSegmentCost : 0) >= u1", "0 >= u1"),                     # the last unit of a CTA
    ("seg0 < u0 || seg0 + sh.tiles > u1", "seg0 < u0"),                             # parts that go on in the next CTA
    ("seen_from(window, pos0) / kCdTile", "(seen_from(window, pos0) + kCdTile - 1) / kCdTile"),    # the first tile
])
def test_the_check_notices_mistakes(tmp_path, line, instead):
    with open(os.path.join(CSRC, "cache_partition.h")) as f:
        text = f.read()
    assert text.count(line) == 1
    for name in ("cache_plan.h", "cache_schedule.h"):      # they include what stands beside them
        with open(os.path.join(CSRC, name)) as f:
            (tmp_path / name).write_text(f.read().replace("../../include/", ""))
    (tmp_path / "cache_partition.h").write_text(text.replace(line, instead))
    shutil.copy(os.path.join(CSRC, "..", "..", "include", "w4a16.h"), tmp_path)
    r = build_and_run(tmp_path, tmp_path)
    assert r.returncode == 1 and "FAIL" in r.stdout
