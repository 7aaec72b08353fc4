"""CPU test of which form an expert layer's call takes: the plan, compiled by itself, at the borders of its rule."""
import os
import subprocess

PLAN = r"""
#include <cstdio>
#include <initializer_list>
#include "moe_plan.h"
using namespace w4a16;
int main() {
    for (int experts : {1, 8, 64, 128})
        for (int k : {1, 2, 8})
            for (int wide = 0; wide < 2; ++wide)
                for (long long tokens = 1; tokens < 3000; ++tokens) {
                    const MoePlan p = moe_plan(tokens, k, experts, 512, 256, 148, wide != 0);
                    const long long entries = tokens * k;
                    if (p.grouped != (entries > (wide ? 10 : 14) * experts)) return 1;
                    if (p.rows != (p.grouped ? 64 : 8) || p.few != (!p.grouped && entries <= 1024)) return 2;
                    if (wide == 0 && p.bytes != moe_plan(tokens, k, experts, 512, 256, 148).bytes) return 3;
                }
    std::puts("ok");
}
"""


def test_the_form_follows_entries_and_groups(tmp_path):
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "w4a16-gemm_b200", "csrc")
    (tmp_path / "plan.cpp").write_text(PLAN)
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Wextra", "-I", csrc, str(tmp_path / "plan.cpp"), "-o", str(tmp_path / "plan")], check=True)
    run = subprocess.run([str(tmp_path / "plan")], capture_output=True, text=True)
    assert run.returncode == 0 and run.stdout == "ok\n", run.returncode
