"""CPU tests of the expert layer's entry points: what they refuse.  No call here reaches a device: what is not refused by its
arguments ends at the check for one."""
import ctypes

import pytest
import torch

from w4a16_opt import capi

DEVICE = (13, 14)


@pytest.fixture(autouse=True)
def _no_device():
    """The addresses of these calls are not real: with a device they would be used."""
    if torch.cuda.is_available():
        pytest.skip("for machines without a GPU")


def args(**kw):
    a = dict(x=0x100000, gate_up_wp=0x200000, gate_up_scales=0x300000, down_wp=0x400000, down_scales=0x500000, experts=0x600000,
             weights=0x700000, y=0x800000, tokens=4, num_experts=8, k=2, hidden=256, inner=128, gate_up_group=128, down_group=64,
             activation=2)
    a.update(kw)
    return capi.MoeArgs(**a)


def call(**kw):
    lib = capi.load()
    a = args(**kw)
    st = lib.w4a16_moe_experts(ctypes.byref(a), 0x10000000, 1 << 40, None)
    return st, capi.last_error(lib)


@pytest.mark.parametrize("kw,status,msg", [
    (dict(num_experts=0), 24, "num_experts"), (dict(num_experts=1025), 24, "num_experts"), (dict(k=0), 24, "k must"), (dict(k=33), 24, "k must"),
    (dict(hidden=96), 5, "multiples of 64"), (dict(inner=0), 5, "multiples of 64"), (dict(hidden=-64), 5, "multiples of 64"),
    (dict(gate_up_group=32), 10, "group size"), (dict(down_group=0), 10, "group size"), (dict(hidden=320), 7, "group sizes"),
    (dict(inner=192, down_group=128), 7, "group sizes"), (dict(hidden=(1 << 20) + 128), 4, "2^20"), (dict(activation=5), 21, "activation"),
    (dict(tokens=-1), 4, "2^31"), (dict(tokens=1 << 62), 4, "2^31"), (dict(tokens=1 << 24, hidden=1024), 4, "2^31"),
    (dict(x=None), 1, "non-null"), (dict(weights=None), 1, "non-null"), (dict(x=0x100008), 9, "aligned"), (dict(residual=0x900008), 9, "aligned"),
    (dict(experts=0x600002), 9, "aligned"), (dict(y=0x100010), 22, "apart"), (dict(residual=0x800010), 22, "apart"), (dict(y=0x600010), 22, "apart"),
    (dict(y=0x700010), 22, "apart"), (dict(y=0x200000 + 8 * 256 * 128 - 16), 22, "apart"), (dict(y=0x400000 + 8 * 256 * 64 - 16), 22, "apart"),
    (dict(y=0x300000 + 8 * 2 * 256 * 2 - 16), 22, "apart"), (dict(y=0x500000 + 8 * 2 * 256 * 2 - 16), 22, "apart"),
])
def test_refuses(kw, status, msg):
    st, err = call(**kw)
    assert st == status and msg in err, (st, err)


@pytest.mark.parametrize("kw", [dict(), dict(y=0x100000), dict(residual=0x800000), dict(residual=0x100000), dict(k=32, num_experts=1),
                                dict(hidden=1 << 20, inner=64, tokens=1, y=1 << 40, x=1 << 41)])
def test_accepts(kw):
    st, err = call(**kw)
    assert st in DEVICE, (st, err)


def test_no_tokens_is_fine_and_workspaces_are_asked_for():
    lib, n = capi.load(), ctypes.c_uint64(7)
    assert call(tokens=0, x=None, y=None)[0] == 0
    a = args(tokens=0)
    assert lib.w4a16_moe_workspace(ctypes.byref(a), ctypes.byref(n)) == 0 and n.value == 0
    a = args()
    assert lib.w4a16_moe_workspace(ctypes.byref(a), ctypes.byref(n)) in DEVICE
    assert lib.w4a16_moe_workspace(ctypes.byref(a), None) == 1
    assert lib.w4a16_moe_workspace(None, ctypes.byref(n)) == 1 and lib.w4a16_moe_experts(None, None, 0, None) == 1
    a = args(k=0)
    assert lib.w4a16_moe_workspace(ctypes.byref(a), ctypes.byref(n)) == 24


PLAN = r"""
#include <cstdio>
#include <cstdlib>
#include "moe_plan.h"
using namespace w4a16;
// Every routing's tiles fit, and the regions of a workspace follow one another.
int main() {
    unsigned seed = 1;
    auto rnd = [&](int n) { seed = seed * 1664525u + 1013904223u; return (int)((seed >> 8) % (unsigned)n); };
    for (int i = 0; i < 200000; ++i) {
        const int experts = 1 + rnd(rnd(4) ? 64 : 1024), k = 1 + rnd(32), hidden = 64 * (1 + rnd(64)), inner = 64 * (1 + rnd(64));
        const long long tokens = 1 + rnd(rnd(3) ? 40 : 3000), entries = tokens * k;
        const MoePlan p = moe_plan(tokens, k, experts, hidden, inner, 148);
        long long left = entries, tiles = 0;                    // a routing: uneven loads that end with the entries
        int touched = 0;
        for (int e = 0; e < experts && left > 0; ++e) {
            const long long n = e + 1 == experts ? left : rnd((int)(left < 300 ? left + 1 : 300));
            tiles += (n + p.rows - 1) / p.rows;
            touched += n > 0;
            left -= n;
        }
        const bool order = p.tiles_at >= sizeof(MoeHead) && p.order_at >= p.tiles_at + (size_t)p.max_tiles * sizeof(MoeTile) &&
                           p.place_at >= p.order_at + (size_t)entries * 4 && p.rows_at >= p.place_at + (p.grouped ? (size_t)entries * 4 : 0) &&
                           p.inner_at >= p.rows_at + (p.grouped ? (size_t)entries * hidden * 2 : 0) &&
                           p.out_at >= p.inner_at + (size_t)entries * inner * 2 && p.bytes >= p.out_at + (size_t)p.splits * entries * hidden * 4;
        const int stages = (inner / 64 + kMoeChunks - 1) / kMoeChunks;
        const bool splits = p.splits >= 1 && p.splits <= stages && p.splits <= 4 && (!p.grouped || p.splits == 1);
        const bool kinds = !(p.few && p.grouped) && (!p.few || entries <= kMoeFewEntries) && p.rows == (p.grouped ? kMoeGroupedRows : kMoeRows);
        if (tiles > p.max_tiles || !order || !splits || !kinds || p.out_at % 256 || p.inner_at % 256 || p.rows_at % 256) {
            std::printf("experts %d k %d tokens %lld: tiles %lld of %d\n", experts, k, tokens, tiles, p.max_tiles);
            return 1;
        }
    }
    // batches of one size to within a block cover a range
    for (int left = 1; left < 400; ++left) {
        int done = 0, least = 1 << 30, most = 0;
        for (int r = left; r > 0;) {
            const int batches = (r + 9) / 10, n = (r + batches - 1) / batches;
            if (n > 10) return 2;
            least = n < least ? n : least;
            most = n > most ? n : most;
            done += n;
            r -= n;
        }
        if (done != left || most - least > 1) return 3;
    }
    std::puts("ok");
}
"""


def test_the_plan_holds_every_routing(tmp_path):
    import os
    import subprocess
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "w4a16-gemm_b200", "csrc")
    (tmp_path / "plan.cpp").write_text(PLAN)
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Wextra", "-I", csrc, str(tmp_path / "plan.cpp"), "-o", str(tmp_path / "plan")], check=True)
    assert subprocess.run([str(tmp_path / "plan")], capture_output=True, text=True, check=True).stdout == "ok\n"
