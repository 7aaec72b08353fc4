"""GPU tests of the forms that an attention call may take: up to 128 rows a (sequence, key head), where the
prompt kernel's halves take alternate tiles, blocks of rows split over several CTAs, and the joins of the
decode kernel's parts.  Tolerances are those of test_cache_gpu."""
import math

import pytest
import torch

from test_cache_gpu import Problem

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu(cuda_device):
    yield
    import w4a16_opt
    assert w4a16_opt.device_status(reset=True) == 0


# ------------------------------------------------------------------------------ 33 to 128 rows

@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 1), (True, 64), (True, 100), (False, 90), (True, 5000)])
@pytest.mark.parametrize("d,g,dtype", [(128, 128, "fp16"), (128, 64, "bf16"), (64, 64, "fp16"), (64, 64, "bf16")])
def test_masks_on_alternate_tiles(d, g, dtype, causal, window):
    p = Problem([70, 513, 150, 1300], [9, 20, 32, 12], 8, 2, d, g, 16, dtype, seed=window)
    out, lse = p.run(causal=causal, window=window, return_lse=True)
    p.check(out, lse, causal=causal, window=window)


@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 7), (False, 9)])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_rows_that_see_nothing_on_alternate_tiles(dtype, causal, window):
    p = Problem([0, 1, 70, 300], [20, 9, 40, 3], 4, 2, 64, 64, 16, dtype)
    out, lse = p.run(causal=causal, window=window, return_lse=True, out=torch.full_like(p.q, math.nan))
    p.check(out, lse, causal=causal, window=window)


@pytest.mark.parametrize("gain,scale", [(0.0, None), (40.0, None), (1.0, 0.0), (1.0, -0.3), (3000.0, 1e-4), (1e-4, 300.0)])
def test_scores_of_every_size_on_alternate_tiles(gain, scale):
    p = Problem([400, 1030], [16, 16], 8, 2, 128, 128, 64, gain=gain, seed=3)
    out, lse = p.run(scale=scale, return_lse=True)
    p.check(out, lse, scale=scale)


@pytest.mark.parametrize("rows", [33, 127, 128, 129])
@pytest.mark.parametrize("length", [129, 256, 300])
def test_rows_about_the_limits(rows, length):
    """One key head, one query head: as many rows as queries."""
    p = Problem([length], [rows], 1, 1, 128, 128, 64, seed=rows)
    out, lse = p.run(return_lse=True)
    p.check(out, lse)


def test_a_query_that_is_not_finite_on_alternate_tiles():
    p = Problem([400, 200], [20, 20], 4, 2, 128, 128, 64)
    want = p.run()
    q = p.q.clone()
    q[0, 1] = math.nan
    got = p.run(q)
    assert torch.isnan(got[0, 1]).all()
    got[0, 1] = want[0, 1]
    assert torch.equal(got, want)


# ------------------------------------------------------------------------------ row blocks split over CTAs

@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 6000), (False, 3000), (False, 0)])
@pytest.mark.parametrize("hq,hk,d,g,lens,q_lens", [
    (8, 1, 128, 128, [20000], [64]), (4, 1, 128, 64, [20000], [20]), (4, 1, 64, 64, [17000, 0, 100], [40, 20, 30]),
    (2, 1, 64, 64, [9000, 9000], [64, 200])])
def test_split_blocks(hq, hk, d, g, lens, q_lens, causal, window, dtype):
    p = Problem(lens, q_lens, hq, hk, d, g, 128, dtype, seed=d + window)
    out, lse = p.run(causal=causal, window=window, return_lse=True, out=torch.full_like(p.q, math.nan))
    p.check(out, lse, causal=causal, window=window)
    assert torch.equal(p.run(causal=causal, window=window), out)


# ------------------------------------------------------------------------------ parts of the decode kernel

@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("hq,hk,q_len", [(4, 1, 1), (8, 8, 1), (3, 1, 3)])
@pytest.mark.parametrize("window", [0, 11000])
def test_long_sequences_with_narrow_heads(hq, hk, q_len, window, dtype):
    p = Problem([23000], [q_len], hq, hk, 64, 64, 64, dtype, seed=hq)
    out, lse = p.run(window=window, return_lse=True)
    p.check(out, lse, window=window)
