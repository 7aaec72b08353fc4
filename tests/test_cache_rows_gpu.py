"""GPU tests of attention calls whose query rows are not all answered: sequences with more queries than
max_q, and rows that belong to no sequence."""
import math

import pytest
import torch

from oracle import cache_oracle as oracle
from test_cache_gpu import Problem

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu(cuda_device):
    yield
    import w4a16_opt
    assert w4a16_opt.device_status(reset=True) == 0


def first_rows(p, out, lse, most, **mask):
    """The first `most` queries of each sequence, checked with the tolerances of Problem.check."""
    q = Problem.__new__(Problem)
    q.__dict__.update(p.__dict__)
    at = 0
    for b, (n, t) in enumerate(zip(p.lens, p.q_lens)):
        # the oracle's answer to all of the sequence's queries; those past `most` are given to the check as they should be
        k, v = oracle.read_slots(p.data, p.d, p.page, p.g, p.slots[b])
        ref, rlse, _, _ = oracle.attention(p.q[at:at + t].double(), k, v, **mask)
        o, s = out[at:at + t].clone(), lse[at:at + t].clone()
        o[most:], s[most:] = ref[most:].to(out.dtype), rlse[most:].float()
        q.lens, q.q_lens, q.slots, q.q = [n], [t], [p.slots[b]], p.q[at:at + t]
        q.check(o, s, **mask)
        at += t


@pytest.mark.parametrize("hq,hk,d,q_lens,max_q", [
    (4, 2, 64, [5, 1, 9], 3),              # few rows
    (8, 2, 128, [40, 7, 20], 10),          # up to 128 rows
    (8, 2, 128, [300, 1, 170], 100),       # more
])
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 50), (False, 0)])
def test_positions_go_by_all_queries_of_a_sequence(hq, hk, d, q_lens, max_q, causal, window):
    """max_q below a sequence's queries: the first max_q are answered, at their own positions."""
    p = Problem([400, 37, 333], q_lens, hq, hk, d, d, 32, seed=max_q)
    out = torch.full_like(p.q, math.nan)
    out, lse = p.run(causal=causal, window=window, return_lse=True, out=out, max_q=max_q)
    first_rows(p, out, lse, max_q, causal=causal, window=window)
