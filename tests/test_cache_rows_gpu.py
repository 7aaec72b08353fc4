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


def padded(p, before, after):
    """The problem's queries with rows of NaN around them, and cu_q to match."""
    pad = lambda n: torch.full((n, *p.q.shape[1:]), math.nan, dtype=p.dtype, device="cuda")      # noqa: E731
    return torch.cat((pad(before), p.q, pad(after))), p.cu + before


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("before,after", [(0, 3), (2, 0), (5, 1000)])
@pytest.mark.parametrize("hq,hk,d,lens,q_lens", [
    (4, 2, 64, [70, 0, 9], [1, 1, 1]),            # few rows, one block a row of the join
    (32, 8, 128, [9000], [1]),                    # few rows, many parts
    (8, 1, 128, [50, 600, 0], [2, 3, 1]),
    (8, 2, 128, [400, 40, 7], [30, 1, 7]),        # up to 128 rows
    (8, 2, 128, [9000], [30]),                    # the same, split
    (4, 2, 64, [400, 300], [200, 300]),           # more
])
def test_rows_of_no_sequence_are_zeros(hq, hk, d, lens, q_lens, before, after, dtype):
    import w4a16_opt as w
    p = Problem(lens, q_lens, hq, hk, d, d, 32, dtype, seed=after)
    q, cu = padded(p, before, after)
    want, want_lse = w.cache_attention(p.q, p.cache, p.table, p.seq_lens, cu_q=p.cu, max_q=max(q_lens), return_lse=True)
    out, lse = w.cache_attention(q, p.cache, p.table, p.seq_lens, cu_q=cu, max_q=max(q_lens), return_lse=True,
                                 out=torch.full_like(q, math.nan))
    inside = slice(before, before + len(p.q))
    if max(q_lens) * (hq // hk) <= 32:           # (longer ones may be split otherwise)
        assert torch.equal(out[inside], want) and torch.equal(lse[inside], want_lse)
    p.check(out[inside], lse[inside])
    for rows in (slice(0, before), slice(before + len(p.q), None)):
        assert not out[rows].any() and (lse[rows] == -math.inf).all()
    assert torch.equal(w.cache_attention(q, p.cache, p.table, p.seq_lens, cu_q=cu, max_q=max(q_lens)), out)


@pytest.mark.parametrize("hq,hk,d,q_lens,max_q", [(4, 2, 64, [5, 1, 9], 3), (8, 2, 128, [40, 7, 20], 10),
                                                  (8, 2, 128, [300, 1, 170], 100)])
def test_queries_past_max_q_are_zeros(hq, hk, d, q_lens, max_q):
    p = Problem([400, 0, 333], q_lens, hq, hk, d, d, 32, seed=max_q)
    out, lse = p.run(return_lse=True, out=torch.full_like(p.q, math.nan), max_q=max_q)
    at = 0
    for t in q_lens:
        assert not out[at + max_q:at + t].any() and (lse[at + max_q:at + t] == -math.inf).all()
        assert torch.isfinite(out[at:at + t]).all()
        at += t


@pytest.mark.parametrize("most", [1, 40])
def test_a_captured_step_of_fixed_size_serves_fewer_queries(most):
    """Queries and lengths are read on the device: a graph of `8 most` rows, replayed for fewer."""
    import w4a16_opt as w
    p = Problem([300] * 8, [most] * 8, 4, 2, 64, 64, 32, seed=most)
    cu, lens = p.cu.clone(), p.seq_lens.clone()
    out = torch.empty_like(p.q)
    kw = dict(cu_q=cu, max_q=most, out=out)
    w.cache_attention(p.q, p.cache, p.table, lens, **kw)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w.cache_attention(p.q, p.cache, p.table, lens, **kw)
    for used in (8, 3, 0):
        now = [most] * used + [0] * (8 - used)
        cu.copy_(torch.tensor([0] + now).cumsum(0).int())
        out.fill_(math.nan)
        graph.replay()
        q = Problem.__new__(Problem)
        q.__dict__.update(p.__dict__)
        q.q_lens = now
        q.check(out)
        assert not out[used * most:].any()


def test_calls_without_sequences_or_queries_give_zeros():
    import w4a16_opt as w
    p = Problem([50, 60], [2, 3], 4, 2, 64, 64, 16)
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    for kw in (dict(page_table=p.table[:0], seq_lens=p.seq_lens[:0], cu_q=none, max_q=3),
               dict(page_table=p.table, seq_lens=p.seq_lens, cu_q=p.cu * 0, max_q=0)):
        out, lse = w.cache_attention(p.q, p.cache, return_lse=True, out=torch.full_like(p.q, math.nan), **kw)
        assert not out.any() and (lse == -math.inf).all()
        assert not w.cache_attention(p.q, p.cache, **kw).any()
