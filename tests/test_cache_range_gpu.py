"""GPU test of attention with bf16 queries at the ends of the type's range: the scores are finite in fp32, and
so must be what is made of them."""
import math

import pytest
import torch

from oracle import cache_oracle as oracle

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu(cuda_device):
    yield
    import w4a16_opt
    assert w4a16_opt.device_status(reset=True) == 0


@pytest.mark.parametrize("q_len", [1, 20, 200])
@pytest.mark.parametrize("d,g", [(64, 64), (128, 64), (128, 128)])
@pytest.mark.parametrize("dtype,size,key,rest", [
    ("fp16", 100.0, 100.0, 1.0), ("fp16", 3000.0, 1000.0, 1.0), ("fp16", 20000.0, 20000.0, 10.0), ("fp16", 60000.0, 50000.0, 10.0),
    ("bf16", 1e30, 1e-2, 1e-4), ("bf16", 1e36, 1e-2, 1e-4), ("bf16", 1e37, 1e-2, 1e-4), ("bf16", 3e38, 1e-2, 1e-4)])
def test_scores_that_leave_one_token(dtype, size, key, rest, d, g, q_len):
    """Scores from 10^4 to nearly 2^127, and one token that every query sees and prefers: its values are the answer.
    The maximum's own weight is one, whatever a score's rounding is."""
    import w4a16_opt as w
    gen = torch.Generator().manual_seed(d + q_len)
    type_ = {"fp16": torch.float16, "bf16": torch.bfloat16}[dtype]
    n, hk, hq, page = 1000, 2, 8, 64
    best = 700                                        # below every query's position
    u = torch.where(torch.rand(d, generator=gen) < 0.5, -1.0, 1.0)
    k = torch.randn(n, hk, d, generator=gen) * rest
    k[best] = u * key
    v = torch.randn(n, hk, d, generator=gen)
    q = (u * (1 - 0.3 * torch.rand(q_len, hq, d, generator=gen)) * size).to(type_)
    assert q.isfinite().all()
    cache = w.Int4KVCache(-(-n // page), hk, d, page, g)
    slots = torch.arange(n).cuda()
    w.cache_append(cache, k.to(type_).cuda(), v.to(type_).cuda(), slots)
    keys, vals = oracle.read_slots(cache.data, d, page, g, slots)
    s = torch.einsum("qhd,nhd->qhn", q.cuda().double(), keys.repeat_interleave(hq // hk, 1)) / math.sqrt(d)
    top = s.topk(2, -1).values
    assert s.abs().max() < 2.0 ** 126 and (s.argmax(-1) == best).all() and (top[..., 0] - top[..., 1]).min() > 200
    out, lse = w.cache_attention(q.cuda(), cache, torch.arange(-(-n // page), dtype=torch.int32).cuda()[None],
                                 torch.tensor([n], dtype=torch.int32).cuda(),
                                 cu_q=torch.tensor([0, q_len], dtype=torch.int32).cuda(), max_q=q_len, return_lse=True)
    want = vals[best].repeat_interleave(hq // hk, 0)
    # rounded to fp16 as an operand at most, as its weight is, and to the output's type
    tol = want.abs() * (2.0 ** -8 if dtype == "bf16" else 2.0 ** -11) + want.abs().amax(-1, keepdim=True) * 2 * 2.0 ** -11
    assert ((out.double() - want).abs() <= tol).all()
    # keys rounded to fp16 (2^-11 each), products and sums in fp32
    assert ((lse.double() - top[..., 0]).abs() <= top[..., 0] * 2.0 ** -10).all()


@pytest.mark.parametrize("q_len", [1, 20, 200])
@pytest.mark.parametrize("size", [1e-30, 1e-38])
def test_queries_near_zero(size, q_len):
    """Every score is as good as zero: the mean of the values."""
    import w4a16_opt as w
    gen = torch.Generator().manual_seed(q_len)
    n, d, page = 300, 128, 64
    k, v = torch.randn(n, 1, d, generator=gen).half().cuda(), torch.randn(n, 1, d, generator=gen).half().cuda()
    q = (torch.randn(q_len, 4, d, generator=gen) * size).bfloat16().cuda()
    cache = w.Int4KVCache(-(-n // page), 1, d, page)
    slots = torch.arange(n).cuda()
    w.cache_append(cache, k, v, slots)
    vals = oracle.read_slots(cache.data, d, page, d, slots)[1]
    out = w.cache_attention(q, cache, torch.arange(-(-n // page), dtype=torch.int32).cuda()[None],
                            torch.tensor([n], dtype=torch.int32).cuda(), causal=False,
                            cu_q=torch.tensor([0, q_len], dtype=torch.int32).cuda(), max_q=q_len)
    want = vals.mean(0)[0]
    tol = 2.0 ** -8 * want.abs() + vals.abs().mean() * (2 * 2.0 ** -11 + 2.0 ** -12)
    assert ((out.double() - want).abs() <= tol).all()
