"""GPU tests of the expert router against its definition in 64 bits on the CPU.

Tolerances, before the first run: the weights' exponentials are good to 2 units of 2^-23 (expf) and their sums of up
to 1024 terms to 40 units (32 in a lane, 5 across lanes), the division to half a unit: 2^-17 relative; weights
below the smallest normal number may be 0 (2^-126 absolute).  The choice of experts is exact.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def expected(logits, k, renormalize):
    l = logits.detach().cpu().double()
    weights, experts = torch.zeros(l.shape[0], k, dtype=torch.float64), torch.full((l.shape[0], k), -1, dtype=torch.int32)
    for t, row in enumerate(l.tolist()):
        row = [-math.inf if math.isnan(v) else v for v in row]
        best = sorted((e for e in range(len(row)) if row[e] > -math.inf), key=lambda e: (-row[e], e))
        if not best:
            continue
        top = row[best[0]]
        p = {e: 1.0 if row[e] == top else math.exp(row[e] - top) for e in best}
        total = sum(p[e] for e in (best[:k] if renormalize else best))
        for j, e in enumerate(best[:k]):
            experts[t, j], weights[t, j] = e, p[e] / total
    return weights, experts


def check(logits, k, renormalize=True):
    from w4a16_opt import moe_route
    w, e = moe_route(logits, k, renormalize=renormalize)
    ww, ee = expected(logits, k, renormalize)
    assert w.dtype == torch.float32 and e.dtype == torch.int32
    assert torch.equal(e.cpu(), ee)
    assert bool(((w.cpu().double() - ww).abs() <= ww * 2.0 ** -17 + 2.0 ** -126).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("tokens,experts,k", [(1, 1, 1), (1, 8, 2), (5, 7, 7), (9, 33, 4), (16, 64, 6), (130, 60, 4), (3, 65, 1), (17, 128, 8),
                                              (6, 256, 8), (4, 257, 32), (2, 1000, 31), (3, 1024, 32), (0, 8, 2)])
def test_route(cuda_device, dtype, renormalize, tokens, experts, k):
    gen = torch.Generator().manual_seed(experts)
    check((3 * torch.randn(tokens, experts, generator=gen)).to(dtype).cuda(), k, renormalize)


def test_ties_go_to_the_lowest_index(cuda_device):
    check(torch.zeros(3, 100).cuda(), 8)
    check(torch.randint(-2, 3, (40, 130), generator=torch.Generator().manual_seed(0)).float().cuda(), 16, False)
    signed = torch.zeros(2, 40)
    signed[0, ::2], signed[1, 1::2] = -0.0, -0.0                        # zeros of both signs are equal
    check(signed.cuda(), 5)


def test_masked_experts(cuda_device):
    gen = torch.Generator().manual_seed(3)
    l = torch.randn(50, 70, generator=gen)
    l[torch.rand(50, 70, generator=gen) < 0.9] = -math.inf
    l[0] = -math.inf                                                    # nothing is left
    l[1, :] = -math.inf
    l[1, 69] = -2.0                                                     # one is
    l[2, ::3] = math.nan
    l[3] = torch.finfo(torch.float32).min                               # the lowest value is not a mask
    for renormalize in (True, False):
        check(l.cuda(), 12, renormalize)
    check(l.bfloat16().cuda(), 12)


def test_infinite_and_distant_logits(cuda_device):
    l = torch.tensor([[math.inf, 0.0, math.inf, -5.0], [1e38, -1e38, 3e38, 0.0], [-3e38, -3.2e38, -3.4e38, -math.inf], [200.0, 100.0, 0.0, -100.0]])
    for k in (1, 2, 4):
        check(l.cuda(), k, True)
        check(l.cuda(), k, False)


def test_rows_of_a_wider_matrix(cuda_device):
    wide = torch.randn(20, 100, generator=torch.Generator().manual_seed(4)).cuda()
    check(wide[:, 3:40], 5)
    check(wide[::3, :33], 5)
    check(wide[0].expand(4, 100), 5)


def test_captured(cuda_device):
    from w4a16_opt import moe_route
    l = torch.randn(16, 128, device="cuda")
    moe_route(l, 8)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w, e = moe_route(l, 8)
    l.copy_(torch.randn(16, 128))
    graph.replay()
    w2, e2 = moe_route(l, 8)
    assert torch.equal(w, w2) and torch.equal(e, e2)


def test_refusals(cuda_device):
    from w4a16_opt import moe_route
    l = torch.randn(4, 16, device="cuda")
    for bad, k, match in ((l, 0, "k must be"), (l, 17, "k must be"), (l.double(), 2, "fp16, bf16 or fp32"), (l[0], 2, "tokens, experts"),
                          (l.t(), 2, "last dimension"), (l.cpu(), 2, "CUDA"), (torch.zeros(2, 1025, device="cuda"), 2, "num_experts"),
                          (torch.zeros(2, 100, device="cuda"), 33, "k must be"), (torch.zeros(2, 0, device="cuda"), 1, "k must be")):
        with pytest.raises(RuntimeError, match=match):
            moe_route(bad, k)
