"""GPU tests of the root-mean-square norm against its formula in 64 bits on the CPU.

Tolerances, before the first run: the sum of squares is off by at most 64 units of 2^-24 relative (32 in a
thread, 10 across threads, and the squares' own roundings), its root half of that, the reciprocal root and the three
products a few units more: 2^-18 relative in all.  The result is rounded once, half a step of its type
(fp16 2^-11, with subnormals 2^-25 absolute; bf16 2^-8).  The stored sum is one fp32 addition, rounded once: equal.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def check(y, h, weight, eps):
    """h: the rows in 64 bits, on the CPU."""
    want = h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * weight.cpu().double()
    tol = want.abs() * (HALF_STEP[y.dtype] + 2.0 ** -18) + 2.0 ** -25
    assert y.shape == want.shape
    off = (y.cpu().double() - want).abs() / tol
    assert bool((off <= 1).all()), off.max()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("residual", [None, "same", "fp32"])
@pytest.mark.parametrize("shape", [(1, 8), (3, 64), (5, 72), (17, 128), (129, 136), (9, 256), (33, 264), (2, 1024), (7, 2040), (8, 4096),
                                   (3, 8192), (2, 8200), (1, 32768), (0, 64)])
def test_norm(cuda_device, dtype, residual, shape):
    from w4a16_opt import rms_norm
    gen = torch.Generator().manual_seed(shape[1])
    x, w = torch.randn(shape, generator=gen).to(dtype).cuda(), (1 + 0.3 * torch.randn(shape[1], generator=gen)).to(dtype).cuda()
    if residual is None:
        y = rms_norm(x, w, 1e-5)
        check(y, x.cpu().double(), w, 1e-5)
        return
    rtype = dtype if residual == "same" else torch.float32
    r = (5 * torch.randn(shape, generator=gen)).to(rtype).cuda()
    y, h = rms_norm(x, w, 1e-6, residual=r)
    assert h.dtype == rtype and torch.equal(h, (x.float() + r.float()).to(rtype))
    check(y, x.cpu().double() + r.cpu().double(), w, 1e-6)
    # in place: the stream of residuals, and the norm over its input
    x2, r2 = x.clone(), r.clone()
    y2, h2 = rms_norm(x2, w, 1e-6, residual=r2, out=x2, residual_out=r2)
    assert y2.data_ptr() == x2.data_ptr() and h2.data_ptr() == r2.data_ptr()
    assert torch.equal(x2, y) and torch.equal(r2, h)


@pytest.mark.parametrize("dim", [64, 128, 192, 256, 512])
@pytest.mark.parametrize("heads", [1, 3, 8])
def test_heads_of_a_fused_projection(cuda_device, dim, heads):
    from w4a16_opt import rms_norm
    gen = torch.Generator().manual_seed(dim)
    qkv = torch.randn(13, heads + 2, dim, generator=gen).half().cuda()
    w = torch.rand(dim, generator=gen).half().cuda()
    q = qkv[:, 1:heads + 1]
    y = rms_norm(q, w)
    check(y, q.cpu().double(), w, 1e-5)
    before = qkv.clone()
    rms_norm(q, w, out=q)                                # the heads between others, in place
    assert torch.equal(qkv[:, 1:heads + 1], y)
    assert torch.equal(qkv[:, 0], before[:, 0]) and torch.equal(qkv[:, -1], before[:, -1])
    t = qkv.transpose(0, 1)                              # heads first
    check(rms_norm(t, w), t.cpu().double(), w, 1e-5)
    one = rms_norm(q[2, 0], w)
    assert one.shape == (dim,) and torch.equal(one, rms_norm(q, w)[2, 0])


def test_a_broadcast_residual(cuda_device):
    from w4a16_opt import rms_norm
    x, r, w = torch.randn(6, 128).half().cuda(), torch.randn(128).half().cuda(), torch.ones(128).half().cuda()
    y, h = rms_norm(x, w, residual=r.expand(6, 128))
    assert torch.equal(h, x + r)
    check(y, x.cpu().double() + r.cpu().double(), w, 1e-5)


def test_zero_rows_and_eps(cuda_device):
    from w4a16_opt import rms_norm
    w = torch.ones(512).half().cuda()
    assert (rms_norm(torch.zeros(2, 512).half().cuda(), w) == 0).all()
    x = (torch.randn(4, 512) * 1e-3).half().cuda()       # eps beside the mean of squares
    for eps in (1e-6, 1e-2, 1.0):
        check(rms_norm(x, w, eps), x.cpu().double(), w, eps)


@pytest.mark.parametrize("dim", [128, 4096])
def test_large_values_whose_squares_pass_fp32(cuda_device, dim):
    from w4a16_opt import rms_norm
    gen = torch.Generator().manual_seed(1)
    x = (torch.randn(5, dim, generator=gen) * 1e37).bfloat16().cuda()
    x[1] *= 1e-15
    x[2, 1:] = 0
    w = torch.ones(dim).bfloat16().cuda()
    check(rms_norm(x, w), x.cpu().double(), w, 1e-5)


def test_infinities_and_nan_stay_in_their_rows(cuda_device):
    from w4a16_opt import rms_norm
    x = torch.randn(4, 256).half().cuda()
    w = torch.ones(256).half().cuda()
    clean = rms_norm(x, w)
    x[1, 5], x[3, 9] = float("inf"), float("nan")
    y = rms_norm(x, w)
    assert torch.equal(y[0], clean[0]) and torch.equal(y[2], clean[2])
    assert y[1, 5].isnan() and (y[1, :5] == 0).all() and y[3].isnan().all()


def test_captured(cuda_device):
    from w4a16_opt import rms_norm
    x, r, w = torch.randn(8, 4096).half().cuda(), torch.randn(8, 4096).half().cuda(), torch.rand(4096).half().cuda()
    graph = torch.cuda.CUDAGraph()
    rms_norm(x, w, residual=r)
    with torch.cuda.graph(graph):
        y, h = rms_norm(x, w, residual=r)
    x.copy_(torch.randn(8, 4096))
    graph.replay()
    y2, h2 = rms_norm(x, w, residual=r)
    assert torch.equal(y, y2) and torch.equal(h, h2)


def test_refusals(cuda_device):
    from w4a16_opt import rms_norm
    x, w = torch.randn(4, 64).half().cuda(), torch.ones(64).half().cuda()

    def refused(match, *args, **kw):
        with pytest.raises(RuntimeError, match=match):
            rms_norm(*args, **kw)

    refused("fp16 or bf16", x.float(), w.float())
    refused("weight must be", x, w.bfloat16())
    refused("weight must be", x, w[:32])
    refused("one to three dimensions", x.view(1, 1, 4, 64), w)
    refused("last dimension must be contiguous", torch.randn(64, 64).half().cuda().t(), w)
    refused("multiple of 8", x[:, :60].contiguous(), w[:60].contiguous())
    refused("multiple of 8", torch.zeros(1, 32776).half().cuda(), torch.zeros(32776).half().cuda())
    refused("aligned", torch.randn(4, 72).half().cuda()[:, 1:65], w)
    refused("aligned", torch.randn(4, 68).half().cuda()[:, :64], w)
    refused("eps", x, w, -1.0)
    refused("eps", x, w, float("nan"))
    refused("residual_out needs", x, w, residual_out=x.clone())
    refused("of x's shape", x, w, residual=x[:2])
    refused("x's dtype or fp32", x, w, residual=x.bfloat16())
    refused("residual_out must have", x, w, residual=x.float(), residual_out=x.clone())
    refused("out must have", x, w, out=x.bfloat16())
    refused("very view or apart", x, w, residual=x.clone(), out=x, residual_out=x)
    both = torch.randn(5, 64).half().cuda()
    refused("very view or apart", both[:4], w, out=both[1:])
    refused("must not overlap one another", x, w, out=torch.zeros(64).half().cuda().expand(4, 64))
    refused("very view or apart", w.view(1, 64), w, out=w.view(1, 64))
