"""GPU tests of the norm's rows that share a warp (dim up to 128: four or two of them), where some need their squares summed again
at another scale and their neighbours do not.  Tolerances as in test_norm_gpu, derived there."""
import pytest
import torch

from test_norm_gpu import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pattern", ["alternate", "first", "last", "pairs"])
@pytest.mark.parametrize("kind", ["bf16", "bf16 + bf16", "bf16 + fp32", "fp16 + fp32"])
@pytest.mark.parametrize("rows,dim", [(37, 8), (64, 40), (66, 64), (35, 72), (34, 128), (20, 136), (9, 256), (6, 1024)])
def test_large_rows_beside_ordinary_ones(cuda_device, rows, dim, kind, pattern):
    from w4a16_opt import rms_norm
    gen = torch.Generator().manual_seed(rows + dim)
    dtype = torch.float16 if kind.startswith("fp16") else torch.bfloat16
    rtype = torch.float32 if kind.endswith("fp32") else dtype
    x = torch.randn(rows, dim, generator=gen).to(dtype).cuda()
    r = torch.randn(rows, dim, generator=gen).to(rtype).cuda() if "+" in kind else None
    w = (1 + 0.3 * torch.randn(dim, generator=gen)).to(dtype).cuda()
    at = torch.arange(rows)
    large = {"alternate": at % 2 == 1, "first": at % 4 == 0, "last": at == rows - 1, "pairs": at % 4 > 1}[pattern].cuda()
    norm = lambda x, r: (rms_norm(x, w), x) if r is None else rms_norm(x, w, residual=r)      # noqa: E731
    clean, h_clean = norm(x, r)
    target = x if r is None else r
    target[large] = (target[large].float() * 1e37).to(target.dtype)
    y, h = norm(x, r)
    assert torch.equal(y[~large], clean[~large]) and torch.equal(h[~large], h_clean[~large])
    full = x.cpu().double() if r is None else x.cpu().double() + r.cpu().double()
    check(y, full, w, 1e-5)


# the means of squares leave fp32 where eps is at the ends of its range too: rows from subnormals to near the largest value, each its own size
@pytest.mark.parametrize("eps", [0.0, 1e-45, 1e-38, 1e-30, 1e-19, 1.0, 1e30, 1e38, 3e38])
@pytest.mark.parametrize("residual", [None, "same", "fp32"])
@pytest.mark.parametrize("dim", [8, 64, 128, 264, 2048, 16640])
def test_rows_of_every_size_with_every_eps(cuda_device, dim, residual, eps):
    from w4a16_opt import rms_norm
    gen = torch.Generator().manual_seed(dim)
    sizes = torch.logspace(-39, 37, 39).double()[:, None]
    x = (torch.randn(39, dim, generator=gen).double() * sizes).bfloat16().cuda()
    w = (1 + 0.3 * torch.randn(dim, generator=gen)).bfloat16().cuda()
    if residual is None:
        y, h = rms_norm(x, w, eps), x.cpu().double()
    else:
        r = (torch.randn(39, dim, generator=gen).double() * sizes).to(torch.bfloat16 if residual == "same" else torch.float32).cuda()
        y, _ = rms_norm(x, w, eps, residual=r)
        h = (x.float() + r.float()).cpu().double()        # the sum itself is one fp32 addition
    eps = torch.tensor(eps, dtype=torch.float32).double().item()      # as the entry point takes it
    want = h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * w.cpu().double()
    # results below bf16's normal numbers: half a step of its subnormals, 2^-134, and fp32's own steps on the way there (2^-149 of a
    # scaled value, times a scale of at most 2^19 and a weight of at most 2^2: 2^-128)
    tol = want.abs() * (2.0 ** -8 + 2.0 ** -17) + 2.0 ** -127
    off = (y.cpu().double() - want).abs() / tol
    assert bool((off <= 1).all()), (off.max(), off.max(1).values)


@pytest.mark.parametrize("dim", [8, 64, 128])
def test_infinities_and_nan_beside_ordinary_rows(cuda_device, dim):
    from w4a16_opt import rms_norm
    gen = torch.Generator().manual_seed(dim)
    x, w = torch.randn(11, dim, generator=gen).half().cuda(), torch.ones(dim).half().cuda()
    clean = rms_norm(x, w)
    x[1, 5], x[6, 2] = float("inf"), float("nan")
    y = rms_norm(x, w)
    keep = [t for t in range(11) if t not in (1, 6)]
    assert torch.equal(y[keep], clean[keep])
    assert y[1, 5].isnan() and (y[1, :5] == 0).all() and y[6].isnan().all()


@pytest.mark.parametrize("large", [False, True])
@pytest.mark.parametrize("rows,dim", [(9, 64), (5, 136), (4, 2048), (3, 8200), (2, 20480)])
def test_outputs_in_each_others_inputs(cuda_device, rows, dim, large):
    """The norm over the residual's place and the sum over x's; one tensor as both inputs and the sum."""
    from w4a16_opt import rms_norm
    gen = torch.Generator().manual_seed(dim)
    draw = lambda: torch.randn(rows, dim, generator=gen).bfloat16().cuda()      # noqa: E731
    x, r, w = draw(), draw(), draw()[0]
    if large:
        r[::2] *= 1e37
    y, h = rms_norm(x, w, residual=r)
    x2, r2 = x.clone(), r.clone()
    rms_norm(x2, w, residual=r2, out=r2, residual_out=x2)
    assert torch.equal(r2, y) and torch.equal(x2, h)
    y, h = rms_norm(r, w, residual=r)
    r2 = r.clone()
    y2, _ = rms_norm(r2, w, residual=r2, residual_out=r2)
    assert torch.equal(y2, y) and torch.equal(r2, h)
