"""GPU tests of the product with an epilogue against its formula in 64 bits on the CPU.

Tolerances, before the first run.  A sum z of K products in fp32 by tensor cores, 16 a step, is off by at most
(K / 16 + 8) 2^-22 S, S = sum |x w| (each step and each join of partial sums loses at most two units of 2^-23 of
what it adds to).  Activations have slope at most 1.13 and are themselves good to 2^-18 relative in fp32 (fast exp and
division, a few units for the arguments here); the result is rounded to fp16 once (2^-11 relative, 2^-25
absolute among its subnormals).
"""
import numpy as np
import pytest
import torch

from helpers import make_workload, make_problem
from oracle import w4a16_oracle as oracle

pytestmark = pytest.mark.gpu

# both kernels, split and whole column groups, one block of columns, ragged tiles of tokens and channels
SHAPES = [(1, 16, 64, 64), (3, 48, 192, 64), (8, 512, 1024, 128), (5, 4096, 1152, 128), (16, 272, 640, 128), (11, 4112, 256, 64),
          (17, 272, 448, 64), (77, 416, 1152, 128), (130, 128, 256, 128), (300, 1040, 512, 64)]
EPILOGUES = [
    dict(activation="relu"), dict(activation="silu", bias=True), dict(activation="gelu", bias=True, residual=True),
    dict(activation="gelu_tanh", residual=True), dict(residual=True), dict(bias=True),
    dict(activation="silu", gated=True), dict(activation="gelu", gated=True, bias=True), dict(gated=True, residual=True),
    dict(activation="gelu_tanh", gated=True, bias=True, residual=True), dict(activation="relu", gated=True, residual=True),
]


def act64(z, name):
    t = torch.as_tensor(z)
    if name == "relu":
        return t.clamp_min(0)
    if name == "silu":
        return t * torch.sigmoid(t)
    if name == "gelu":
        return t * torch.special.ndtr(t)
    if name == "gelu_tanh":
        return 0.5 * t * (1 + torch.tanh((2 / np.pi) ** 0.5 * (t + 0.044715 * t ** 3)))
    return t


def expected(x, q, scales, G, activation=None, gated=False, bias=None, residual=None, fp32_scale=False):
    """(y in 64 bits, what it may be off by)."""
    W = torch.from_numpy(oracle.dequantize_w4(q.cpu().numpy(), scales.cpu().numpy(), G)).double()
    x64, K = x.cpu().double(), x.shape[1]
    z, S = x64 @ W.t(), x64.abs() @ W.abs().t()
    dz = (K / 16 + 8) * 2.0 ** -22 * S + (2.0 ** -11 * S if fp32_scale else 0)     # unrounded weights
    if bias is not None:
        z = z + bias.cpu().double()
        dz = dz + 2.0 ** -23 * z.abs()
    if gated:
        zz, dd = z.view(z.shape[0], -1, 2, 8), dz.view(z.shape[0], -1, 2, 8)
        flat = lambda t: t.reshape(z.shape[0], -1)      # noqa: E731
        zg, zu, dg, du = flat(zz[:, :, 0]), flat(zz[:, :, 1]), flat(dd[:, :, 0]), flat(dd[:, :, 1])
        a = act64(zg, activation)
        y, d = a * zu, 1.13 * dg * (zu.abs() + du) + a.abs() * du + 2.0 ** -18 * (a * zu).abs()
    else:
        y = act64(z, activation)
        d = 1.13 * dz + 2.0 ** -18 * y.abs()
    if residual is not None:
        y = y + residual.cpu().double()
    return y, d * 1.001 + 2.0 ** -11 * (y.abs() + d) + 2.0 ** -25


def operands(M, N, K, G, seed, activation=None, gated=False, bias=False, residual=False):
    x, q, scales, Wp = make_problem(M, N, K, G, seed=seed)
    gen = torch.Generator().manual_seed(seed + 1)
    cols = N // 2 if gated else N
    b = torch.randn(N, generator=gen).half().cuda() if bias else None
    r = (2 * torch.randn(M, cols, generator=gen)).half().cuda() if residual else None
    return x, q, scales, Wp, b, r


def check(y, ref, tol):
    assert y.dtype == torch.float16 and y.shape == ref.shape
    off = (y.cpu().double() - ref).abs() / tol
    assert bool((off <= 1).all()), off.max()


@pytest.mark.parametrize("epilogue", EPILOGUES, ids=lambda e: "-".join(str(v) if isinstance(v, str) else k for k, v in e.items()))
@pytest.mark.parametrize("M,N,K,G", SHAPES)
def test_linear(cuda_device, M, N, K, G, epilogue):
    from w4a16_opt import w4a16_linear
    x, q, scales, Wp, b, r = operands(M, N, K, G, M + N + K, **epilogue)
    act, gated = epilogue.get("activation"), epilogue.get("gated", False)
    y = w4a16_linear(Wp, x, scales, bias=b, activation=act, gated=gated, residual=r)
    check(y, *expected(x, q, scales, G, act, gated, b, r))
    if r is not None:       # in place
        out = w4a16_linear(Wp, x, scales, bias=b, activation=act, gated=gated, residual=r, out=r)
        assert out is r or out.data_ptr() == r.data_ptr()
        assert torch.equal(r, y)


@pytest.mark.parametrize("variant", [1, 2, 3, 4])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("M", [1, 31, 65, 200, 257])
def test_every_token_tile(cuda_device, variant, gated, M):
    from w4a16_opt import w4a16_linear
    x, q, scales, Wp, b, r = operands(M, 176, 320, 64, 3 * M, gated=gated, bias=True, residual=True)
    y = w4a16_linear(Wp, x, scales, bias=b, activation="silu", gated=gated, residual=r, variant=variant)
    check(y, *expected(x, q, scales, 64, "silu", gated, b, r))


@pytest.mark.parametrize("M,N,K,G", [(1, 4096, 1024, 128), (8, 272, 448, 64)])
@pytest.mark.parametrize("gated", [False, True])
def test_fp32_scale(cuda_device, M, N, K, G, gated):
    from w4a16_opt import w4a16_linear
    x, q, scales, Wp, b, r = operands(M, N, K, G, N, gated=gated, bias=True, residual=True)
    y = w4a16_linear(Wp, x, scales, bias=b, activation="gelu", gated=gated, residual=r, fp32_scale=True)
    check(y, *expected(x, q, scales, G, "gelu", gated, b, r, fp32_scale=True))


@pytest.mark.parametrize("M,N,K,G", SHAPES)
def test_without_an_epilogue_it_is_the_gemm(cuda_device, M, N, K, G):
    from w4a16_opt import w4a16_gemm, w4a16_linear
    x, q, scales, Wp = make_workload(M, N, K, G, seed=7)
    assert torch.equal(w4a16_linear(Wp, x, scales), w4a16_gemm(Wp, x, scales))


@pytest.mark.parametrize("M", [2, 40])
def test_a_plain_epilogue_of_nothing_rounds_as_the_gemm_does(cuda_device, M):
    """relu of the sums is relu of the rounded sums; a residual of zeros changes nothing."""
    from w4a16_opt import w4a16_gemm, w4a16_linear
    x, q, scales, Wp = make_workload(M, 1040, 1024, 128, seed=8)
    y = w4a16_gemm(Wp, x, scales)
    assert torch.equal(w4a16_linear(Wp, x, scales, activation="relu"), y.clamp_min(0))
    assert torch.equal(w4a16_linear(Wp, x, scales, residual=torch.zeros_like(y)), y)


@pytest.mark.parametrize("M", [1, 33])
def test_infinities_and_nan_stay_in_their_rows_and_columns(cuda_device, M):
    from w4a16_opt import w4a16_linear
    x, q, scales, Wp, b, r = operands(M, 64, 128, 64, 5, bias=True, residual=True)
    clean = w4a16_linear(Wp, x, scales, bias=b, activation="silu", residual=r)
    b2, r2 = b.clone(), r.clone()
    b2[3], b2[20], r2[0, 40] = float("nan"), float("inf"), float("-inf")
    y = w4a16_linear(Wp, x, scales, bias=b2, activation="silu", residual=r2)
    assert y[:, 3].isnan().all() and (y[:, 20] == float("inf")).all() and y[0, 40] == float("-inf")
    keep = torch.ones_like(y, dtype=torch.bool)
    keep[:, 3], keep[:, 20], keep[0, 40] = False, False, False
    assert torch.equal(y[keep], clean[keep])
    x2 = x.clone()
    x2[-1, 7] = float("nan")
    y = w4a16_linear(Wp, x2, scales, bias=b, activation="relu", residual=r)
    assert y[-1].isnan().all()
    assert torch.equal(y[:-1], w4a16_linear(Wp, x, scales, bias=b, activation="relu", residual=r)[:-1])
    big = torch.full((64,), 60000.0, dtype=torch.float16, device="cuda")
    assert (w4a16_linear(Wp, x, scales, bias=big, residual=torch.full_like(r, 60000.0)) == float("inf")).all()
    assert (w4a16_linear(Wp, x, scales, bias=-big, activation="silu") == 0).all()


@pytest.mark.parametrize("M", [4, 50])
def test_captured_on_a_stream_of_its_own(cuda_device, M):
    from w4a16_opt import w4a16_linear
    x, q, scales, Wp, b, r = operands(M, 4096, 1024, 128, 9, gated=True, bias=True, residual=True)
    call = lambda: w4a16_linear(Wp, x, scales, bias=b, activation="silu", gated=True, residual=r)     # noqa: E731
    first = call().clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        call()
        with torch.cuda.graph(graph, stream=stream):
            y = call()
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, first)
    x.mul_(-1)
    graph.replay()
    second = call()
    torch.cuda.synchronize()
    assert torch.equal(y, second) and not torch.equal(first, second)


def test_interleaved_weights_of_both_factors(cuda_device):
    """The helper's order, through quantisation: gate and up as two products give the same sums."""
    from w4a16_opt import interleave_gate_up, quantize_pack, quantize_w4, w4a16_gemm, w4a16_linear
    gen = torch.Generator().manual_seed(4)
    gate, up = torch.randn(48, 256, generator=gen) * 0.05, torch.randn(48, 256, generator=gen) * 0.05
    x = torch.randn(21, 256, generator=gen).half().cuda()
    Wp, s = quantize_pack(interleave_gate_up(gate, up).cuda(), 64)
    (gq, gs), (uq, us) = quantize_w4(gate, 64), quantize_w4(up, 64)
    from w4a16_opt import pack_int4
    assert torch.equal(Wp.cpu(), pack_int4(interleave_gate_up(gq, uq)))
    assert torch.equal(s.cpu(), interleave_gate_up(gs, us, dim=1))
    g = w4a16_gemm(pack_int4(gq).cuda(), x, gs.cuda()).float()
    u = w4a16_gemm(pack_int4(uq).cuda(), x, us.cuda()).float()
    y = w4a16_linear(Wp, x, s, activation="silu", gated=True).float()
    # the two rounded sums: 2^-11 each, slope at most 1.13, and the result's own rounding
    want = torch.nn.functional.silu(g) * u
    assert bool(((y - want).abs() <= 2.0 ** -11 * (1.2 * g.abs() * u.abs() + 2 * want.abs()) + 2.0 ** -24).all())


def test_refusals(cuda_device):
    from w4a16_opt import w4a16_linear
    x, q, scales, Wp, b, r = operands(4, 64, 128, 64, 5, bias=True, residual=True)

    def refused(match, **kw):
        with pytest.raises(RuntimeError, match=match):
            w4a16_linear(Wp, x, scales, **kw)

    refused("activation must be one of", activation="swish")
    refused("bias must be", bias=b[:32])
    refused("bias must be", bias=b.float())
    refused("bias must be", bias=b.cpu())
    refused("residual must be", residual=r[:, :32])
    refused("residual must be", residual=r, gated=True)
    refused("residual must be", residual=r.bfloat16())
    refused("out must be", out=r.float())
    refused("must not overlap", out=torch.empty(0, dtype=torch.float16, device="cuda").set_(x.untyped_storage(), 0, (4, 64), (64, 1)))
    both = torch.zeros(5, 64, dtype=torch.float16, device="cuda")
    refused("must not overlap", out=both[1:], residual=both[:4])
    refused("variant must be", variant=5)
    refused("workspace", workspace=torch.zeros(16, dtype=torch.uint8))
