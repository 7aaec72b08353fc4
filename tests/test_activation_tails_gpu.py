"""GPU tests of the activations where they are small and the other factor of a gate is large: the result keeps its digits.

The sums are exact here (weights of zero and a bias; or one weight of a row and one value of x), so that only the
activation's own error and the result's rounding are left.  Tolerances, before the first run, relative to the result:
    gelu: exp of -z^2 / 2 2 + 0.6 z^2 ulps, its argument z^2 2^-25, a fit of 7.7e-7, some 16 roundings beside: (z^2 + 12) 2^-22
    silu: exp 2 + 1.2 |z| ulps, sum, division and product 4: (1.2 |z| + 6) 2^-23
    gelu_tanh: the exponent t is off by 7 steps of 2^-24 |t|, exp by 2 + 1.2 |t| ulps: (4.7 |t| + 8) 2^-23
and y's rounding: 2^-11 relative, 2^-25 among fp16's subnormals.
"""
import pytest
import torch

from test_linear_gpu import act64

pytestmark = pytest.mark.gpu


def expected(zg, zu, activation):
    zg, zu = zg.cpu().double(), zu.cpu().double()
    y = act64(zg, activation) * zu
    t = 2 * (2 / torch.pi) ** 0.5 * (zg + 0.044715 * zg ** 3)
    rel = {"gelu": (zg ** 2 + 12) * 2.0 ** -22, "silu": (1.2 * zg.abs() + 6) * 2.0 ** -23, "gelu_tanh": (4.7 * t.abs() + 8) * 2.0 ** -23}[activation]
    return y, y.abs() * (rel + 2.0 ** -11) * 1.001 + 2.0 ** -25


def close(y, want):
    ref, tol = want
    off = (y.cpu().double() - ref).abs() / tol
    assert bool((off <= 1).all()), (off.max(), int(off.argmax()))


@pytest.mark.parametrize("activation", ["gelu", "silu", "gelu_tanh"])
@pytest.mark.parametrize("factor", [1.0, 100.0, 1000.0, 60000.0])
@pytest.mark.parametrize("M,variant", [(1, -1), (8, -1), (13, -1), (3, 1), (40, -1), (70, 2), (130, 3), (257, 4)])
def test_gated_product(cuda_device, M, variant, factor, activation):
    from w4a16_opt import interleave_gate_up, pack_int4, w4a16_linear
    cols, K = 512, 1024
    Wp = pack_int4(torch.full((2 * cols, K), 8, dtype=torch.uint8)).cuda()          # weights of zero
    scales = torch.ones(K // 128, 2 * cols, dtype=torch.float16, device="cuda")
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).half().cuda()
    zg = torch.linspace(-9, 3, cols).half()
    zu = torch.full((cols,), factor).half() * torch.where(torch.arange(cols) % 3 == 0, -1, 1).half()
    y = w4a16_linear(Wp, x, scales, bias=interleave_gate_up(zg, zu).cuda(), activation=activation, gated=True, variant=variant)
    ref, tol = expected(zg, zu, activation)
    fits = (ref.abs() < 65000).expand(M, cols)
    close(torch.where(fits.cuda(), y, 0), (torch.where(fits, ref.expand(M, cols), 0), tol.expand(M, cols)))


@pytest.mark.parametrize("activation", ["gelu", "silu", "gelu_tanh"])
@pytest.mark.parametrize("T", [1, 6, 100])
def test_experts(cuda_device, T, activation):
    """Gate and other factor from one value of x each: channel i is -s_i x_0 and 64 x_0; the second product passes channel i on."""
    from w4a16_opt import interleave_gate_up, moe_experts, pack_int4
    E, H, I = 2, 512, 512
    zg = torch.linspace(0.5, 9, I).half()
    gate, up = torch.full((I, H), 8, dtype=torch.uint8), torch.full((I, H), 8, dtype=torch.uint8)
    gate[:, 0], up[:, 0] = 7, 9
    down = torch.full((H, I), 8, dtype=torch.uint8)
    down[torch.arange(I), torch.arange(I)] = 9
    s1 = interleave_gate_up(zg, torch.full((I,), 64.0).half()).expand(H // 64, 2 * I).contiguous()
    s2 = torch.ones(I // 64, H).half()
    stack = lambda t: torch.stack([t] * E).cuda()       # noqa: E731
    x = torch.zeros(T, H).half()
    x[:, 0] = 1.0
    experts = (torch.arange(T) % E).int()[:, None].cuda()
    y = moe_experts(x.cuda(), (stack(pack_int4(interleave_gate_up(gate, up))), stack(s1)), (stack(pack_int4(down)), stack(s2)), experts,
                    torch.ones(T, 1, device="cuda"), activation=activation)
    ref, tol = expected(-zg, torch.full((I,), 64.0), activation)
    close(y, (ref.expand(T, I), tol.expand(T, I) * 2))       # the inner result's rounding, y's


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("M", [2, 40])
def test_infinite_and_not_a_number(cuda_device, M, gated):
    """z of +inf passes, large negative z vanishes, NaN stays, beside ordinary columns."""
    from w4a16_opt import interleave_gate_up, pack_int4, w4a16_linear
    cols, K, inf = 16, 128, float("inf")
    zg = torch.tensor([inf, -60000.0, float("nan"), 60000.0, 0.0, 1.0, -1.0, 30.0] * 2).half()
    N = 2 * cols if gated else cols
    Wp = pack_int4(torch.full((N, K), 8, dtype=torch.uint8)).cuda()
    x, scales = torch.ones(M, K).half().cuda(), torch.ones(K // 64, N).half().cuda()
    bias = interleave_gate_up(zg, torch.ones(cols).half()) if gated else zg
    for activation in ("gelu", "silu", "gelu_tanh"):
        y = w4a16_linear(Wp, x, scales, bias=bias.cuda(), activation=activation, gated=gated).cpu()
        assert (y[:, ::8] == inf).all() and (y[:, 1::8] == 0).all() and y[:, 2::8].isnan().all() and (y[:, 3::8] == 60000).all()
        assert (y[:, 4::8] == 0).all() and (y[:, 7::8] == 30).all()
        one = act64(torch.tensor([1.0, -1.0]).double(), activation)
        assert ((y[:, 5:7].double() - one).abs() <= 2.0 ** -10 * one.abs()).all()
