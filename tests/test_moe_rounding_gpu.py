"""GPU tests of the one rounding inside the expert layer: inner results h = act(gate) * up become fp16, the operands of the second
product.  Nothing else is rounded before y, and what does not fit in fp16 is not finite.

Tolerances, before the first run.  h itself is known to d_h (fp32 sums of tensor-core products, the activation: as in
test_moe_experts_gpu).  Rounding is monotonic, so the kernel's fp16 h lies between fp16(h - d_h) and fp16(h + d_h): that
interval, a point for almost every value, is all that the second product's operand may be off by.  Its sums are off by (I / 16 + 12)
2^-22 S, the weighted sum of k products by (k + 2) 2^-23 of its terms' sizes, y by one rounding.
"""
import pytest
import torch

from test_linear_gpu import act64
from test_moe_experts_gpu import dequantised, make, run

pytestmark = pytest.mark.gpu


def with_h_rounded(c, activation):
    """(y in 64 bits from inner results rounded to fp16, what it may be off by, y without that rounding)."""
    x, (T, H), k, I = c["x"].double(), c["x"].shape, c["experts"].shape[1], c["q2"].shape[2]
    y, d, size, wide = (torch.zeros(T, H).double() for _ in range(4))
    for e in range(c["q1"].shape[0]):
        token, slot = (c["experts"] == e).nonzero(as_tuple=True)
        if not token.numel():
            continue
        W1, W2 = dequantised(c["q1"][e], c["s1"][e], c["groups"][0]), dequantised(c["q2"][e], c["s2"][e], c["groups"][1])
        z, dz = x[token] @ W1.t(), (H / 16 + 12) * 2.0 ** -22 * (x[token].abs() @ W1.abs().t())
        pick = lambda t, i: t.view(len(token), -1, 2, 8)[:, :, i].reshape(len(token), -1)      # noqa: E731
        zg, zu, dg, du = pick(z, 0), pick(z, 1), pick(dz, 0), pick(dz, 1)
        a = act64(zg, activation)
        h = a * zu
        dh = (1.13 * dg * (zu.abs() + du) + a.abs() * du + 2.0 ** -18 * h.abs()) * 1.001
        low, mid, high = (h - dh).half().double(), h.half().double(), (h + dh).half().double()
        off = torch.maximum(high - mid, mid - low)
        w = c["weights"][token, slot, None].double()
        out, S2 = mid @ W2.t(), (mid.abs() + off) @ W2.abs().t()
        y.index_add_(0, token, w * out)
        wide.index_add_(0, token, w * (h @ W2.t()))
        d.index_add_(0, token, w.abs() * (off @ W2.abs().t() + (I / 16 + 12) * 2.0 ** -22 * S2))
        size.index_add_(0, token, (w * out).abs())
    d = d + (k + 2) * 2.0 ** -23 * size
    return y, d * 1.001 + 2.0 ** -11 * (y.abs() + d) + 2.0 ** -25, wide


# both forms, groups of 64 and 128 in the second product
@pytest.mark.parametrize("activation", ["silu", "gelu_tanh", None])
@pytest.mark.parametrize("shape", [(1, 8, 2, 512, 1024, 128, 128), (8, 16, 4, 256, 512, 64, 64), (40, 8, 6, 256, 512, 128, 64), (130, 6, 2, 384, 640, 64, 128)],
                         ids=str)
def test_nothing_but_h_is_rounded(cuda_device, shape, activation):
    c = make(*shape, seed=21)
    y = run(c, activation).cpu().double()
    ref, tol, wide = with_h_rounded(c, activation)
    assert bool(((y - ref).abs() <= tol).all()), ((y - ref).abs() / tol).max()
    # and the rounding is there: the formula without it is farther away
    assert (y - ref).norm() < (y - wide).norm()


@pytest.mark.parametrize("T", [3, 120])
def test_an_inner_result_beyond_fp16(cuda_device, T):
    """h of 65504 is kept, h of 65520 (where rounding goes up to 2^16) and above is infinite: that token's y is not finite, no other's
    changes."""
    c = make(T, 3, 1, 64, 64, 64, 64, seed=22)
    c["experts"][:] = torch.arange(T)[:, None] % 3
    # channel 0 of the gate and of the other factor read x[:, 0] alone, with weight 1; all other products of theirs vanish
    c["q1"][:, 0], c["q1"][:, 8] = 8, 8
    c["q1"][:, 0, 0], c["q1"][:, 8, 0] = 9, 9
    c["s1"][:, :, 0], c["s1"][:, :, 8] = 1.0, 1.0
    c["weights"][:] = 2.0 ** -6
    from w4a16_opt import pack_int4
    c["w1"] = torch.stack([pack_int4(q) for q in c["q1"]])
    c["x"][:, 0] = 1.0
    clean = run(c, "relu").cpu()
    c["x"][1, 0] = 255.9                      # 255.875 in fp16: squared 65472.02
    below = run(c, "relu").cpu()
    assert below.isfinite().all()
    ref, tol, _ = with_h_rounded(c, "relu")
    assert bool(((below.double() - ref).abs() <= tol).all())
    c["x"][1, 0] = 256.0
    above = run(c, "relu").cpu()
    # codes of 8 are weights of 0: 0 * inf is not finite either
    assert not above[1].isfinite().any()
    others = [t for t in range(T) if t != 1]
    assert torch.equal(above[others], clean[others]) and torch.equal(below[others], clean[others])
