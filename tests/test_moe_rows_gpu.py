"""GPU tests of what a token's result in the expert layer depends on: its own inputs and the call's sizes, bit for bit, whatever the
other tokens hold, wherever they are sent, in whatever order the tokens stand and the sort meets them."""
import pytest
import torch

from test_moe_experts_gpu import make, run

pytestmark = pytest.mark.gpu

# few entries sorted by every CTA (one warp, all of them), by the kernel in front; many entries an expert, at one and two tiles each
SHAPES = [(4, 8, 2, 256, 512, 128, 64), (40, 16, 4, 256, 192, 64, 64), (90, 40, 6, 128, 320, 64, 64), (200, 128, 8, 64, 64, 64, 64),
          (70, 5, 3, 256, 320, 128, 64), (300, 6, 2, 128, 448, 64, 64)]
ROWS = ("x", "experts", "weights", "residual")


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_other_tokens_do_not_matter(cuda_device, shape):
    T = shape[0]
    c = make(*shape, seed=31)
    y = run(c, residual=True)
    kept = list(range(0, T, 3))
    for seed in (32, 33):
        other = make(*shape, seed=seed)
        mixed = dict(c)
        for name in ROWS:
            mixed[name] = other[name].clone()
            mixed[name][kept] = c[name][kept]
        if seed == 33:              # all the others to one expert, or to none
            mixed["experts"][[t for t in range(T) if t % 3 == 1]] = 0
            mixed["experts"][[t for t in range(T) if t % 3 == 2]] = -1
        assert torch.equal(run(mixed, residual=True)[kept], y[kept])


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_the_order_of_tokens_does_not_matter(cuda_device, shape):
    c = make(*shape, seed=34)
    y = run(c, residual=True)
    p = torch.randperm(shape[0], generator=torch.Generator().manual_seed(1))
    assert torch.equal(run(dict(c, **{n: c[n][p].contiguous() for n in ROWS}), residual=True), y[p.cuda()])
    for _ in range(3):
        assert torch.equal(run(c, residual=True), y)
