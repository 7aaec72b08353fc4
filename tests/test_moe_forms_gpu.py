"""GPU test of the expert layer on either side of the border between its forms; tolerances as in test_moe_experts_gpu."""
import pytest

from test_moe_experts_gpu import check, make, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("groups", [(128, 128), (64, 128), (128, 64), (64, 64)], ids=str)
@pytest.mark.parametrize("T", [20, 21, 24, 28, 29])
def test_both_sides_of_the_border(cuda_device, T, groups):
    c = make(T, 4, 2, 256, 384, *groups, seed=51)        # 4 experts of 2 choices: 10 entries an expert at 20 tokens, 14 at 28
    check(c, run(c, residual=True), residual=True)
