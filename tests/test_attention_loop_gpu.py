"""GPU test of a decode loop's end: the steps up to it, its refusal, and the steps after a place is given away."""
import pytest
import torch

from test_attention_block_gpu import HIDDEN, PAGE, close, make_block, reference

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu(cuda_device):
    yield


def test_a_loop_ends_with_its_table_and_goes_on_with_another_sequence():
    from w4a16_opt.attention_block import DecodeLoop, slots_of
    lens, width = [44, 9], 3
    block, gen = make_block(64, 2 * width)
    table = torch.randperm(2 * width, generator=gen).int().view(2, width).cuda()
    seq_lens = torch.tensor(lens, dtype=torch.int32).cuda()
    seq = torch.repeat_interleave(torch.arange(2), torch.tensor(lens)).cuda()
    pos = torch.cat([torch.arange(n) for n in lens]).cuda()
    x = torch.randn(sum(lens), HIDDEN, generator=gen).half().cuda()
    block(x, pos, slots_of(table, seq, pos, PAGE), table, seq_lens,
          cu_q=torch.tensor([0] + lens).cumsum(0).int().cuda(), max_q=max(lens))
    all_slots = lambda i, n: slots_of(table, torch.full((n,), i).cuda(), torch.arange(n).cuda(), PAGE)      # noqa: E731
    loop = DecodeLoop(block, x[:2], table, seq_lens)

    def step(now):
        x = torch.randn(2, HIDDEN, generator=gen).half().cuda()
        before = seq_lens.long()
        y = loop.step(x).clone()
        assert seq_lens.tolist() == now
        close(y, reference(block, x, before, [(i, 1, all_slots(i, n)) for i, n in enumerate(now)]))

    for i in range(1, 5):
        step([44 + i, 9 + i])
    data = block.cache.data.clone()
    with pytest.raises(RuntimeError, match="no step is left"):
        loop.step(x[:2])
    assert torch.equal(block.cache.data, data) and seq_lens.tolist() == [48, 13]
    seq_lens[0] = 0                          # a new sequence in the first place
    for i in range(1, 4):
        step([i, 13 + i])
