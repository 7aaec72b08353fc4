"""CPU tests of the attention block's host side: slots of positions, and where a decode loop ends."""
from types import SimpleNamespace

import pytest
import torch

from w4a16_opt.attention_block import DecodeLoop, slots_of


@pytest.mark.parametrize("page_size", [16, 64])
def test_slots(page_size):
    table = torch.tensor([[5, 0, 7], [2, 1 << 26, -1]], dtype=torch.int32)
    pos = torch.arange(3 * page_size)
    for b in (0, 1):
        slots = slots_of(table, torch.full_like(pos, b), pos, page_size)
        assert slots.dtype == torch.int64
        want = table[b].long()[pos // page_size] * page_size + pos % page_size
        assert torch.equal(slots[want >= 0], want[want >= 0]) and (slots[want < 0] < 0).all()


def test_positions_outside_the_table_have_no_slot():
    table = torch.tensor([[5, 0], [2, 1]], dtype=torch.int32)
    pos = torch.tensor([31, 32, 33, 1 << 40, -1, -17, 0])
    slots = slots_of(table, torch.tensor([0, 1, 0, 1, 0, 1, 1]), pos, 16)
    assert slots.tolist() == [15, -1, -1, -1, -1, -1, 32]
    none = torch.empty(2, 0, dtype=torch.int32)
    assert slots_of(none, torch.tensor([0, 1]), torch.tensor([0, 3]), 16).tolist() == [-1, -1]


def test_a_loop_is_refused_where_a_table_is_full():
    block = SimpleNamespace(cache=SimpleNamespace(page_size=16))
    table = torch.zeros(2, 3, dtype=torch.int32)
    for full in (48, 49, 1000):
        with pytest.raises(RuntimeError, match="fills its page table"):
            DecodeLoop(block, torch.zeros(2, 8), table, torch.tensor([5, full], dtype=torch.int32))


def test_a_loop_ends_with_its_table():
    """The steps are stood in for: a replay counts the lengths up."""
    loop = DecodeLoop.__new__(DecodeLoop)
    loop.block = SimpleNamespace(cache=SimpleNamespace(page_size=16))
    loop.page_table, loop.seq_lens = torch.zeros(2, 2, dtype=torch.int32), torch.tensor([29, 7], dtype=torch.int32)
    loop.x, loop.out, loop._left = torch.zeros(2, 8), torch.zeros(2, 8), 3
    replays = []

    def replay():
        loop.seq_lens += 1
        replays.append(loop.seq_lens.tolist())
        assert max(replays[-1]) <= 32

    loop.graph = SimpleNamespace(replay=replay)
    for _ in range(3):
        loop.step(torch.ones(2, 8))
    for _ in range(2):
        with pytest.raises(RuntimeError, match="no step is left"):
            loop.step(torch.ones(2, 8))
    assert replays[-1] == [32, 10] and len(replays) == 3
    loop.seq_lens[0] = 4                     # its place is given to another sequence
    for _ in range(22):
        loop.step(torch.ones(2, 8))
    assert replays[-1] == [26, 32]
    with pytest.raises(RuntimeError, match="no step is left"):
        loop.step(torch.ones(2, 8))
