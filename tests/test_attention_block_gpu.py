"""GPU test of the attention block: 4-bit projections, rotary append and attention over the 4-bit
cache together, prompts and captured decode steps, against a 64-bit composition of the same steps."""
import pytest
import torch

from oracle import cache_oracle as oracle

pytestmark = pytest.mark.gpu

HQ, HK, D, HIDDEN, PAGE = 8, 2, 64, 512, 16


@pytest.fixture(autouse=True)
def _gpu(cuda_device):
    yield


def make_block(max_pos, pages, group=64):
    from w4a16_opt import Int4KVCache, quantize_pack
    from w4a16_opt.attention_block import AttentionBlock, rotary_table
    gen = torch.Generator().manual_seed(3)
    wqkv = quantize_pack((torch.randn((HQ + 2 * HK) * D, HIDDEN, generator=gen) * 0.05).cuda(), 128)
    wo = quantize_pack((torch.randn(HIDDEN, HQ * D, generator=gen) * 0.05).cuda(), 128)
    cache = Int4KVCache(pages, HK, D, PAGE, group)
    return AttentionBlock(wqkv, wo, HQ, cache, rotary_table(max_pos, D)), gen


def reference(block, x, positions, sequences):
    """The block's output in 64 bits, from its weights and what its cache holds.

    sequences: (first row, rows, slots of every cached token) of each sequence."""
    from w4a16_opt import w4a16_dequant, w4a16_gemm
    # the projection's own fp16 output: it decides what the cache holds
    qkv = w4a16_gemm(block.wqkv[0], x, block.wqkv[1]).view(len(x), HQ + 2 * HK, D)
    q = oracle.rotate(qkv[:, :HQ], positions[None], block.cos_sin)
    out = torch.empty(len(x), HQ * D, dtype=torch.float64, device="cuda")
    for at, rows, slots in sequences:
        k, v = oracle.read_slots(block.cache.data, D, PAGE, block.cache.group_size, slots)
        out[at:at + rows] = oracle.attention(q[at:at + rows], k, v)[0].reshape(rows, -1)
    wo = w4a16_dequant(block.wo[0], block.wo[1], HQ * D).double()
    return out @ wo.T


def close(got, want):
    # four values rounded to fp16 (queries, weights and values of the attention, its output), keys and the
    # projection's products too: each 2^-11 at most, 2^-12.5 or so in the mean; they add up as squares
    rel = ((got.double() - want).norm() / want.norm()).item()
    assert rel < 1.5e-3, rel


def test_prompts_then_decode_steps():
    from w4a16_opt.attention_block import DecodeLoop, slots_of
    lens, steps = [37, 1, 130], 5
    b, width = len(lens), -(-(max(lens) + steps + 1) // PAGE)
    block, gen = make_block(max(lens) + steps + 1, b * width)
    table = torch.randperm(b * width, generator=gen).int().view(b, width).cuda()
    seq_lens = torch.tensor(lens, dtype=torch.int32).cuda()
    cu = torch.tensor([0] + lens).cumsum(0).int().cuda()
    seq = torch.repeat_interleave(torch.arange(b), torch.tensor(lens)).cuda()
    pos = torch.cat([torch.arange(n) for n in lens]).cuda()
    x = torch.randn(sum(lens), HIDDEN, generator=gen).half().cuda()
    y = block(x, pos, slots_of(table, seq, pos, PAGE), table, seq_lens, cu_q=cu, max_q=max(lens))
    all_slots = lambda i, n: slots_of(table, torch.full((n,), i).cuda(), torch.arange(n).cuda(), PAGE)      # noqa: E731
    close(y, reference(block, x, pos, [(int(cu[i]), n, all_slots(i, n)) for i, n in enumerate(lens)]))

    loop = DecodeLoop(block, x[:b], table, seq_lens)
    assert seq_lens.tolist() == lens
    for step in range(steps):
        x = torch.randn(b, HIDDEN, generator=gen).half().cuda()
        before = seq_lens.long()
        y = loop.step(x).clone()
        now = [n + step + 1 for n in lens]
        assert seq_lens.tolist() == now
        close(y, reference(block, x, before, [(i, 1, all_slots(i, n)) for i, n in enumerate(now)]))


def test_a_prompt_in_chunks_fills_the_same_cache():
    from w4a16_opt.attention_block import slots_of
    n = 200
    width = -(-n // PAGE)
    whole, gen = make_block(n, width)
    parts, _ = make_block(n, width)
    table = torch.arange(width, dtype=torch.int32).cuda()[None]
    pos = torch.arange(n).cuda()
    slots = slots_of(table, torch.zeros_like(pos), pos, PAGE)
    x = torch.randn(n, HIDDEN, generator=gen).half().cuda()

    def run(block, a, e):
        cu = torch.tensor([0, e - a], dtype=torch.int32).cuda()
        return block(x[a:e], pos[a:e], slots[a:e], table, torch.tensor([e], dtype=torch.int32).cuda(), cu_q=cu, max_q=e - a)

    want = run(whole, 0, n)
    got = torch.cat([run(parts, 0, 90), run(parts, 90, 95), run(parts, 95, 96), run(parts, 96, n)])
    # rows differ between the kernels for few and for many rows (roundings), and from the 17th row on between
    # the projections' kernels
    rel = ((got.double() - want.double()).norm() / want.double().norm()).item()
    assert rel < 5e-3, rel


def test_the_command_runs(capsys):
    from w4a16_opt import attention_block
    attention_block.main(["--batch", "3", "--prompt", "300", "--steps", "4", "--page-size", "32", "--group-size", "64"])
    out = capsys.readouterr().out
    assert "prompts: 3 sequences" in out and "finite: True" in out
