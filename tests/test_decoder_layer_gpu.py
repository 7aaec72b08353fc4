"""GPU test of a whole decoder layer from 4-bit weights: norm, attention over the 4-bit cache, products with their epilogues or routed
experts, together, on prompts and captured decode steps, against a 64-bit composition of the same steps."""
import pytest
import torch

from oracle import cache_oracle
from test_attention_block_gpu import HIDDEN, HK, HQ, PAGE, D
from test_linear_gpu import act64

pytestmark = pytest.mark.gpu

INNER, EXPERTS, K, EXPERT_INNER = 448, 8, 2, 192


@pytest.fixture(autouse=True)
def _gpu(cuda_device):
    yield


def make_layer(kind, max_pos, pages):
    from w4a16_opt import Int4KVCache, interleave_gate_up, quantize_pack
    from w4a16_opt.attention_block import AttentionBlock, rotary_table
    from w4a16_opt.mlp_block import DecoderLayer, ExpertBlock, MLPBlock
    gen = torch.Generator().manual_seed(11)
    rand = lambda *s: torch.randn(*s, generator=gen) * 0.05     # noqa: E731
    pack = lambda w, g=128: quantize_pack(w.cuda(), g)          # noqa: E731
    norms = [(1 + 4 * rand(HIDDEN)).half().cuda() for _ in range(2)]
    cache = Int4KVCache(pages, HK, D, PAGE, 64)
    attention = AttentionBlock(pack(rand((HQ + 2 * HK) * D, HIDDEN)), pack(rand(HIDDEN, HQ * D)), HQ, cache, rotary_table(max_pos, D), norms[0])
    if kind == "dense":
        mlp = MLPBlock(pack(interleave_gate_up(rand(INNER, HIDDEN), rand(INNER, HIDDEN))), pack(rand(HIDDEN, INNER), 64), norms[1])
    else:
        stacked = lambda ws: tuple(torch.stack(t) for t in zip(*ws))        # noqa: E731
        mlp = ExpertBlock((4 * rand(HIDDEN, EXPERTS)).half().cuda(),
                          stacked([pack(interleave_gate_up(rand(EXPERT_INNER, HIDDEN), rand(EXPERT_INNER, HIDDEN))) for _ in range(EXPERTS)]),
                          stacked([pack(rand(HIDDEN, EXPERT_INNER), 64) for _ in range(EXPERTS)]), K, norms[1])
    return DecoderLayer(attention, mlp), gen


def weight(pair, k):
    from w4a16_opt import w4a16_dequant
    return w4a16_dequant(pair[0], pair[1], k).double()


def norm64(x, w):
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-5) * w.double()


def gated(z):
    z = z.view(len(z), z.shape[1] // 16, 2, 8)
    return (act64(z[:, :, 0], "silu") * z[:, :, 1]).flatten(1)


def reference(layer, x, positions, sequences):
    """In 64 bits, from the layer's weights and what its cache holds; the experts that the layer's own fp16 logits choose."""
    from w4a16_opt import moe_route, rms_norm, w4a16_gemm
    a, m = layer.attention, layer.mlp
    qkv = w4a16_gemm(a.wqkv[0], rms_norm(x, a.norm), a.wqkv[1]).view(len(x), HQ + 2 * HK, D)     # it decides what the cache holds
    q = cache_oracle.rotate(qkv[:, :HQ], positions[None], a.cos_sin)
    out = torch.empty(len(x), HQ * D, dtype=torch.float64, device="cuda")
    for at, rows, slots in sequences:
        k, v = cache_oracle.read_slots(a.cache.data, D, PAGE, a.cache.group_size, slots)
        out[at:at + rows] = cache_oracle.attention(q[at:at + rows], k, v)[0].reshape(rows, -1)
    x = x.double() + out @ weight(a.wo, HQ * D).t()
    h = norm64(x, m.norm)
    if not hasattr(m, "router"):
        return x + gated(h @ weight(m.gate_up, HIDDEN).t()) @ weight(m.down, INNER).t()
    weights, experts = moe_route(rms_norm(x.half(), m.norm) @ m.router, m.k)
    y = x.clone()
    for e in range(EXPERTS):
        token, slot = (experts == e).nonzero(as_tuple=True)
        z = gated(h[token] @ weight([t[e] for t in m.gate_up], HIDDEN).t()) @ weight([t[e] for t in m.down], EXPERT_INNER).t()
        y.index_add_(0, token, z * weights[token, slot, None].double())
    return y


def close(got, want):
    # some ten values rounded to fp16 on the way (norms, queries, keys, attention, the stream, inner results, weights, the result): 2^-11 at
    # most, 2^-12.5 or so in the mean each; they add up as squares
    rel = ((got.double() - want).norm() / want.norm()).item()
    assert rel < 1.5e-3, rel


@pytest.mark.parametrize("kind", ["dense", "experts"])
@pytest.mark.parametrize("lens", [[37, 1, 130], [4, 9]], ids=["many", "few"])
def test_prompts_then_decode_steps(kind, lens):
    from w4a16_opt.attention_block import DecodeLoop, slots_of
    steps, b = 4, len(lens)
    width = -(-(max(lens) + steps + 1) // PAGE)
    layer, gen = make_layer(kind, max(lens) + steps + 1, b * width)
    table = torch.randperm(b * width, generator=gen).int().view(b, width).cuda()
    seq_lens = torch.tensor(lens, dtype=torch.int32).cuda()
    cu = torch.tensor([0] + lens).cumsum(0).int().cuda()
    seq = torch.repeat_interleave(torch.arange(b), torch.tensor(lens)).cuda()
    pos = torch.cat([torch.arange(n) for n in lens]).cuda()
    x = torch.randn(sum(lens), HIDDEN, generator=gen).half().cuda()
    y = layer(x, pos, slots_of(table, seq, pos, PAGE), table, seq_lens, cu_q=cu, max_q=max(lens))
    every = lambda s, n: slots_of(table, torch.full((n,), s).cuda(), torch.arange(n).cuda(), PAGE)      # noqa: E731
    close(y, reference(layer, x, pos, [(int(cu[s]), lens[s], every(s, lens[s])) for s in range(b)]))

    x = torch.randn(b, HIDDEN, generator=gen).half().cuda()
    loop = DecodeLoop(layer, x, table, seq_lens)
    for step in range(steps):
        y = loop.step(x).clone()
        lengths = [n + step + 1 for n in lens]
        assert seq_lens.tolist() == lengths
        close(y, reference(layer, x, torch.tensor(lengths).cuda() - 1, [(s, 1, every(s, lengths[s])) for s in range(b)]))
        x = y


def test_the_command_runs_a_layer(capsys):
    from w4a16_opt import attention_block
    for kind in ("dense", "experts"):
        attention_block.main(["--batch", "2", "--prompt", "40", "--steps", "3", "--layer", kind])
        out = capsys.readouterr().out
        assert "prompts: 2 sequences" in out and "finite: True" in out


def test_a_layer_needs_the_attention_blocks_norm():
    from w4a16_opt.attention_block import AttentionBlock
    from w4a16_opt.mlp_block import DecoderLayer
    with pytest.raises(RuntimeError, match="needs its norm"):
        DecoderLayer(AttentionBlock(None, None, 8, None, None), None)
