"""GPU tests of the 4-bit key/value cache: append, read back and attention against the plain
64-bit oracle, at the sizes and masks where they can go wrong.

Tolerances.  Codes, scales and minima of an append, and read-back values, are exact.  For
attention, with u = 2^-11 (fp16), an output may be off by
    u_out |out| + A (2 u + 2 dS + 2^-12) + n 2^-24 max|V|
where A = sum_t p_t |V_t|: weights and values may be rounded to fp16 (2 u); scores may be off by
dS = (u + 2^-13) max_t scale sum_d |q_d K_td| (keys rounded to fp16, sums in fp32), which moves a
normalised weight by at most 2 dS; 2^-12 covers exp2 and fp32 sums; the last term is what n weights
below fp16's normal range may lose.  u_out is 2^-11 for fp16 and 2^-8 for bf16.
"""
import math

import pytest
import torch

from oracle import cache_oracle as oracle

pytestmark = pytest.mark.gpu

U16 = 2.0 ** -11
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(autouse=True)
def _gpu(cuda_device):
    yield
    import w4a16_opt
    assert w4a16_opt.device_status(reset=True) == 0


def rand(gen, *shape):
    return torch.randn(*shape, generator=gen, dtype=torch.float32).cuda()


class Problem:
    """A cache filled through cache_append, with garbage in every row that no token was written to."""

    def __init__(self, lens, q_lens, hq, hk, d, g=None, page=64, dtype="fp16", seed=0, gain=1.0, extra_pages=2, width=None):
        import w4a16_opt as w
        gen = torch.Generator().manual_seed(seed)
        self.d, self.g, self.page, self.hq, self.hk = d, g or d, page, hq, hk
        self.lens, self.q_lens, self.dtype = lens, q_lens, DT[dtype]
        used = [-(-n // page) for n in lens]
        pages = sum(used) + extra_pages
        nbytes = oracle.block_bytes(page, d, self.g)
        # 0xFF pairs are NaN, 0x7C00 infinities
        self.data = torch.randint(0, 256, (pages, hk, nbytes), generator=gen, dtype=torch.uint8).cuda()
        self.data[:, :, page * d:].view(torch.int16)[:, :, ::3] = 0x7C00
        self.data[:, :, page * d:].view(torch.int16)[:, :, 1::3] = -1
        self.cache = w.Int4KVCache.wrap(self.data, d, page, self.g)
        order = torch.randperm(pages, generator=gen)
        width = width or max(used + [1]) + 1
        self.table = torch.full((len(lens), width), -1, dtype=torch.int32)
        at = 0
        for b, u in enumerate(used):
            self.table[b, :u] = order[at:at + u].int()
            at += u
        slots = [self.table[b].long()[torch.arange(n) // page] * page + torch.arange(n) % page for b, n in enumerate(lens)]
        self.slots = [s.cuda() for s in slots]
        self.table = self.table.cuda()
        total = sum(lens)
        self.k = (rand(gen, total, hk, d) * (1 + 5 * (torch.rand(d, generator=gen) < 0.05).float()).cuda()).to(self.dtype)
        self.v = rand(gen, total, hk, d).to(self.dtype)
        if total:
            w.cache_append(self.cache, self.k, self.v, torch.cat(self.slots))
        self.seq_lens = torch.tensor(lens, dtype=torch.int32).cuda()
        self.cu = torch.tensor([0] + q_lens).cumsum(0).int().cuda()
        self.q = (rand(gen, sum(q_lens), hq, d) * gain).to(self.dtype)

    def run(self, q=None, **kw):
        import w4a16_opt as w
        q = self.q if q is None else q
        if max(self.q_lens + [0]) != 1 or min(self.q_lens) != 1:
            kw.setdefault("cu_q", self.cu)
            kw.setdefault("max_q", max(self.q_lens))
        return w.cache_attention(q, self.cache, self.table, self.seq_lens, **kw)

    def check(self, out, lse=None, scale=None, causal=True, window=0):
        u_out = U16 if self.dtype == torch.float16 else 2.0 ** -8
        at = 0
        for b, (n, t) in enumerate(zip(self.lens, self.q_lens)):
            k, v = oracle.read_slots(self.data, self.d, self.page, self.g, self.slots[b])
            q = self.q[at:at + t].double()
            ref, rlse, spread, drift = oracle.attention(q, k, v, scale, causal, window)
            got = out[at:at + t].double()
            assert torch.isfinite(got).all(), f"sequence {b}: not finite"
            ds = (U16 + 2.0 ** -13) * drift[..., None]
            vmax = v.abs().max() if n else 0.0
            tol = u_out * ref.abs() + spread * (2 * U16 + 2 * ds + 2.0 ** -12) + n * 2.0 ** -24 * vmax + 1e-7
            worst = ((got - ref).abs() / tol).max().item() if t else 0.0
            assert worst <= 1.0, f"sequence {b} (L {n}, T {t}): {worst:.3g} of the tolerance"
            if lse is not None:
                gl = lse[at:at + t].double()
                empty = rlse == -math.inf
                assert torch.equal(gl == -math.inf, empty)
                lim = ((U16 + 2.0 ** -13) * drift + 2.0 ** -12 + rlse.abs() * 2.0 ** -22)[~empty]
                assert ((gl - rlse)[~empty].abs() <= lim).all()
            at += t


# ------------------------------------------------------------------------------ append, read back

def append_reference(data, d, g, page, slots, k, v):
    """The bytes that appending k, v (fp64) leaves, token by token."""
    data = data.clone().cpu()
    kq, vq = oracle.quantise(k.cpu(), g), oracle.quantise(v.cpu(), g)
    for t, s in enumerate(slots.tolist()):
        if not 0 <= s < data.shape[0] * page:
            continue
        for h in range(k.shape[1]):
            oracle.write_block(data[s // page, h], page, s % page, [x[t, h] for x in kq], [x[t, h] for x in vq])
    return data


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("d,g", [(64, 64), (128, 64), (128, 128)])
@pytest.mark.parametrize("tokens,hk,page", [(1, 1, 16), (37, 3, 16), (130, 8, 64), (33, 2, 256)])
def test_append_writes_exactly_its_slots(tokens, hk, page, d, g, dtype):
    import w4a16_opt as w
    gen = torch.Generator().manual_seed(tokens + d + g)
    pages = -(-tokens // page) + 2
    data = torch.randint(0, 256, (pages, hk, oracle.block_bytes(page, d, g)), generator=gen, dtype=torch.uint8).cuda()
    slots = torch.randperm(pages * page, generator=gen)[:tokens]
    if tokens > 4:
        slots[2], slots[3] = -1, pages * page       # both outside: skipped
    k, v = rand(gen, tokens, hk, d).to(DT[dtype]), (rand(gen, tokens, hk, d) * 30).to(DT[dtype])
    k[0, 0] = 0                                     # a constant group: scale 0
    v[-1, -1, :g] = 1e-7
    before = data.clone()
    assert w.cache_append(w.Int4KVCache.wrap(data, d, page, g), k, v, slots.cuda()) is None
    assert torch.equal(data.cpu(), append_reference(before, d, g, page, slots, k.double(), v.double()))


def test_append_of_values_that_are_not_finite_or_too_large():
    import w4a16_opt as w
    d = 128
    x = torch.zeros(6, 1, d)
    x[0, 0, :4] = torch.tensor([math.nan, 1.0, -1.0, 0.5])
    x[1, 0, :2] = torch.tensor([math.inf, -3.0])
    x[2, 0, :2] = torch.tensor([-math.inf, 3e38])
    x[3] = math.nan
    x[4, 0] = torch.linspace(-1e5, 1e5, d)
    x[5, 0] = torch.arange(d) % 16 + 0.5           # half codes: ties go to even
    for dtype in (torch.float16, torch.bfloat16):
        y = x.to(dtype).cuda()
        cache = w.Int4KVCache(2, 1, d, 16)
        slots = torch.arange(6).cuda() + 3
        w.cache_append(cache, y, y, slots)
        want = append_reference(torch.zeros_like(cache.data), d, d, 16, slots, y.double(), y.double())
        assert torch.equal(cache.data.cpu(), want)
        for out in w.cache_read(cache, slots, dtype):
            assert torch.isfinite(out).all()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("d,g,page,hk,tokens", [(64, 64, 16, 5, 77), (128, 64, 32, 1, 1), (128, 128, 64, 8, 300)])
def test_read_gives_the_values_that_the_codes_stand_for(d, g, page, hk, tokens, dtype):
    import w4a16_opt as w
    p = Problem([tokens], [1], hk, hk, d, g, page, dtype)
    slots = p.slots[0].clone()
    slots[0] = -1
    k, v = w.cache_read(p.cache, slots, DT[dtype])
    for got, ref in zip((k, v), oracle.read_slots(p.data, d, page, g, p.slots[0])):
        assert torch.equal(got[1:], ref[1:].float().to(DT[dtype]))       # the sum is rounded to fp32, then 16 bits
        assert (got[0] == 0).all()
    k, v = w.cache_read(p.cache, slots[:0], DT[dtype])
    assert k.shape == (0, hk, d)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rotary,hq,hk,axes,sections", [
    (128, 128, 32, 8, 1, None), (128, 64, 7, 1, 1, None), (64, 64, 5, 5, 3, (8, 12, 12)), (64, 32, 2, 1, 2, (3, 13)),
    (128, 128, 28, 4, 3, (16, 24, 24)), (128, 128, 4, 2, 3, (0, 64, 0))])
def test_append_with_rotary_positions(d, rotary, hq, hk, axes, sections, interleaved):
    import w4a16_opt as w
    gen = torch.Generator().manual_seed(d + rotary + hq)
    tokens, page, top = 45, 32, 600
    x = rand(gen, tokens, hq + 2 * hk, d).half()        # one fused projection: strided views
    q, k, v = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
    angle = torch.arange(top, dtype=torch.float64)[:, None] * 500000.0 ** (-torch.arange(rotary // 2) / (rotary // 2))
    cs = torch.cat((angle.cos(), angle.sin()), 1).float().cuda()
    pos = torch.randint(0, top, (axes, tokens), generator=gen)
    pos[0, 0], pos[-1, 1] = -5, top + 9                 # led back into the table
    pos = pos.cuda()
    cache = w.Int4KVCache(3, hk, d, page)
    slots = torch.arange(tokens).flip(0).cuda()
    kept = x.clone()
    out = w.cache_append(cache, k, v, slots, q=q, positions=pos if axes > 1 else pos[0], cos_sin=cs, sections=sections,
                         interleaved=interleaved)
    assert torch.equal(x, kept)
    ref = oracle.rotate(q, pos, cs, sections, interleaved)
    # two products and a sum in fp32, one rounding to fp16
    assert ((out.double() - ref).abs() <= U16 * ref.abs() + 2.0 ** -22 * (1 + q.double().abs().max()) + 2.0 ** -25).all()
    kt = oracle.rotate(k, pos, cs, sections, interleaved)
    got_k, got_v = oracle.read_slots(cache.data, d, page, d, slots)
    want_k = oracle.values(*oracle.quantise(kt, d), d)
    want_v = oracle.values(*oracle.quantise(v.double(), d), d)
    assert torch.equal(got_v, want_v)
    # a turned key differs in its last fp32 bit from the oracle's: a value next to the middle of two
    # codes may take the other, and a scale or minimum next to the middle of two fp16 numbers too
    step = (kt.amax(-1, keepdim=True) - kt.amin(-1, keepdim=True)) / 15
    off = (got_k - want_k).abs()
    assert (off <= step * 1.01).all() and (off > step * 0.01).double().mean() < 1e-3
    # keys alone
    other = w.Int4KVCache(3, hk, d, page)
    assert w.cache_append(other, k, v, slots, positions=pos if axes > 1 else pos[0], cos_sin=cs, sections=sections,
                          interleaved=interleaved) is None
    assert torch.equal(other.data, cache.data)


# ------------------------------------------------------------------------------ attention

@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("d,g,hq,hk,page", [(64, 64, 4, 4, 16), (64, 64, 16, 1, 64), (128, 64, 8, 2, 32), (128, 128, 32, 8, 64),
                                           (128, 128, 5, 1, 256), (128, 64, 28, 4, 128), (128, 128, 24, 1, 64),
                                           (64, 64, 3, 1, 16)])
def test_decode_ragged(d, g, hq, hk, page, dtype):
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 200, 511, 777, 1500]
    p = Problem(lens, [1] * len(lens), hq, hk, d, g, page, dtype, seed=d + hq)
    out, lse = p.run(return_lse=True)
    assert out.dtype == p.dtype and lse.dtype == torch.float32
    p.check(out, lse)


@pytest.mark.parametrize("batch,length", [(1, 1), (1, 40000), (3, 9001), (200, 33), (37, 500)])
def test_decode_batches(batch, length):
    lens = [max(1, length - 7 * b) for b in range(batch)]
    p = Problem(lens, [1] * batch, 8, 2, 128, 128, 64, seed=batch)
    out, lse = p.run(return_lse=True)
    p.check(out, lse)


@pytest.mark.parametrize("hq,hk,d,g", [(4, 1, 128, 128), (8, 8, 64, 64), (16, 2, 128, 64), (7, 1, 128, 128)])
@pytest.mark.parametrize("nq", [2, 3, 4, 5, 8, 16, 17])
def test_few_queries(nq, hq, hk, d, g):
    lens = [nq, nq + 1, 64 + nq, 300, 130, 1025]
    p = Problem(lens, [nq] * len(lens), hq, hk, d, g, 32, seed=nq)
    out, lse = p.run(return_lse=True)
    p.check(out, lse)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("hq,hk,d,g,page", [(8, 2, 128, 128, 64), (4, 4, 64, 64, 16), (28, 4, 128, 64, 32), (3, 1, 128, 128, 256)])
def test_prompts_ragged(hq, hk, d, g, page, dtype):
    lens = [1, 31, 100, 128, 129, 257, 600, 1000]
    q_lens = [1, 31, 33, 128, 1, 200, 600, 129]
    p = Problem(lens, q_lens, hq, hk, d, g, page, dtype, seed=hq)
    out, lse = p.run(return_lse=True)
    p.check(out, lse)


@pytest.mark.parametrize("hq,hk,d,lens,q_lens", [(32, 8, 128, [2000], [2000]), (8, 1, 128, [20000], [64]),
                                                  (4, 1, 64, [9000, 50], [40, 50]), (16, 2, 64, [1300, 1300], [1300, 700])])
def test_prompts_long(hq, hk, d, lens, q_lens):
    p = Problem(lens, q_lens, hq, hk, d, d, 64, seed=len(lens) + hq)
    out, lse = p.run(return_lse=True)
    p.check(out, lse)


@pytest.mark.parametrize("causal,window", [(False, 0), (True, 1), (True, 64), (True, 100), (False, 90), (True, 5000)])
@pytest.mark.parametrize("q_lens", [[1, 1, 1, 1], [3, 1, 2, 3], [70, 10, 150, 300]])
def test_masks(q_lens, causal, window):
    p = Problem([70, 513, 150, 300], q_lens, 8, 2, 128, 128, 16, seed=window)
    out, lse = p.run(causal=causal, window=window, return_lse=True)
    p.check(out, lse, causal=causal, window=window)


@pytest.mark.parametrize("q_lens,causal,window", [([1, 1, 1], True, 0), ([4, 3, 2], True, 0), ([4, 3, 2], False, 0),
                                                   ([90, 40, 200], True, 0), ([90, 40, 200], True, 7), ([4, 3, 2], True, 2),
                                                   ([4, 3, 2], False, 2), ([90, 40, 200], False, 9)])
def test_rows_that_see_nothing(q_lens, causal, window):
    """Empty sequences, and more queries than cached tokens: the first rows have nothing to look at."""
    p = Problem([0, 1, 2 if max(q_lens) < 50 else 70], q_lens, 4, 2, 64, 64, 16)
    out = torch.full_like(p.q, math.nan)
    got, lse = p.run(causal=causal, window=window, return_lse=True, out=out)
    assert got.data_ptr() == out.data_ptr()
    p.check(out, lse, causal=causal, window=window)


def test_sequences_without_queries_and_empty_calls():
    import w4a16_opt as w
    p = Problem([50, 60, 70], [0, 5, 0], 4, 2, 64, 64, 16)
    p.check(p.run())
    p = Problem([50, 300, 70], [0, 150, 0], 4, 2, 64, 64, 16)
    p.check(p.run())
    none = torch.empty(0, 4, 64, dtype=torch.half, device="cuda")
    out = w.cache_attention(none, p.cache, p.table[:0], p.seq_lens[:0])
    assert out.shape == (0, 4, 64)


@pytest.mark.parametrize("q_len", [1, 6, 200])
@pytest.mark.parametrize("gain,scale", [(0.0, None), (40.0, None), (1.0, 0.0), (1.0, -0.3), (3000.0, 1e-4), (1e-4, 300.0)])
def test_scores_of_every_size(gain, scale, q_len):
    """Uniform weights, weights that are all on one token, negative and tiny scales."""
    p = Problem([400, 1030], [q_len, q_len], 8, 2, 128, 128, 64, gain=gain, seed=3)
    out, lse = p.run(scale=scale, return_lse=True)
    p.check(out, lse, scale=scale)


@pytest.mark.parametrize("q_len", [1, 5, 150])
@pytest.mark.parametrize("d,g", [(64, 64), (128, 64), (128, 128)])
def test_a_token_with_all_the_weight_and_tiny_values(d, g, q_len):
    """An attention sink: the first token draws nearly all the weight and its values are near zero, so
    the output comes from weights thousands of times smaller."""
    import w4a16_opt as w
    p = Problem([900], [q_len], 4, 1, d, g, 32, seed=1)
    first = p.q.double().mean((0, 1))
    p.q = (first + 0.05 * p.q.double()).to(p.dtype)
    key = first / (first * first).sum() * 9.0 * math.sqrt(d)
    p.k = (p.k.double() * 0.05).half()
    p.k[0, 0] = key.half()
    p.v[0, 0] *= 1e-3
    p.v[5, 0] *= 40                                    # and one token with large values
    w.cache_append(p.cache, p.k, p.v, p.slots[0])
    out, lse = p.run(return_lse=True)
    p.check(out, lse)


@pytest.mark.parametrize("q_len", [1, 7, 140])
def test_query_strides_and_offsets(q_len):
    """Queries that are views of a wider buffer, and lengths that are views too."""
    p = Problem([500, 333], [q_len, q_len], 8, 2, 128, 128, 64, seed=2)
    want = p.run()
    wide = torch.full((p.q.shape[0], 12, 136), math.nan, dtype=p.dtype, device="cuda")
    wide[:, 2:10, 8:] = p.q
    assert torch.equal(p.run(wide[:, 2:10, 8:]), want)
    heads_first = p.q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(p.run(heads_first), want)
    import w4a16_opt as w
    table = torch.cat((p.table, p.table), 1)[:, :p.table.shape[1]]
    assert table.stride(0) != table.shape[1]
    p.check(w.cache_attention(p.q, p.cache, table, p.seq_lens, cu_q=p.cu, max_q=q_len + 3))


@pytest.mark.parametrize("q_len", [1, 9, 300])
def test_same_inputs_same_bits(q_len):
    lens = [3000, 77, 1400, 640]
    p = Problem(lens, [min(q_len, n) for n in lens], 8, 2, 128, 64, 32, seed=5)
    first = p.run()
    for _ in range(5):
        assert torch.equal(p.run(), first)


@pytest.mark.parametrize("q_len", [1, 9, 150])
def test_other_streams_and_graphs(q_len):
    import w4a16_opt as w
    p = Problem([700, 2100], [q_len, q_len], 8, 2, 128, 128, 64, seed=8)
    want = p.run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(p.run(), want)
        graph = torch.cuda.CUDAGraph()
        q, out = p.q.clone(), torch.empty_like(p.q)
        with torch.cuda.graph(graph, stream=side):
            p.run(q, out=out)
        q.copy_(p.q.flip(0))
        graph.replay()
        q.copy_(p.q)
        graph.replay()
    side.synchronize()
    assert torch.equal(out, want)


def test_lengths_may_change_between_replays():
    """A captured decode step serves sequences as they grow: lengths are read on the device."""
    import w4a16_opt as w
    p = Problem([900, 400], [1, 1], 8, 2, 128, 128, 64, seed=4)
    lens = p.seq_lens.clone()
    p.run()
    graph = torch.cuda.CUDAGraph()
    out = torch.empty_like(p.q)
    with torch.cuda.graph(graph):
        w.cache_attention(p.q, p.cache, p.table, lens, out=out)
    for now in ([900, 400], [1, 399], [0, 64], [65, 900]):
        now = [min(a, b) for a, b in zip(now, p.lens)]
        lens.copy_(torch.tensor(now, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        q = Problem.__new__(Problem)
        q.__dict__.update(p.__dict__)
        q.lens, q.slots = now, [s[:n] for s, n in zip(p.slots, now)]
        q.check(out)


@pytest.mark.parametrize("q_len", [1, 130])
def test_lengths_past_the_table_are_clamped(q_len):
    p = Problem([128, 64], [q_len, q_len], 4, 2, 128, 128, 64, width=2)
    p.seq_lens = torch.tensor([100000, 64], dtype=torch.int32).cuda()
    out = p.run()
    p.check(out)


@pytest.mark.parametrize("q_len", [1, 140])
def test_caches_beyond_four_gigabytes(q_len):
    """Pages whose byte offsets pass 32 bits."""
    import w4a16_opt as w
    d, page, hk = 128, 256, 8
    nbytes = oracle.block_bytes(page, d, d)
    pages = (5 << 30) // (hk * nbytes)
    cache = w.Int4KVCache(pages, hk, d, page)
    gen = torch.Generator().manual_seed(0)
    n = 700
    table = torch.tensor([[pages - 1, pages // 2 + 1, pages - 2]], dtype=torch.int32).cuda()
    at = torch.arange(n).cuda()
    slots = table[0].long()[at // page] * page + at % page
    k, v = rand(gen, n, hk, d).half(), rand(gen, n, hk, d).half()
    w.cache_append(cache, k, v, slots)
    got = w.cache_read(cache, slots)
    for a, x in zip(got, (k, v)):
        assert torch.equal(a, oracle.values(*oracle.quantise(x.double(), d), d).float().half())
    small = w.Int4KVCache(3, hk, d, page)
    w.cache_append(small, k, v, at)
    q = rand(gen, q_len, 16, d).half()
    lens = torch.tensor([n], dtype=torch.int32).cuda()
    kw = dict(cu_q=torch.tensor([0, q_len], dtype=torch.int32).cuda(), max_q=q_len)
    want = w.cache_attention(q, small, torch.arange(3, dtype=torch.int32).cuda()[None], lens, **kw)
    assert torch.equal(w.cache_attention(q, cache, table, lens, **kw), want)


def test_a_query_that_is_not_finite_spoils_its_own_row_only():
    for q_len in (1, 6, 140):
        p = Problem([400, 200], [q_len, q_len], 4, 2, 128, 128, 64)
        want = p.run()
        q = p.q.clone()
        q[0, 1] = math.nan
        got = p.run(q)
        assert torch.isnan(got[0, 1]).all()
        got[0, 1] = want[0, 1]
        assert torch.equal(got, want)


# ------------------------------------------------------------------------------ refusals of the binding

def test_attention_refuses_what_it_cannot_take():
    import w4a16_opt as w
    p = Problem([50, 60], [1, 1], 4, 2, 128, 128, 64)
    ok = dict(q=p.q, cache=p.cache, page_table=p.table, seq_lens=p.seq_lens)

    def refused(match, **kw):
        with pytest.raises(RuntimeError, match=match):
            w.cache_attention(**{**ok, **kw})

    refused("fp16 or bf16", q=p.q.float())
    refused("last dimension", q=torch.randn(2, 128, 4, device="cuda").half().transpose(1, 2))
    refused("multiples of 8", q=torch.zeros(2, 4, 132, device="cuda").half()[:, :, :128].as_strided((2, 4, 128), (516, 129, 1)))
    refused("16-byte aligned", q=torch.zeros(2 * 4 * 128 + 8, device="cuda").half()[4:4 + 1024].view(2, 4, 128))
    refused("multiple of kv_heads", q=torch.zeros(2, 3, 128, device="cuda").half())
    refused("must be", q=torch.zeros(2, 4, 64, device="cuda").half())
    refused("one token for each sequence", q=torch.zeros(3, 4, 128, device="cuda").half())
    refused("page_table must be int32", page_table=p.table.long())
    refused("seq_lens must be int32", seq_lens=p.seq_lens[:1])
    refused("cu_q must be int32", cu_q=p.cu.long(), max_q=1)
    refused("CUDA|device", seq_lens=p.seq_lens.cpu())
    refused("window", window=-3)
    refused("out must be", out=torch.empty(2, 4, 128, device="cuda"))
    refused("workspace too small", workspace=torch.empty(256, dtype=torch.uint8, device="cuda"))
    big = torch.empty(1 << 24, dtype=torch.uint8, device="cuda")
    refused("256-byte aligned", workspace=big[16:])
    assert torch.equal(w.cache_attention(**ok, workspace=big), p.run())


def test_append_and_read_refuse_what_they_cannot_take():
    import w4a16_opt as w
    cache = w.Int4KVCache(4, 2, 128, 64)
    k = torch.zeros(3, 2, 128, device="cuda").half()
    slots = torch.arange(3, device="cuda")
    cs = torch.zeros(8, 128, device="cuda")
    pos = torch.zeros(3, dtype=torch.long, device="cuda")

    def refused(match, **kw):
        a = dict(cache=cache, k=k, v=k, slots=slots)
        a.update(kw)
        with pytest.raises(RuntimeError, match=match):
            w.cache_append(**a)

    refused("fp16 or bf16", k=k.float(), v=k.float())
    refused("one dtype", v=k.bfloat16())
    refused("k must be", k=k[:2])
    refused("v must be", v=k[:, :1])
    refused("slots must be", slots=slots.int())
    refused("go together", positions=pos)
    refused("need positions", q=k)
    refused("positions must be", positions=pos.int(), cos_sin=cs)
    refused("cos_sin must be", positions=pos, cos_sin=cs.half())
    refused("rotary_dim must be", positions=pos, cos_sin=cs[:, :96].contiguous())
    refused("need sections", positions=pos.expand(3, 3).contiguous(), cos_sin=cs)
    refused("one entry for each axis", positions=pos.expand(3, 3).contiguous(), cos_sin=cs, sections=(32, 32))
    refused("add up", positions=pos.expand(3, 3).contiguous(), cos_sin=cs, sections=(32, 32, 32))
    refused("q must be", positions=pos, cos_sin=cs, q=k.float())
    with pytest.raises(RuntimeError, match="slots must be"):
        w.cache_read(cache, slots.cpu())
    assert not cache.data.any()
