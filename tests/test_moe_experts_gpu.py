"""GPU tests of the expert layer against its formula in 64 bits on the CPU.

Tolerances, before the first run.  A sum of K products in fp32 by tensor cores is off by at most (K / 16 + 12) 2^-22 S, S the
sum of the products' sizes (each step of 16, each join of partial sums, each scaling loses at most two units of 2^-23 of what it
adds to).
Activations have slope at most 1.13 and 2^-18 of their own; the inner results are rounded to fp16 (2^-11 relative, 2^-25
absolute), the result once more; the weighted sum of k products loses (k + 2) 2^-23 of its terms' sizes.
"""
import numpy as np
import pytest
import torch

from oracle import w4a16_oracle as oracle
from test_linear_gpu import act64

pytestmark = pytest.mark.gpu

# tokens, experts, k, hidden, inner, groups of both products
SHAPES = [(1, 1, 1, 64, 64, 64, 64), (1, 8, 2, 256, 192, 128, 64), (1, 128, 8, 512, 128, 128, 128), (3, 4, 4, 384, 320, 128, 64), (5, 3, 1, 64, 1216, 64, 64),
          (8, 16, 2, 1024, 512, 128, 128), (33, 64, 6, 256, 128, 64, 128), (20, 8, 3, 512, 448, 128, 64), (70, 5, 2, 384, 384, 64, 128),
          (200, 12, 4, 256, 128, 128, 64), (700, 8, 2, 128, 192, 64, 64),
          (200, 128, 8, 64, 64, 64, 64), (2, 40, 32, 128, 64, 64, 64), (40, 40, 32, 64, 128, 64, 128), (120, 6, 2, 448, 320, 64, 64), (31, 1, 1, 64, 64, 64, 64)]


def make(T, E, k, H, I, G1, G2, seed=0):
    """A layer and a call's inputs, drawn on the CPU: dict of CPU tensors, codes beside the packed words."""
    from w4a16_opt import pack_int4
    gen = torch.Generator().manual_seed(seed + T + E + H + I)
    q1 = torch.randint(0, 16, (E, 2 * I, H), generator=gen, dtype=torch.uint8)
    q2 = torch.randint(0, 16, (E, H, I), generator=gen, dtype=torch.uint8)
    s1 = ((0.2 + torch.rand(E, H // G1, 2 * I, generator=gen)) / (4 * H ** 0.5)).half()
    s2 = ((0.2 + torch.rand(E, I // G2, H, generator=gen)) / (4 * I ** 0.5)).half()
    experts = torch.stack([torch.randperm(E, generator=gen)[:k] for _ in range(T)]).int() if T else torch.zeros(0, k).int()
    return dict(x=torch.randn(T, H, generator=gen).half(), q1=q1, s1=s1, q2=q2, s2=s2, experts=experts,
                weights=torch.softmax(torch.randn(T, k, generator=gen), -1), residual=torch.randn(T, H, generator=gen).half(),
                w1=torch.stack([pack_int4(q) for q in q1]), w2=torch.stack([pack_int4(q) for q in q2]), groups=(G1, G2))


def dequantised(q, s, G):
    return (q.double() - 8) * s.double().t().repeat_interleave(G, 1)


def expected(c, activation="silu", residual=False):
    """(y in 64 bits, what it may be off by)."""
    x, E = c["x"].double(), c["q1"].shape[0]
    T, H = x.shape
    k, I = c["experts"].shape[1], c["q2"].shape[2]
    y, d, size = torch.zeros(T, H).double(), torch.zeros(T, H).double(), torch.zeros(T, H).double()
    for e in range(E):
        token, slot = (c["experts"] == e).nonzero(as_tuple=True)
        if not token.numel():
            continue
        W1, W2 = dequantised(c["q1"][e], c["s1"][e], c["groups"][0]), dequantised(c["q2"][e], c["s2"][e], c["groups"][1])
        z, S = x[token] @ W1.t(), x[token].abs() @ W1.abs().t()
        dz = (H / 16 + 12) * 2.0 ** -22 * S
        pick = lambda t, i: t.view(len(token), -1, 2, 8)[:, :, i].reshape(len(token), -1)      # noqa: E731
        zg, zu, dg, du = pick(z, 0), pick(z, 1), pick(dz, 0), pick(dz, 1)
        a = act64(zg, activation)
        h = a * zu
        dh = 1.13 * dg * (zu.abs() + du) + a.abs() * du + 2.0 ** -18 * h.abs()
        dh = dh + 2.0 ** -11 * (h.abs() + dh) + 2.0 ** -25
        out, S2 = h @ W2.t(), (h.abs() + dh) @ W2.abs().t()
        do = dh @ W2.abs().t() + (I / 16 + 12) * 2.0 ** -22 * S2
        w = c["weights"][token, slot, None].double()
        y.index_add_(0, token, w * out)
        d.index_add_(0, token, w.abs() * do)
        size.index_add_(0, token, (w * out).abs())
    if residual:
        y, size = y + c["residual"].double(), size + c["residual"].double().abs()
    d = d + (k + 2) * 2.0 ** -23 * size
    return y, d * 1.001 + 2.0 ** -11 * (y.abs() + d) + 2.0 ** -25


def run(c, activation="silu", residual=False, **kw):
    from w4a16_opt import moe_experts
    g = {n: t.cuda() for n, t in c.items() if isinstance(t, torch.Tensor)}
    return moe_experts(g["x"], (g["w1"], g["s1"]), (g["w2"], g["s2"]), g["experts"], g["weights"], activation=activation,
                       residual=g["residual"] if residual else None, **kw)


def check(c, y, **kw):
    ref, tol = expected(c, **kw)
    assert y.dtype == torch.float16 and y.shape == ref.shape
    off = (y.cpu().double() - ref).abs() / tol
    assert bool((off <= 1).all()), off.max()


@pytest.mark.parametrize("activation,residual", [("silu", False), ("gelu", True), ("gelu_tanh", False), ("relu", True), (None, True)])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_experts(cuda_device, shape, activation, residual):
    c = make(*shape)
    check(c, run(c, activation, residual), activation=activation, residual=residual)


@pytest.mark.parametrize("T", [2, 9, 40, 150])
def test_uneven_loads(cuda_device, T):
    """All tokens to one expert; one expert that nobody chose; the same expert twice for a token."""
    c = make(T, 6, 2, 256, 192, 128, 64, seed=1)
    c["experts"][:, 0] = 5
    c["experts"][:, 1] = torch.arange(T) % 3
    c["experts"][-1] = 4
    check(c, run(c, residual=True), residual=True)


@pytest.mark.parametrize("T", [1, 12, 130])
def test_experts_outside_the_layer_add_nothing(cuda_device, T):
    c = make(T, 7, 3, 128, 128, 64, 64, seed=2)
    gen = torch.Generator().manual_seed(T)
    bad = torch.tensor([-1, 7, 1000, -(1 << 31), (1 << 31) - 1]).int()
    where = torch.rand(T, 3, generator=gen) < 0.5
    c["experts"][where] = bad[torch.randint(0, 5, (int(where.sum()),), generator=gen)]
    c["weights"][where] = float("nan")
    c["experts"][0] = -1
    ref = dict(c, weights=c["weights"].nan_to_num(0.0))
    y = run(c, residual=True)
    check(ref, y, residual=True)
    assert torch.equal(y[0].cpu(), c["residual"][0])
    c["experts"][:] = -1
    assert (run(c) == 0).all() and torch.equal(run(c, residual=True).cpu(), c["residual"])


@pytest.mark.parametrize("T", [1, 50, 300])
def test_in_place_and_no_tokens(cuda_device, T):
    from w4a16_opt import moe_experts
    c = make(T, 8, 2, 256, 128, 128, 128, seed=3)
    y = run(c, residual=True)
    g = {n: t.cuda() for n, t in c.items() if isinstance(t, torch.Tensor)}
    call = lambda x, **kw: moe_experts(x, (g["w1"], g["s1"]), (g["w2"], g["s2"]), g["experts"], g["weights"], **kw)     # noqa: E731
    r = g["residual"].clone()
    assert call(g["x"], residual=r, out=r).data_ptr() == r.data_ptr() and torch.equal(r, y)
    x = g["x"].clone()
    call(x, residual=g["residual"], out=x)
    assert torch.equal(x, y)
    ws = torch.full((1 << 26,), 255, dtype=torch.uint8, device="cuda")        # scratch of any contents
    assert torch.equal(call(g["x"], residual=g["residual"], workspace=ws), y)
    empty = moe_experts(g["x"][:0], (g["w1"], g["s1"]), (g["w2"], g["s2"]), g["experts"][:0], g["weights"][:0])
    assert empty.shape == (0, 256)


@pytest.mark.parametrize("T", [6, 100])
def test_a_bad_row_stays_in_its_row(cuda_device, T):
    c = make(T, 4, 2, 128, 128, 64, 64, seed=4)
    clean = run(c)
    c["x"][1, 5], c["x"][3, 7] = float("nan"), float("inf")
    y = run(c)
    keep = [t for t in range(T) if t not in (1, 3)]
    assert y[1].isnan().all() and not y[3].isfinite().all() and torch.equal(y[keep], clean[keep])


@pytest.mark.parametrize("T", [4, 90])
def test_captured_while_routes_change(cuda_device, T):
    from w4a16_opt import moe_experts
    c = make(T, 16, 2, 256, 128, 128, 64, seed=5)
    g = {n: t.cuda() for n, t in c.items() if isinstance(t, torch.Tensor)}
    call = lambda: moe_experts(g["x"], (g["w1"], g["s1"]), (g["w2"], g["s2"]), g["experts"], g["weights"])     # noqa: E731
    call()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
        y = call()
    for seed in range(3):
        other = make(T, 16, 2, 256, 128, 128, 64, seed=50 + seed)
        g["experts"].copy_(other["experts"] if seed else torch.zeros_like(other["experts"]))
        g["x"].copy_(other["x"])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, call())


def test_streams_side_by_side(cuda_device):
    cases = [make(30, 8, 2, 512, 256, 128, 64, seed=s) for s in range(3)]
    alone = [run(c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    from w4a16_opt import moe_experts
    gpu = [{n: t.cuda() for n, t in c.items() if isinstance(t, torch.Tensor)} for c in cases]
    torch.cuda.synchronize()
    results = []
    for _ in range(5):
        for g, s in zip(gpu, streams):
            with torch.cuda.stream(s):
                results.append(moe_experts(g["x"], (g["w1"], g["s1"]), (g["w2"], g["s2"]), g["experts"], g["weights"]))
    torch.cuda.synchronize()
    for i, y in enumerate(results):
        assert torch.equal(y, alone[i % 3])


def test_refusals(cuda_device):
    from w4a16_opt import moe_experts
    c = make(4, 4, 2, 128, 64, 64, 64, seed=6)
    g = {n: t.cuda() for n, t in c.items() if isinstance(t, torch.Tensor)}

    def refused(match, **kw):
        a = dict(x=g["x"], gate_up=(g["w1"], g["s1"]), down=(g["w2"], g["s2"]), experts=g["experts"], weights=g["weights"])
        a.update(kw)
        with pytest.raises(RuntimeError, match=match):
            moe_experts(**a)

    refused("x must be", x=g["x"].bfloat16())
    refused("x must be", x=g["x"].cpu())
    refused("scales must be", gate_up=(g["w1"], g["s1"].float()))
    refused("gated words", gate_up=(g["w1"][:, :-1].contiguous(), g["s1"]))
    refused("second product's words", down=(g["w2"][:3], g["s2"]))
    refused("second product's scales", down=(g["w2"], g["s2"][:3]))
    refused("experts must be", experts=g["experts"].long())
    refused("experts must be", experts=g["experts"][:3])
    refused("weights must be", weights=g["weights"].half())
    refused("weights must be", weights=g["weights"][:, :1].contiguous())
    refused("residual must be", residual=g["residual"][:3])
    refused("out must be", out=g["residual"].float())
    refused("activation must be", activation="tanh")
    refused("apart from every input", out=g["s2"].view(-1)[:4 * 128].view(4, 128))
    refused("workspace too small", workspace=torch.zeros(256, dtype=torch.uint8, device="cuda"))


@pytest.mark.parametrize("T", [2, 900])
def test_weights_past_4_gb(cuda_device, T):
    """The last expert of a layer of 5 GB gives what it gives alone: few entries, and more than 14 for each expert."""
    from w4a16_opt import moe_experts
    E, H, I = 60, 4096, 14336
    gen = torch.Generator(device="cuda").manual_seed(1)
    words = lambda n: torch.randint(-(1 << 31), 1 << 31, (E, n), dtype=torch.int32, device="cuda", generator=gen)      # noqa: E731
    scales = lambda *s: ((0.5 + torch.rand(*s, device="cuda", generator=gen)) / 500).half()                            # noqa: E731
    gate_up, down = (words(2 * I * H // 8), scales(E, H // 128, 2 * I)), (words(H * I // 8), scales(E, I // 128, H))
    x = torch.randn(T, H, device="cuda", generator=gen).half()
    last, ones = torch.full((T, 1), E - 1, dtype=torch.int32, device="cuda"), torch.ones(T, 1, device="cuda")
    y = moe_experts(x, gate_up, down, last, ones).float()
    alone = moe_experts(x, tuple(t[-1:] for t in gate_up), tuple(t[-1:] for t in down), torch.zeros_like(last), ones).float()
    # the same sums, perhaps in other pieces of K: half a step of fp16 each, and the inner results are the same
    assert bool(((y - alone).abs() <= 2.0 ** -10 * alone.abs() + 2.0 ** -16 * alone.abs().max()).all()) and float(alone.abs().max()) > 0.1
