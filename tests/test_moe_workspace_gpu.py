"""GPU tests of the expert layer's workspace: a prompt's goes back to the allocator, in a graph too."""
import pytest
import torch

from test_moe_experts_gpu import make

pytestmark = pytest.mark.gpu


def layer(T):
    from w4a16_opt import moe_experts
    c = make(T, 4, 2, 512, 256, 128, 64, seed=41)
    g = {n: t.cuda() for n, t in c.items() if isinstance(t, torch.Tensor)}
    return g, lambda **kw: moe_experts(g["x"], (g["w1"], g["s1"]), (g["w2"], g["s2"]), g["experts"], g["weights"], **kw)


def test_a_prompts_workspace_is_not_kept(cuda_device):
    g, call = layer(13000)                  # 26000 entries of 3584 bytes: 93 MB
    out = torch.empty_like(g["x"])
    call(out=out)
    torch.cuda.synchronize()
    before, first = torch.cuda.memory_allocated(), out.clone()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    call(out=out)
    assert torch.cuda.max_memory_allocated() - before > 80 << 20       # the call did take one
    assert torch.cuda.memory_allocated() == before
    others = [torch.full((20 << 20,), 255, dtype=torch.uint8, device="cuda") for _ in range(6)]      # its memory, used again at once
    torch.cuda.synchronize()
    assert torch.equal(out, first)
    del others
    # a given one is used as before
    ws = torch.empty(1 << 27, dtype=torch.uint8, device="cuda")
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    call(out=out, workspace=ws)
    assert torch.cuda.max_memory_allocated() == before and torch.equal(out, first)


def test_two_graphs_of_prompts_on_two_streams(cuda_device):
    """Each capture's workspace is its graph's own, though both are captured on one stream: replayed side by side, both are right."""
    layers = [layer(13000), layer(12000)]
    want = [call().clone() for _, call in layers]
    capture, graphs, outs = torch.cuda.Stream(), [], []
    capture.wait_stream(torch.cuda.current_stream())
    for _, call in layers:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(capture), torch.cuda.graph(graph, stream=capture):
            outs.append([call() for _ in range(3)])
        graphs.append(graph)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for ys, y in zip(outs, want):
        assert all(torch.equal(t, y) for t in ys)
