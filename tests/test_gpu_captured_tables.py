"""A packed call recorded into a graph, replayed after many other packed batches: its table is where it was."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_replays_after_other_batches(gpu_device):
    from oracle import palimpsa_oracle as po
    from palimpsa_amd.ops.palimpsa import chunk_palimpsa
    from palimpsa_amd.ops.short_conv import short_conv

    gen = torch.Generator().manual_seed(2)
    T, D = 300, 64
    x, w = torch.randn(1, T, D, generator=gen).to(gpu_device), torch.randn(D, 4, generator=gen).to(gpu_device)
    inp = {n: t.float().to(gpu_device) for n, t in po.make_inputs(1, T, 2, 16, 16, seed=1).items() if n in ("q", "k", "v", "b", "gt", "g", "Ip")}
    cu = torch.tensor([0, 3, 80, 200, T], dtype=torch.int32, device=gpu_device)

    def call():
        with torch.no_grad():
            return short_conv(x, w, cu_seqlens=cu)[0], chunk_palimpsa(*[inp[n] for n in ("q", "k", "v", "b", "gt", "g", "Ip")], cu_seqlens=cu)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for k in range(3):
        others = [torch.tensor([0, 1 + i + 20 * k, T], dtype=torch.int32, device=gpu_device) for i in range(20)]
        for o in others:
            short_conv(x, w, cu_seqlens=o)
        taken = [torch.full((64,), -1, dtype=torch.int32, device=gpu_device) for _ in range(64)]
        x.mul_(-0.5)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, call()):
            assert torch.equal(a, b), k
        assert all((t == -1).all() for t in taken)
