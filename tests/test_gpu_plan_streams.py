"""Runs of one plan on several streams: its scratch (the operands' tf32 parts)
is one per device, so a run waits for the one before, whatever stream that is on."""
import pytest
import torch

pytestmark = pytest.mark.gpu

M, N, K = 256, 512, 1152
SLABS = [0, 96, 480, 1152]


def _compile():
    import bafe_b200 as bafe
    from bafe_b200.graph import GraphBuilder
    g = GraphBuilder()
    a, b, c = (g.add_input(n, s, 0, t) for n, s, t in (("A", (M, K), 0), ("B", (K, N), 2), ("C", (M, N), 0)))
    g.set_output(g.add("relu", [g.add("add", [g.add("matmul", [a, b]), c])]))
    bafe.set_option("gemm_precision", "3xtf32")
    try:
        return bafe.compile_graph(g)
    finally:
        bafe.set_option("gemm_precision", "auto")


def test_a_run_on_another_stream_waits_for_the_one_before(cuda):
    """The first run's slices wait for an event that a long kernel holds back; the second run is enqueued meanwhile."""
    k = _compile()
    gen = torch.Generator(device="cuda").manual_seed(1)
    a = [torch.randn(M, K, device="cuda", generator=gen) for _ in range(2)]
    b = [torch.randn(K, N, device="cuda", generator=gen) for _ in range(2)]
    c = torch.randn(M, N, device="cuda", generator=gen)
    want = [torch.empty(M, N, device="cuda") for _ in range(2)]
    got = [torch.empty(M, N, device="cuda") for _ in range(2)]
    for i in range(2):
        k.run_torch_ksliced([a[i], b[i], c], want[i], SLABS)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    side = torch.cuda.Stream()
    for kind in ("sliced", "whole"):
        for t in got:
            t.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)                # some 10 ms
        held = torch.cuda.Event()
        held.record(side)
        k.run_torch_ksliced([a[0], b[0], c], got[0], SLABS, ready=[held] * 3, stream=streams[0])
        if kind == "sliced":
            k.run_torch_ksliced([a[1], b[1], c], got[1], SLABS, stream=streams[1])
        else:
            k.run_torch([a[1], b[1], c], got[1], stream=streams[1])
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), kind


def test_captured_runs_are_not_ordered_with_others(cuda):
    """A run inside a graph capture neither waits for runs outside nor is waited for; a replay gives the same bits."""
    k = _compile()
    gen = torch.Generator(device="cuda").manual_seed(2)
    a, b, c = (torch.randn(*s, device="cuda", generator=gen) for s in ((M, K), (K, N), (M, N)))
    want, got = torch.empty(M, N, device="cuda"), torch.empty(M, N, device="cuda")
    k.run_torch([a, b, c], want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        k.run_torch([a, b, c], got)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    k.run_torch([a, b, c], want.zero_(), stream=torch.cuda.Stream())
    torch.cuda.synchronize()
    assert torch.equal(got, want)
