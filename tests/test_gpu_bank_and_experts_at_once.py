"""Calls on banks, their gradients, experts and routers on several streams at once, beside a captured graph of the same calls that is replayed
meanwhile: the bits of calls one after the other."""
import pytest
import torch

from kiln_amd import marlin_gemm
from tests.test_gpu_bank import backward, bits, forward, problem
from tests.test_gpu_moe import layer

pytestmark = pytest.mark.gpu


def calls(seed):
    banks = [problem(m, k, n, 128, 7, 24, "any", seed=seed) for m, k, n in ((1, 2560, 2560), (16, 2560, 5120), (40, 1024, 512), (150, 2560, 2560), (400, 512, 2560), (2100, 640, 8192))]
    experts = [layer(m, 4, 16, 512, 384, 512, 128, seed=seed) for m in (1, 13, 70)]
    logits = torch.randn(300, 96, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))

    def run():
        made = []
        for p in banks:
            made += bits((forward(p), *backward(p)))
        for a in experts:
            made += bits(marlin_gemm.marlin_w4a16_moe(*a))
        return made + [t.clone() for t in marlin_gemm.moe_route(logits, 8)]

    return run


def same(a, b):
    return len(a) == len(b) and all(map(torch.equal, a, b))


def test_streams_and_a_graph_at_once():
    runs = [calls(seed) for seed in range(3)]
    want = [run() for run in runs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for s, run in zip(streams, runs):
        with torch.cuda.stream(s):
            run()                               # the stream's workspace
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[2]):
        captured = runs[2]()
    for _ in range(4):
        for t in captured:
            t.zero_()
        torch.cuda.synchronize()
        made = [[], []]
        with torch.cuda.stream(streams[2]):
            graph.replay()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                made[i] = runs[i]()
        torch.cuda.synchronize()
        assert same(made[0], want[0]) and same(made[1], want[1]) and same(captured, want[2])
