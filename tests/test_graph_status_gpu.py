"""Captured calls: the status block of a stream that is first used then, and workspaces of graphs that are replayed in any order and at once."""
import pytest
import torch

from flydsl_examples_b200 import gemm_a16w16 as module
from flydsl_examples_b200.gemm_a16w16 import check_status, gemm_a16w16
from flydsl_examples_b200.gemm_a8w8 import gemm_a8w8, linear_a8w8, quantize_a8
from flydsl_examples_b200.moe_a16w16 import moe_a16w16

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["gemm_a16w16", "gemm_a8w8", "linear_a8w8", "moe_a16w16"])
def test_status_of_a_stream_first_used_in_a_capture(name):
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(8, 256, generator=g, device="cuda").to(torch.bfloat16)
    w = torch.randn(64, 256, generator=g, device="cuda").to(torch.bfloat16)
    logits = torch.randn(8, 4, generator=g, device="cuda")
    w13 = torch.randn(4, 128, 256, generator=g, device="cuda").to(torch.bfloat16)
    w2 = torch.randn(4, 256, 64, generator=g, device="cuda").to(torch.bfloat16)
    (q, s), (wq, sw) = quantize_a8(x), quantize_a8(w, "block")
    call = {
        "gemm_a16w16": lambda: gemm_a16w16(x, w.t()),
        "gemm_a8w8": lambda: gemm_a8w8(q, s, wq.t(), sw.t()),
        "linear_a8w8": lambda: linear_a8w8(x, w),
        "moe_a16w16": lambda: moe_a16w16(x, logits, w13, w2, 2),
    }[name]
    want = call().clone()
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    for key in [k for k in module._workspaces if k[1] == stream.cuda_stream]:  # torch hands its streams out again
        del module._workspaces[key]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = call()
    status = module._workspaces[torch.cuda.current_device(), stream.cuda_stream].status
    torch.cuda.synchronize()
    assert not status.any()  # before the first replay
    graph.replay()
    check_status()
    assert torch.equal(got, want)
    status[0] = 1  # as a kernel that gave up leaves it: later replays do not hide it
    graph.replay()
    with pytest.raises(RuntimeError, match="gave up"):
        check_status()
    check_status()


def test_graphs_of_split_k_and_repacked_products():
    g = torch.Generator(device="cuda").manual_seed(2)

    def problem(m, n, k, pad, **kw):
        a, b = (torch.randn(r, k + pad, generator=g, device="cuda").to(torch.bfloat16)[:, :k] for r in (m, n))
        out = torch.empty(m, n, device="cuda")
        return lambda: gemm_a16w16(a, b.t(), out, user_kwargs=kw, out_dtype=torch.float32)
    problems = [problem(96, 320, 2048, 0, tile_n=128, split_k=8), problem(200, 264, 2048, 0, tile_n=64, split_k=4), problem(1000, 1100, 300, 1),
                problem(33, 640, 1030, 5, tile_n=64, split_k=3), problem(300, 4000, 1000, 0, tile_n=128, stream_k=True)]
    stream = torch.cuda.Stream()
    outs, want = [], []
    with torch.cuda.stream(stream):
        for p in problems:  # resolved on the stream before it is captured
            outs.append(p())
            want.append(outs[-1].clone())
    torch.cuda.synchronize()
    dirty = torch.full((256 << 20,), 0x5A, dtype=torch.uint8, device="cuda")
    del dirty
    torch.cuda.empty_cache()  # what the graphs' pools get is not clear
    graphs = []
    for p in problems:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=stream):
            p()
    larger = problem(3000, 3000, 500, 1)  # the stream's workspace is replaced
    with torch.cuda.stream(stream):
        larger()
    torch.cuda.synchronize()

    def check():
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
        for o in outs:
            o.fill_(float("nan"))
        torch.cuda.synchronize()
    check()
    for graph in reversed(graphs):
        graph.replay()
    check()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(20):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    check()
    with torch.cuda.stream(stream):
        for p in problems:
            p()
    check()
    check_status()
