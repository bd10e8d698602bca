"""The status block of a stream that is first used while it is captured: no part of the graph."""
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
