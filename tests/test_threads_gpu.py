"""Calls from threads that have used no CUDA before: tensors from torch's cache need none, so the call is the thread's first."""
import threading

import pytest
import torch

from flydsl_examples_b200.gemm_a16w16 import check_status, gemm_a16w16
from flydsl_examples_b200.gemm_a8w8 import gemm_a8w8, linear_a8w8, quantize_a8
from flydsl_examples_b200.moe_a16w16 import moe_a16w16

pytestmark = pytest.mark.gpu


def in_thread(call):
    got = []

    def work():
        try:
            got.append(call())
        except Exception as e:
            got.append(e)
    t = threading.Thread(target=work)
    t.start()
    t.join()
    return got[0]


@pytest.mark.parametrize("name", ["gemm_a16w16", "split_k", "gemm_a8w8", "quantize_a8", "linear_a8w8", "moe_a16w16"])
def test_first_call_of_a_thread(name):
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(8, 256, generator=g, device="cuda").to(torch.bfloat16)
    w = torch.randn(64, 256, generator=g, device="cuda").to(torch.bfloat16)
    logits = torch.randn(8, 4, generator=g, device="cuda")
    w13 = torch.randn(4, 128, 256, generator=g, device="cuda").to(torch.bfloat16)
    w2 = torch.randn(4, 256, 64, generator=g, device="cuda").to(torch.bfloat16)
    (q, s), (wq, sw) = quantize_a8(x), quantize_a8(w, "block")
    call = {
        "gemm_a16w16": lambda: gemm_a16w16(x, w.t()),
        "split_k": lambda: gemm_a16w16(x, w.t(), user_kwargs={"tile_n": 64, "split_k": 2}),
        "gemm_a8w8": lambda: gemm_a8w8(q, s, wq.t(), sw.t()),
        "quantize_a8": lambda: quantize_a8(x)[1],
        "linear_a8w8": lambda: linear_a8w8(x, w),
        "moe_a16w16": lambda: moe_a16w16(x, logits, w13, w2, 2),
    }[name]
    want = call().clone()  # also leaves blocks of the sizes it needs in torch's cache
    torch.cuda.synchronize()
    got = in_thread(call)
    assert isinstance(got, torch.Tensor), got
    assert torch.equal(got, want)
    check_status()
