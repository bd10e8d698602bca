"""Calls from several threads, on one stream and as the first CUDA work of a thread."""
import threading

import pytest
import torch

from flydsl_examples_b200 import gemm_a16w16 as module
from flydsl_examples_b200.gemm_a16w16 import check_status, gemm_a16w16
from flydsl_examples_b200.gemm_a8w8 import gemm_a8w8, linear_a8w8, quantize_a8
from flydsl_examples_b200.moe_a16w16 import moe_a16w16

pytestmark = pytest.mark.gpu


def in_thread(call):
    # a thread that has used no CUDA before: tensors from torch's cache need none, so the call is its first
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


def test_16_bit_gemms_that_are_not_repeats():
    # every call without `out` is resolved anew; repacked operands, partial tiles and tickets lie in the stream's one workspace, which
    # grows meanwhile
    g = torch.Generator(device="cuda").manual_seed(2)

    def problem(m, n, k, pad, **kw):
        a, b = (torch.randn(r, k + pad, generator=g, device="cuda").to(torch.bfloat16)[:, :k] for r in (m, n))
        return lambda: gemm_a16w16(a, b.t(), user_kwargs=kw, out_dtype=torch.float32)
    problems = [problem(96, 320, 2048, 0, tile_n=128, split_k=8), problem(200, 264, 500, 3), problem(1000, 1100, 300, 1), problem(33, 640, 1030, 5)]
    want = [p() for p in problems]
    torch.cuda.synchronize()
    with module._ws_lock:
        for ws in module._workspaces.values():  # small again
            ws.buf, ws.generation = None, ws.generation + 1
    module.clear_prepared_calls()
    bad, go = [], threading.Barrier(len(problems))

    def work(i):
        try:
            go.wait()
            bad.extend(i for y in [problems[i]() for _ in range(100)] if not torch.equal(y, want[i]))
        except Exception as e:
            bad.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(problems))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
    check_status()
