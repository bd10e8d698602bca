"""torch.library registration of the 8-bit product, its quantizer and the mixture-of-experts layer."""
import pytest
import torch

import flydsl_examples_b200.torch_op  # noqa: F401  (registers the operators)

F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}


def test_schemas():
    ops = torch.ops.b200
    assert "Tensor a_scale" in str(ops.gemm_a8w8.default._schema) and "str out_dtype" in str(ops.gemm_a8w8.default._schema)
    assert str(ops.quantize_a8.default._schema).endswith("-> Tensor[]")
    assert "Int top_k" in str(ops.moe_a16w16.default._schema)


def test_fake_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x = torch.empty(33, 200, dtype=torch.bfloat16)
        q, s = torch.ops.b200.quantize_a8(x, "row", "e4m3")
        w, sw = torch.ops.b200.quantize_a8(torch.empty(300, 200, dtype=torch.bfloat16), "block", "e5m2")
        assert q.shape == (33, 200) and s.shape == (33, 2) and w.dtype is torch.float8_e5m2 and sw.shape == (3, 2)
        y = torch.ops.b200.gemm_a8w8(q, s, w.t(), sw.t(), None, "nt", "fp16")
        assert y.shape == (33, 300) and y.dtype is torch.float16
        assert len(torch.ops.b200.quantize_a8(x, "both", "e4m3")) == 4
        m = torch.ops.b200.moe_a16w16(x[:4], torch.empty(4, 8), torch.empty(8, 64, 200, dtype=x.dtype), torch.empty(8, 200, 32, dtype=x.dtype), 2, True)
        assert m.shape == (4, 200) and m.dtype is torch.bfloat16


@pytest.mark.gpu
@pytest.mark.parametrize("group", ["row", "col", "both", "block"])
@pytest.mark.parametrize("shape", [(1, 5), (200, 300), (128, 256)])
def test_fake_quantizer_describes_the_real_one(group, shape):
    from torch._subclasses.fake_tensor import FakeTensorMode

    real = torch.ops.b200.quantize_a8(torch.randn(*shape, device="cuda"), group, "e4m3")
    with FakeTensorMode():
        fake = torch.ops.b200.quantize_a8(torch.empty(*shape, device="cuda"), group, "e4m3")
    for r, f in zip(real, fake, strict=True):
        assert r.shape == f.shape and r.dtype == f.dtype and (r.stride() == f.stride() or 1 in r.shape)


@pytest.mark.gpu
def test_operators_inside_torch_compile():
    from flydsl_examples_b200.gemm_a16w16 import check_status
    from flydsl_examples_b200.gemm_a8w8 import gemm_a8w8, quantize_a8
    from flydsl_examples_b200.moe_a16w16 import moe_a16w16

    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(20, 256, generator=g, device="cuda").bfloat16()
    w = torch.randn(384, 256, generator=g, device="cuda").bfloat16()
    logits = torch.randn(20, 6, generator=g, device="cuda")
    w13, w2 = torch.randn(6, 128, 256, generator=g, device="cuda").bfloat16(), torch.randn(6, 256, 64, generator=g, device="cuda").bfloat16()

    @torch.compile(fullgraph=True, backend="aot_eager")
    def f(x, w, logits, w13, w2):
        h = torch.ops.b200.moe_a16w16(x, logits, w13, w2, 2, True) * 1.0
        q, s = torch.ops.b200.quantize_a8(h, "row", "e4m3")
        wq, sw = torch.ops.b200.quantize_a8(w, "block", "e4m3")
        return torch.ops.b200.gemm_a8w8(q, s, wq.t(), sw.t(), None, "nt", "fp32")

    got = f(x, w, logits, w13, w2)
    h = moe_a16w16(x, logits, w13, w2, 2)
    q, s = quantize_a8(h)
    wq, sw = quantize_a8(w, "block")
    assert torch.equal(got, gemm_a8w8(q, s, wq.t(), sw.t(), out_dtype=torch.float32))
    check_status()
