"""`torch.library` registration of the GEMM so that it can sit inside `torch.compile`d graphs and CUDA-graph
captured decode loops as an opaque operator (no tracing into ctypes).

Plays the role the reference's benchmark gives to a "FLYDSL" inductor backend living in a PyTorch fork
(torch_benchmark.py:32-49, :62-77): there the compiler picks the kernel as a GEMM template; here the compiled graph
simply calls `torch.ops.b200.gemm_a16w16`. Importing this module registers the operator.

    import flydsl_examples_b200.torch_op            # registers torch.ops.b200.gemm_a16w16
    y = torch.ops.b200.gemm_a16w16(a, b, bias, "nt", None)

The 8-bit product, its quantizer and the few-token mixture-of-experts layer are registered the same way
(`torch.ops.b200.gemm_a8w8`, `quantize_a8`, `moe_a16w16`).
"""
from __future__ import annotations

from typing import Optional

import torch

from .gemm_a16w16 import gemm_a16w16 as _gemm
from .gemm_a8w8 import gemm_a8w8 as _gemm8, quantize_a8 as _quantize8
from .moe_a16w16 import moe_a16w16 as _moe

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


@torch.library.custom_op("b200::gemm_a16w16", mutates_args=())
def gemm_a16w16_op(a: torch.Tensor, b: torch.Tensor, bias: Optional[torch.Tensor], layout: str,
                   out_dtype: Optional[str]) -> torch.Tensor:
    """C = A @ B (+ bias). `layout` as in gemm_a16w16; `out_dtype` is None (input dtype), "fp32", "bf16" or "fp16"."""
    dt = None if out_dtype is None else _DTYPES[out_dtype]
    return _gemm(a, b, None, bias=bias, layout=layout, out_dtype=dt)


@gemm_a16w16_op.register_fake
def _(a, b, bias, layout, out_dtype):
    if layout.lower() not in ("nn", "nt", "tn", "tt"):
        raise ValueError(f"unsupported GEMM layout: {layout!r}")
    torch._check(a.dim() == 2 and b.dim() == 2)
    torch._check(a.shape[1] == b.shape[0])
    dt = a.dtype if out_dtype is None else _DTYPES[out_dtype]
    return a.new_empty((a.shape[0], b.shape[1]), dtype=dt)


_F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}


@torch.library.custom_op("b200::gemm_a8w8", mutates_args=())
def gemm_a8w8_op(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor, bias: Optional[torch.Tensor],
                 layout: str, out_dtype: str) -> torch.Tensor:
    """C = A @ B (+ bias) from 8-bit operands with block scales, see gemm_a8w8; `out_dtype` is "fp32", "bf16" or "fp16"."""
    return _gemm8(a, a_scale, b, b_scale, None, bias=bias, layout=layout, out_dtype=_DTYPES[out_dtype])


@gemm_a8w8_op.register_fake
def _(a, a_scale, b, b_scale, bias, layout, out_dtype):
    torch._check(a.dim() == 2 and b.dim() == 2)
    torch._check(a.shape[1] == b.shape[0])
    return a.new_empty((a.shape[0], b.shape[1]), dtype=_DTYPES[out_dtype])


@torch.library.custom_op("b200::quantize_a8", mutates_args=())
def quantize_a8_op(x: torch.Tensor, group: str, dtype: str) -> list[torch.Tensor]:
    """Values and scales, see quantize_a8 ("both": four tensors); `dtype` is "e4m3" or "e5m2"."""
    return list(_quantize8(x, group, _F8[dtype]))


@quantize_a8_op.register_fake
def _(x, group, dtype):
    rows, cols = x.shape
    rb, cb = (rows + 127) // 128, (cols + 127) // 128
    pitch = (cols + 15) // 16 * 16
    q = lambda: x.new_empty((rows, pitch), dtype=_F8[dtype])[:, :cols]  # noqa: E731
    s = lambda n, m: x.new_empty((m, n), dtype=torch.float32).t()  # noqa: E731
    row, col = [q(), s(rows, cb)], [q(), x.new_empty((rb, cols), dtype=torch.float32)]
    return {"row": row, "col": col, "both": row + col, "block": [q(), s(rb, cb)]}[group]


@torch.library.custom_op("b200::moe_a16w16", mutates_args=())
def moe_a16w16_op(x: torch.Tensor, logits: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor, top_k: int, renormalize: bool) -> torch.Tensor:
    """A mixture-of-experts layer for a few tokens from the router's logits, see moe_a16w16."""
    return _moe(x, logits, w13, w2, top_k, renormalize=renormalize)


@moe_a16w16_op.register_fake
def _(x, logits, w13, w2, top_k, renormalize):
    torch._check(x.dim() == 2 and logits.dim() == 2 and w13.dim() == 3 and w2.dim() == 3)
    return x.new_empty(x.shape)
