"""A mixture-of-experts layer for a few tokens (decoding), from the router's logits to the layer's output.

    logits = gemm_a16w16(x, w_router, out_dtype=torch.float32)      # the router's product
    y = moe_a16w16(x, logits, w13, w2, top_k)

Two kernels of libb200_gemm.so (hand-written sm_100a CUDA) read the weights of the chosen experts once; there is no CPU path.
"""
from __future__ import annotations

import functools
import struct
from typing import Optional

import torch

from . import _lib
from ._launch import on_device, raw_stream
from .gemm_a16w16 import _workspace_for

MAX_TOKENS, MAX_EXPERTS, MAX_TOP_K = 64, 512, 16
_IDS = {torch.float32: _lib.DTYPE_FP32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16}
_KWARGS = ("wait_limit_us", "pdl")

# b200_gemm_moe_args in parts; the last member is the status address
_POINTERS, _SIZES, _SCRATCH = struct.Struct("@5P"), struct.Struct("@12q6i"), struct.Struct("@PQ")


def _check_matrix(name: str, have, strides, shape: tuple) -> None:
    if have != shape:
        raise ValueError(f"{name} must be {shape}, got {tuple(have)}")
    ok = strides[-1] == 1 and (shape[-2] == 1 or strides[-2] % 8 == 0 and strides[-2] >= shape[-1])
    if ok and len(shape) == 3 and shape[0] > 1:
        ok = strides[0] % 8 == 0 and strides[0] >= (shape[1] - 1) * strides[1] + shape[2]
    if not ok:
        raise ValueError(f"{name} must have contiguous rows on 16-byte boundaries (strides that are multiples of 8 elements); "
                         f"got shape={tuple(have)} and stride={strides}")


def _scratch_bytes(t: int, i: int, e: int, top_k: int) -> int:
    """b200_gemm_moe_workspace_bytes: the list of chosen experts, and h for each that t tokens can choose."""
    return 4096 + 4 * min(t * top_k, e) * t * i


@functools.lru_cache(maxsize=4096)
def _call_plan(x_shape, x_stride, x_dtype, l_shape, l_stride, l_dtype, w13_shape, w13_stride, w13_dtype, w2_shape, w2_stride, w2_dtype,
               out_shape, out_dtype, top_k, renormalize, kwargs) -> tuple:
    """(scratch bytes, sizes of the argument block) of a call with tensors of these shapes, strides and types; raises what the
    call raises. Everything here follows from the sizes, so a repeated call pays for it once."""
    assert len(x_shape) == len(l_shape) == 2 and len(w13_shape) == len(w2_shape) == 3, "x and logits are matrices, the weights have three dimensions"
    t, h = x_shape
    e, i2, _ = w13_shape
    i = i2 // 2
    kwargs = dict(kwargs)
    for key in kwargs:
        if key not in _KWARGS:
            raise ValueError(f"unknown moe_a16w16 key {key!r}; expected some of {_KWARGS}")
    if x_dtype not in (torch.bfloat16, torch.float16) or not x_dtype == w13_dtype == w2_dtype == out_dtype:
        raise ValueError(f"moe_a16w16 takes x, w13, w2 and out of one 16-bit type, got {x_dtype}, {w13_dtype}, {w2_dtype}, {out_dtype}")
    if l_dtype not in _IDS:
        raise ValueError(f"logits must be float32, bfloat16 or float16, not {l_dtype}")
    if t > MAX_TOKENS or e > MAX_EXPERTS or not 1 <= top_k <= min(MAX_TOP_K, e):
        raise ValueError(f"moe_a16w16 serves up to {MAX_TOKENS} tokens, {MAX_EXPERTS} experts and top_k up to {MAX_TOP_K} (and the number "
                         f"of experts); got {t} tokens, {e} experts, top_k {top_k}")
    if i2 % 2 or h % 8 or i % 8 or not h or not i:
        raise ValueError(f"hidden and inner sizes must be multiples of 8, got hidden {h} and w13 with {i2} rows")
    if l_shape != (t, e):
        raise ValueError(f"logits must be {(t, e)}, got {tuple(l_shape)}")
    _check_matrix("w13", w13_shape, w13_stride, (e, 2 * i, h))
    _check_matrix("w2", w2_shape, w2_stride, (e, h, i))
    if t:
        _check_matrix("x", x_shape, x_stride, (t, h))
    assert out_shape == x_shape, f"out must be contiguous {(t, h)}, got {tuple(out_shape)}"
    sizes = _SIZES.pack(t, h, i, e, x_stride[0] if t > 1 else h, *l_stride, *w13_stride[:2], *w2_stride[:2], h, top_k, renormalize,
                        _IDS[x_dtype], _IDS[l_dtype], kwargs.get("wait_limit_us", 0), 0 if kwargs.get("pdl", True) else 1)
    return _scratch_bytes(t, i, e, top_k), sizes


def _launch_moe(x, logits, w13, w2, out, need, sizes, index) -> torch.Tensor:
    """On the current device and stream."""
    device = x.device
    stream_ptr = raw_stream(index)
    # Scratch of this call's own, from the stream's (or a graph's) pool. Its two launches are not one step: another thread's call on
    # this stream, or a GEMM that uses the stream's workspace, may come between them. (With a buffer that the stream's calls
    # shared one token took 10.3 us of host time, it takes 12.0 so; a replayed graph pays nothing.)
    scratch = torch.empty(need, dtype=torch.uint8, device=device)
    args = (_POINTERS.pack(x.data_ptr(), logits.data_ptr(), w13.data_ptr(), w2.data_ptr(), out.data_ptr()) + sizes
            + _SCRATCH.pack(scratch.data_ptr(), need) + _workspace_for(device, stream_ptr).status_bytes)
    rc = _lib.fast("b200_gemm_moe_a16w16")(args, stream_ptr)
    if rc != 0:
        raise RuntimeError(f"b200_gemm_moe_a16w16 failed ({rc}): {_lib.strerror(rc)}")
    return out


def moe_a16w16(
    x: torch.Tensor,
    logits: torch.Tensor,
    w13: torch.Tensor,
    w2: torch.Tensor,
    top_k: int,
    out: Optional[torch.Tensor] = None,
    renormalize: bool = True,
    user_kwargs: dict = {},
    stream: Optional[torch.cuda.Stream] = None,
) -> torch.Tensor:
    """y[t] = sum over the top_k experts e of token t of p[t, e] * w2[e] @ (silu(g) * u), [g; u] = w13[e] @ x[t].

    x [T, H] with 1 to 64 tokens (0: nothing is done), logits [T, E] of the router (float32, bfloat16 or float16, any strides),
    w13 [E, 2 I, H] (gate rows, then up rows), w2 [E, H, I]; x, weights and `out` [T, H] are all bfloat16 or all float16. p is the
    softmax over all experts, ties go to the lowest index, and with `renormalize` the chosen weights are divided by their sum.
    Sums, softmax and SiLU are fp32; p * silu(g) * u, the second product's operand, is carried as a 16-bit value and a 16-bit
    remainder: to 2^-16 of it in bfloat16; in float16 to 2^-22 of it, or 2^-32 where it is below 2^-10, and infinite from 2^20 on.

    An expert of weight zero (a logit of -inf) is not evaluated, a token whose logits are all -inf gets zeros, a NaN logit
    makes its token's row NaN. Non-finite values in a chosen expert's weights reach every token of the call.
    user_kwargs: wait_limit_us, pdl. Asynchronous on `stream`; `gemm_a16w16.check_status` reports abandoned waits."""
    index = x.get_device()
    need, sizes = _call_plan(x.shape, x.stride(), x.dtype, logits.shape, logits.stride(), logits.dtype, w13.shape, w13.stride(), w13.dtype,
                             w2.shape, w2.stride(), w2.dtype, x.shape if out is None else out.shape, x.dtype if out is None else out.dtype,
                             top_k, bool(renormalize), tuple(user_kwargs.items()) if user_kwargs else ())
    if logits.get_device() != index or w13.get_device() != index or w2.get_device() != index or out is not None and out.get_device() != index:
        raise ValueError("moe_a16w16's tensors are on different devices")
    assert out is None or out.is_contiguous(), "out must be contiguous"
    if x.shape[0] and (x.data_ptr() | w13.data_ptr() | w2.data_ptr()) & 15:
        raise ValueError("x, w13 and w2 must start on a 16-byte-aligned address")
    assert index >= 0, "moe_a16w16 runs on CUDA tensors only (there is no CPU path)"
    with on_device(index, stream):
        if out is None:
            out = torch.empty_like(x, memory_format=torch.contiguous_format)
        return out if x.shape[0] == 0 else _launch_moe(x, logits, w13, w2, out, need, sizes, index)
