"""A mixture-of-experts layer for a few tokens (decoding), from the router's logits to the layer's output.

    logits = gemm_a16w16(x, w_router, out_dtype=torch.float32)      # the router's product
    y = moe_a16w16(x, logits, w13, w2, top_k)

Two kernels of libb200_gemm.so (hand-written sm_100a CUDA) read the weights of the chosen experts once; there is no CPU path.
"""
from __future__ import annotations

import struct
from typing import Optional

import torch

from . import _lib
from ._launch import on_device, raw_stream
from .gemm_a16w16 import _workspace_for

MAX_TOKENS, MAX_EXPERTS, MAX_TOP_K = 64, 512, 16
_IDS = {torch.float32: _lib.DTYPE_FP32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16}
_KWARGS = ("wait_limit_us", "pdl")

_ARGS = struct.Struct("@5P12q6iPQP")  # b200_gemm_moe_args


def _check_matrix(name: str, t: torch.Tensor, shape: tuple) -> None:
    if t.shape != shape:
        raise ValueError(f"{name} must be {shape}, got {tuple(t.shape)}")
    strides = t.stride()
    ok = strides[-1] == 1 and t.data_ptr() % 16 == 0 and (shape[-2] == 1 or strides[-2] % 8 == 0 and strides[-2] >= shape[-1])
    if ok and len(shape) == 3 and shape[0] > 1:
        ok = strides[0] % 8 == 0 and strides[0] >= (shape[1] - 1) * strides[1] + shape[2]
    if not ok:
        raise ValueError(f"{name} must have contiguous rows on 16-byte boundaries (strides that are multiples of 8 elements); "
                         f"got shape={tuple(t.shape)} and stride={strides}")


def _scratch_bytes(t: int, i: int, e: int, top_k: int) -> int:
    """b200_gemm_moe_workspace_bytes: the list of chosen experts, and h for each that t tokens can choose."""
    return 4096 + 4 * min(t * top_k, e) * t * i


def _arguments(x, logits, w13, w2, top_k, out, renormalize, user_kwargs, workspace, workspace_bytes, status) -> bytes:
    """Checks the tensors and packs a b200_gemm_moe_args."""
    assert x.ndim == 2 and logits.ndim == 2 and w13.ndim == 3 and w2.ndim == 3
    t, h = x.shape
    e, i2, _ = w13.shape
    i = i2 // 2
    for key in user_kwargs:
        if key not in _KWARGS:
            raise ValueError(f"unknown moe_a16w16 key {key!r}; expected some of {_KWARGS}")
    dtype = x.dtype
    if dtype not in (torch.bfloat16, torch.float16) or w13.dtype != dtype or w2.dtype != dtype or out.dtype != dtype:
        raise ValueError(f"moe_a16w16 takes x, w13, w2 and out of one 16-bit type, got {dtype}, {w13.dtype}, {w2.dtype}, {out.dtype}")
    if logits.dtype not in _IDS:
        raise ValueError(f"logits must be float32, bfloat16 or float16, not {logits.dtype}")
    device = x.device
    if logits.device != device or w13.device != device or w2.device != device or out.device != device:
        raise ValueError("moe_a16w16's tensors are on different devices")
    if t > MAX_TOKENS or e > MAX_EXPERTS or not 1 <= top_k <= min(MAX_TOP_K, e):
        raise ValueError(f"moe_a16w16 serves up to {MAX_TOKENS} tokens, {MAX_EXPERTS} experts and top_k up to {MAX_TOP_K} (and the number "
                         f"of experts); got {t} tokens, {e} experts, top_k {top_k}")
    if i2 % 2 or h % 8 or i % 8 or not h or not i:
        raise ValueError(f"hidden and inner sizes must be multiples of 8, got hidden {h} and w13 with {i2} rows")
    if logits.shape != (t, e):
        raise ValueError(f"logits must be {(t, e)}, got {tuple(logits.shape)}")
    _check_matrix("w13", w13, (e, 2 * i, h))
    _check_matrix("w2", w2, (e, h, i))
    if t:
        _check_matrix("x", x, (t, h))
    assert out.is_contiguous() and out.shape == x.shape, f"out must be contiguous {(t, h)}, got {tuple(out.shape)}"
    return _ARGS.pack(
        x.data_ptr(), logits.data_ptr(), w13.data_ptr(), w2.data_ptr(), out.data_ptr(),
        t, h, i, e, x.stride(0) if t > 1 else h, *logits.stride(), *w13.stride()[:2], *w2.stride()[:2], h,
        top_k, bool(renormalize), _IDS[dtype], _IDS[logits.dtype], user_kwargs.get("wait_limit_us", 0), 0 if user_kwargs.get("pdl", True) else 1,
        workspace, workspace_bytes, status)


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
    remainder.

    An expert of weight zero (a logit of -inf) is not evaluated, a token whose logits are all -inf gets zeros, a NaN logit
    makes its token's row NaN. Non-finite values in a chosen expert's weights reach every token of the call.
    user_kwargs: wait_limit_us, pdl. Asynchronous on `stream`; `gemm_a16w16.check_status` reports abandoned waits."""
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if not x.is_cuda:
        _arguments(x, logits, w13, w2, top_k, out, renormalize, user_kwargs, 0, 0, 0)
        raise AssertionError("moe_a16w16 runs on CUDA tensors only (there is no CPU path)")
    device = x.device
    index = device.index
    with on_device(index, stream):
        stream_ptr = raw_stream(index)
        ws = _workspace_for(device, stream_ptr)
        need = _scratch_bytes(x.shape[0], w2.shape[-1], w13.shape[0], top_k) if w2.ndim == 3 and w13.ndim == 3 else 0
        if torch.cuda.is_current_stream_capturing():
            # a graph keeps scratch of its own (its memory pool's), so that two graphs may run at once
            scratch = torch.empty(max(need, 256), dtype=torch.uint8, device=device)
            at = scratch.data_ptr()
        else:
            # behind the split-K tickets that the 16-bit GEMM keeps at the start of the stream's workspace
            if ws.buf is None or ws.buf.numel() < _lib.COUNTER_BYTES + need:
                ws.ensure(_lib.COUNTER_BYTES + need, device, torch.cuda.current_stream(index))
            at = ws.buf.data_ptr() + _lib.COUNTER_BYTES
        args = _arguments(x, logits, w13, w2, top_k, out, renormalize, user_kwargs, at, need, ws.status_ptr)
        if x.shape[0] == 0:
            return out
        rc = _lib.fast("b200_gemm_moe_a16w16")(args, stream_ptr)
    if rc != 0:
        raise RuntimeError(f"b200_gemm_moe_a16w16 failed ({rc}): {_lib.strerror(rc)}")
    return out
