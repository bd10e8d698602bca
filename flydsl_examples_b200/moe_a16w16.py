"""A mixture-of-experts layer for a few tokens (decoding), from the router's logits to the layer's output.

    logits = gemm_a16w16(x, w_router, out_dtype=torch.float32)      # the router's product
    y = moe_a16w16(x, logits, w13, w2, top_k)

Two kernels of libb200_gemm.so (hand-written sm_100a CUDA) read the weights of the chosen experts once; there is no CPU path.
"""
from __future__ import annotations

import ctypes as C
import threading
from collections import OrderedDict
from typing import Optional

import torch

from . import _lib
from .gemm_a16w16 import _workspace_for

MAX_TOKENS, MAX_EXPERTS, MAX_TOP_K = 64, 512, 16
_IDS = {torch.float32: _lib.DTYPE_FP32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16}
_KWARGS = ("wait_limit_us", "pdl")

_PREPARED_MAX = 512
_prepared: "OrderedDict[tuple, tuple]" = OrderedDict()
_prepared_lock = threading.Lock()


def clear_prepared_calls() -> None:
    """Drop every cached launch handle."""
    with _prepared_lock:
        items = list(_prepared.values())
        _prepared.clear()
    for ent in items:
        _lib.load().b200_gemm_moe_release(ent[0])


def _check_matrix(name: str, t: torch.Tensor, shape: tuple) -> None:
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} must be {shape}, got {tuple(t.shape)}")
    strides_ok = t.stride(-1) == 1 and all(n == 1 or s % 8 == 0 for n, s in zip(t.shape[:-1], t.stride()[:-1]))
    rows_ok = t.shape[-2] == 1 or t.stride(-2) >= t.shape[-1]
    if t.ndim == 3 and t.shape[0] > 1:
        rows_ok = rows_ok and t.stride(0) >= (t.shape[1] - 1) * t.stride(1) + t.shape[2]
    if not strides_ok or not rows_ok or t.data_ptr() % 16 != 0:
        raise ValueError(f"{name} must have contiguous rows on 16-byte boundaries (strides that are multiples of 8 elements); "
                         f"got shape={tuple(t.shape)} and stride={t.stride()}")


def _fill_args(x, logits, w13, w2, top_k, out, renormalize, user_kwargs) -> _lib.MoeArgs:
    assert x.ndim == 2 and logits.ndim == 2 and w13.ndim == 3 and w2.ndim == 3
    t, h = x.shape
    e, i2, _ = w13.shape
    i = i2 // 2
    for key in user_kwargs:
        if key not in _KWARGS:
            raise ValueError(f"unknown moe_a16w16 key {key!r}; expected some of {_KWARGS}")
    if x.dtype not in (torch.bfloat16, torch.float16) or w13.dtype != x.dtype or w2.dtype != x.dtype or out.dtype != x.dtype:
        raise ValueError(f"moe_a16w16 takes x, w13, w2 and out of one 16-bit type, got {x.dtype}, {w13.dtype}, {w2.dtype}, {out.dtype}")
    if logits.dtype not in _IDS:
        raise ValueError(f"logits must be float32, bfloat16 or float16, not {logits.dtype}")
    if not (x.device == logits.device == w13.device == w2.device == out.device):
        raise ValueError("moe_a16w16's tensors are on different devices")
    if t > MAX_TOKENS or e > MAX_EXPERTS or not 1 <= top_k <= min(MAX_TOP_K, e):
        raise ValueError(f"moe_a16w16 serves up to {MAX_TOKENS} tokens, {MAX_EXPERTS} experts and top_k up to {MAX_TOP_K} (and the number "
                         f"of experts); got {t} tokens, {e} experts, top_k {top_k}")
    if i2 % 2 or h % 8 or i % 8 or not h or not i:
        raise ValueError(f"hidden and inner sizes must be multiples of 8, got hidden {h} and w13 with {i2} rows")
    if tuple(logits.shape) != (t, e):
        raise ValueError(f"logits must be {(t, e)}, got {tuple(logits.shape)}")
    _check_matrix("w13", w13, (e, 2 * i, h))
    _check_matrix("w2", w2, (e, h, i))
    assert out.is_contiguous() and tuple(out.shape) == (t, h), f"out must be contiguous {(t, h)}, got {tuple(out.shape)}"
    args = _lib.MoeArgs()
    if t:
        _check_matrix("x", x, (t, h))
    args.x, args.logits, args.w13, args.w2, args.out = (v.data_ptr() for v in (x, logits, w13, w2, out))
    args.tokens, args.hidden, args.inner, args.experts = t, h, i, e
    args.ldx = x.stride(0) if t > 1 else h
    args.logits_row, args.logits_col = logits.stride()
    args.w13_expert, args.w13_row = w13.stride(0), w13.stride(1)
    args.w2_expert = w2.stride(0)
    args.w2_row = w2.stride(1) if h > 1 else i
    args.ldo = h
    args.top_k, args.renormalize = top_k, int(bool(renormalize))
    args.dtype, args.logits_dtype = _IDS[x.dtype], _IDS[logits.dtype]
    args.wait_limit_us = user_kwargs.get("wait_limit_us", 0)
    args.no_pdl = 0 if user_kwargs.get("pdl", True) else 1
    return args


def _capturing(stream: Optional[torch.cuda.Stream]) -> bool:
    if stream is None:
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.stream(stream):
        return torch.cuda.is_current_stream_capturing()


def _describe(t: torch.Tensor):
    return t.data_ptr(), t.shape, t.stride(), t.dtype, t.get_device()


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
    Sums, softmax and SiLU are fp32; p * silu(g) * u is rounded to the 16-bit type as the second product's operand.

    An expert of weight zero (a logit of -inf) is not evaluated, a token whose logits are all -inf gets zeros, a NaN logit
    makes its token's row NaN. Non-finite values in a chosen expert's weights reach every token of the call.
    user_kwargs: wait_limit_us, pdl. Asynchronous on `stream`; `gemm_a16w16.check_status` reports abandoned waits."""
    capturing = x.is_cuda and _capturing(stream)
    key = None
    if out is not None and x.is_cuda and not capturing:
        stream_ptr = (torch.cuda.current_stream(x.device) if stream is None else stream).cuda_stream
        key = (_describe(x), _describe(logits), _describe(w13), _describe(w2), _describe(out), top_k, bool(renormalize),
               tuple(sorted(user_kwargs.items())) if user_kwargs else (), stream_ptr)
        with _prepared_lock:  # held over the launch: a handle is released only after it has left the table
            ent = _prepared.get(key)
            hit = ent is not None and ent[2] == ent[1].generation
            if hit:
                with torch.cuda.device(ent[3]):
                    rc = _lib.load().b200_gemm_moe_launch(ent[0], stream_ptr)
        if hit:
            if rc != 0:
                raise RuntimeError(f"b200_gemm_moe_launch failed ({rc}): {_lib.strerror(rc)}")
            return out

    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    args = _fill_args(x, logits, w13, w2, top_k, out, renormalize, user_kwargs)
    assert x.is_cuda, "moe_a16w16 runs on CUDA tensors only (there is no CPU path)"
    device = x.device
    if stream is None:
        stream = torch.cuda.current_stream(device)
    if x.shape[0] == 0:
        return out
    lib = _lib.load()
    ws = _workspace_for(device, stream)
    args.status = ws.status.data_ptr()
    need = lib.b200_gemm_moe_workspace_bytes(C.byref(args))
    handle = C.c_void_p()
    with torch.cuda.device(device):
        if capturing:
            # A graph keeps scratch of its own (its memory pool's), so that two graphs may run at once.
            with torch.cuda.stream(stream):
                scratch = torch.empty(need, dtype=torch.uint8, device=device)
            args.workspace, args.workspace_bytes = scratch.data_ptr(), need
        else:
            # behind the split-K tickets that the 16-bit GEMM keeps at the start of the stream's workspace
            ws.ensure(_lib.COUNTER_BYTES + need, device, stream)
            args.workspace, args.workspace_bytes = ws.buf.data_ptr() + _lib.COUNTER_BYTES, ws.buf.numel() - _lib.COUNTER_BYTES
        rc = lib.b200_gemm_moe_prepare(C.byref(args), C.byref(handle))
        if rc != 0:
            raise RuntimeError(f"b200_gemm_moe_prepare failed ({rc}): {_lib.strerror(rc)}")
        rc = lib.b200_gemm_moe_launch(handle, stream.cuda_stream)
    if rc != 0 or key is None:
        lib.b200_gemm_moe_release(handle)
        if rc != 0:
            raise RuntimeError(f"b200_gemm_moe_launch failed ({rc}): {_lib.strerror(rc)}")
        return out
    evicted = []
    with _prepared_lock:
        old = _prepared.pop(key, None)
        if old is not None:
            evicted.append(old)
        _prepared[key] = (handle, ws, ws.generation, x.get_device())
        while len(_prepared) > _PREPARED_MAX:
            evicted.append(_prepared.popitem(last=False)[1])
    for ent in evicted:
        lib.b200_gemm_moe_release(ent[0])
    return out
