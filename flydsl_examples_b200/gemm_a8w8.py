"""8-bit floating-point products with one scale for each block of 128: the operators next to `gemm_a16w16`.

    q, s = quantize_a8(x, group="row")                     # values and power-of-two scales
    c = gemm_a8w8(a, a_scale, b, b_scale, layout="nt")     # C[M, N] = A[M, K] @ B[K, N] (+ bias[N])
    y = linear_a8w8(x, weight, bias)                       # a linear layer on the two, with its backward pass

Operands are `torch.float8_e4m3fn` or `torch.float8_e5m2`, each its own. Products are exact, sums are fp32, the result is
rounded once to `out_dtype`. Layout letters, `user_kwargs`, streams, `out` and errors follow `gemm_a16w16`; the kernels are in
libb200_gemm.so (hand-written sm_100a CUDA), there is no CPU path.
"""
from __future__ import annotations

import ctypes as C
import functools
import struct
from typing import Optional

import torch

from . import _lib
from ._launch import device_sms, on_device, raw_stream
from .gemm_a16w16 import _workspace_for

GROUP = 128
_F8_ID = {torch.float8_e4m3fn: _lib.DTYPE_E4M3, torch.float8_e5m2: _lib.DTYPE_E5M2}
_F_ID = {torch.float32: _lib.DTYPE_FP32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16}
_POLICY_KEYS = ("tile_n", "cta_group", "split_k", "group_m", "swap_ab", "max_ctas", "pdl", "wait_limit_us")


def _blocks(n: int) -> int:
    return -(-n // GROUP)


# ------------------------------------------------------------------------------------------------------------ policy
@functools.lru_cache(maxsize=4096)
def _heuristic_items(m, n, k, a_t, b_t, num_sms) -> tuple:
    pol = heuristic_a8w8(m, n, k, a_t, b_t, num_sms)
    return pol["tile_n"], pol["cta_group"], pol["split_k"], pol.get("group_m", 0), int(pol["swap_ab"])


def heuristic_a8w8(m: int, n: int, k: int, a_transposed: bool, b_transposed: bool, num_sms: int = 148) -> dict:
    """Tile, split and operand order for a call without a tiling of its own.

    Up to 64 rows of A the product streams the weights: B takes the 128-row side (swap_ab), the tokens fill a tile of 16 to
    64 columns, and a cluster splits K until the CTAs fill the SMs. Above that the time of a call is taken as whole waves
    times the measured cycles of a K block, and the cheapest of the tiles is used."""
    kb = _blocks(k)
    if m <= 64 and not a_transposed:
        tile = 16 if m <= 16 else 32 if m <= 32 else 64
        tiles = _blocks(n)
        split = 1
        while split < 16 and tiles * split * 2 <= num_sms and kb >= split * 4:
            split *= 2
        return {"tile_n": tile, "cta_group": 1, "swap_ab": True, "split_k": split}
    best = None
    # cycles of a K block and of a cluster's reduction, measured at 256 ... 8192 rows
    for tile, cg, cycles, reduction in ((256, 2, 830, 0), (128, 2, 640, 0), (128, 1, 560, 8500), (64, 1, 400, 3000)):
        if not b_transposed and tile // cg != 128:
            continue  # a row-contiguous B arrives in boxes of 128 columns per CTA
        tiles = -(-m // (128 * cg)) * -(-n // tile)
        slots = num_sms // cg
        for split in (1, 2, 4, 8) if cg == 1 else (1,):
            if split > 1 and (tiles * split > slots or kb < 4 * split):
                continue
            waves = -(-tiles * split // slots)
            cost = waves * (-(-kb // split) * cycles + 1500) + (reduction if split > 1 else 0)
            if best is None or cost < best[0]:
                best = (cost, {"tile_n": tile, "cta_group": cg, "swap_ab": False, "split_k": split})
    pol = best[1]
    pol["group_m"] = 8 if m > 1024 else 0  # eight tile rows share the columns of B that L2 holds
    return pol


def _policy(m, n, k, a_t, b_t, user_kwargs, num_sms) -> tuple:
    """The fields of b200_gemm_policy, in its order."""
    if not user_kwargs:
        tile_n, cta_group, split_k, group_m, swap_ab = _heuristic_items(m, n, k, a_t, b_t, num_sms)
        return tile_n, 0, split_k, group_m, swap_ab, cta_group, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0
    for key in user_kwargs:
        if key not in _POLICY_KEYS:
            raise ValueError(f"unknown gemm_a8w8 policy key {key!r}; expected some of {_POLICY_KEYS}")
    if "tile_n" in user_kwargs:
        pol = {"cta_group": 1, "swap_ab": False, "split_k": 1}
    else:
        pol = heuristic_a8w8(m, n, k, a_t, b_t, num_sms)
        for key in ("cta_group", "split_k", "swap_ab"):
            if key in user_kwargs:
                raise ValueError(f"gemm_a8w8 policy key {key!r} needs 'tile_n' beside it")
    pol.update(user_kwargs)
    return (pol["tile_n"], 0, pol["split_k"], pol.get("group_m", 0), int(pol["swap_ab"]), pol["cta_group"], 0, pol.get("max_ctas", 0), 0,
            0 if pol.get("pdl", True) else 1, 0, pol.get("wait_limit_us", 0), 0, 0, 0, 0)


# -------------------------------------------------------------------------------------------------------------- GEMM
_LAYOUTS = {"nn": (False, False), "nt": (False, True), "tn": (True, False), "tt": (True, True)}
_ARGS = struct.Struct("@6P10q8i16iP")  # b200_gemm_a8w8_args


def _check_operand(name: str, t: torch.Tensor, transposed: bool) -> int:
    """Leading stride of an operand; raises unless the contiguous dimension has stride 1 and rows start on 16 bytes."""
    rows, cols = t.shape
    lead, inner = t.stride()
    n_lead, n_inner = rows, cols
    if transposed:
        lead, inner, n_lead, n_inner = inner, lead, n_inner, n_lead
    if n_inner == 1:
        inner = 1  # a stride of a size-1 dimension is arbitrary in torch
    if n_lead == 1:
        lead = max(-(-n_inner // 16) * 16, 16)
    if inner != 1 or lead % 16 != 0 or lead < n_inner or t.data_ptr() % 16 != 0:
        raise ValueError(
            f"{name} does not satisfy the layout requirements for a {'column' if transposed else 'row'}-major input: expected "
            f"stride({0 if transposed else 1}) == 1 and a 16-byte-aligned data pointer and leading stride; "
            f"got shape={tuple(t.shape)} and stride={t.stride()}"
        )
    return lead


def _check_scale(name: str, s: torch.Tensor, rows: int, kb: int, have_rows: int, have_kb: int) -> int:
    """1 when the scale is one per 128 rows, 0 when one per row."""
    if s.dtype is not torch.float32 or have_kb != kb or have_rows != rows and have_rows != _blocks(rows):
        raise ValueError(
            f"{name} must be a float32 tensor with one scale per block of {GROUP} along K and per row (column) or block of {GROUP}: "
            f"expected {rows} or {_blocks(rows)} and {kb}, got shape {tuple(s.shape)}, {s.dtype}"
        )
    return 0 if have_rows == rows else 1


def _arguments(a, a_scale, b, b_scale, out_ptr, out_dtype, bias, layout, user_kwargs, num_sms, status) -> bytes:
    """Checks the operands and packs a b200_gemm_a8w8_args."""
    a_t, b_t = _LAYOUTS[layout]
    m, k = a.shape
    n = b.shape[1]
    kb = _blocks(k)
    if a.dtype not in _F8_ID or b.dtype not in _F8_ID:
        raise ValueError(f"gemm_a8w8 takes float8_e4m3fn or float8_e5m2 operands, got {a.dtype} and {b.dtype}")
    lda, ldb = _check_operand("A", a, a_t), _check_operand("B", b, b_t)
    sa_rows, sa_kbs = a_scale.shape
    sb_kbs, sb_cols = b_scale.shape
    a_block = _check_scale("a_scale", a_scale, m, kb, sa_rows, sa_kbs)
    b_block = _check_scale("b_scale", b_scale, n, kb, sb_cols, sb_kbs)
    sa_row, sa_kb = a_scale.stride()
    sb_kb, sb_col = b_scale.stride()
    return _ARGS.pack(
        a.data_ptr(), b.data_ptr(), a_scale.data_ptr(), b_scale.data_ptr(), out_ptr, 0 if bias is None else bias.data_ptr(),
        m, n, k, lda, ldb, n, sa_row, sa_kb, sb_col, sb_kb,
        a_t, b_t, _F8_ID[a.dtype], _F8_ID[b.dtype], a_block, b_block, _F_ID[out_dtype], 0 if bias is None else _F_ID[bias.dtype],
        *_policy(m, n, k, a_t, b_t, user_kwargs, num_sms), status)


def _layout(layout: str) -> str:
    low = layout.lower()
    if low not in _LAYOUTS:
        raise ValueError(f"unsupported GEMM layout: {layout!r}; expected 'nn', 'nt', 'tn', or 'tt'")
    return low


def gemm_a8w8(
    a: torch.Tensor,
    a_scale: torch.Tensor,
    b: torch.Tensor,
    b_scale: torch.Tensor,
    out: Optional[torch.Tensor] = None,
    bias: Optional[torch.Tensor] = None,
    user_kwargs: dict = {},
    stream: Optional[torch.cuda.Stream] = None,
    layout: str = "nt",
    out_dtype: Optional[torch.dtype] = None,
) -> torch.Tensor:
    """C[M, N] = A[M, K] @ B[K, N] (+ bias[N]) from 8-bit operands with scales, fp32 sums and one final rounding.

    a [M, K], b [K, N]: logical shapes; `layout` says which dimension of each is contiguous ('n' row-major, 't' column-major), as
    in `gemm_a16w16`. Bases and leading strides are multiples of 16 bytes (`quantize_a8` pads its outputs).
    a_scale: float32 [M, ceil(K / 128)] or [ceil(M / 128), ceil(K / 128)]; b_scale: float32 [ceil(K / 128), N] or
    [ceil(K / 128), ceil(N / 128)]; any strides. `out` may be any contiguous tensor of M * N elements; `out_dtype` (default:
    out's, else bfloat16) and the bias are float32, bfloat16 or float16. Asynchronous on `stream`.

    user_kwargs: tile_n (16, 32, 64, 128; with cta_group 2: 128, 256), cta_group, split_k (K blocks of a tile over the CTAs of a
    cluster), swap_ab, group_m, max_ctas, pdl, wait_limit_us; without tile_n the tiling is chosen by `heuristic_a8w8`."""
    layout = _layout(layout)
    assert a.ndim == 2 and b.ndim == 2 and a_scale.ndim == 2 and b_scale.ndim == 2, "operands and scales are matrices"
    m, k = a.shape
    n = b.shape[1]
    assert b.shape[0] == k, f"A is {tuple(a.shape)}, B is {tuple(b.shape)}"
    device = a.device
    if b.device != device or a_scale.device != device or b_scale.device != device:
        raise ValueError(f"operands and scales are on different devices: {device}, {b.device}, {a_scale.device}, {b_scale.device}")
    if out_dtype is None:
        out_dtype = torch.bfloat16 if out is None else out.dtype
    if out_dtype not in _F_ID:
        raise ValueError(f"unsupported output dtype {out_dtype}; expected float32, bfloat16 or float16")
    if bias is not None:
        if bias.dtype not in _F_ID:
            raise ValueError(f"unsupported bias dtype {bias.dtype}; expected float32, bfloat16 or float16")
        assert bias.ndim == 1 and bias.shape[0] == n and bias.device == device
    if out is not None:
        assert out.dtype == out_dtype
        assert out.device == device
        assert out.is_contiguous()
        assert out.numel() == m * n, f"out has {out.numel()} elements, the product {m * n}"
    if not a.is_cuda:
        _arguments(a, a_scale, b, b_scale, 0, out_dtype, bias, layout, user_kwargs, 148, 0)
        raise AssertionError("gemm_a8w8 runs on CUDA tensors only (there is no CPU path)")
    index = device.index
    with on_device(index, stream):
        if out is None:
            out = torch.empty(m, n, dtype=out_dtype, device=device)
        elif out.shape != (m, n):
            out = out.view(m, n)
        if bias is not None and not bias.is_contiguous():
            bias = bias.contiguous()
        if m == 0 or n == 0:
            return out
        if k == 0:
            return out.zero_() if bias is None else out.copy_(bias.expand(m, n))
        stream_ptr = raw_stream(index)
        args = _arguments(a, a_scale, b, b_scale, out.data_ptr(), out_dtype, bias, layout, user_kwargs, device_sms(index),
                          _workspace_for(device, stream_ptr).status_ptr)
        rc = _lib.fast("b200_gemm_a8w8")(args, stream_ptr)
    if rc != 0:
        raise RuntimeError(f"b200_gemm_a8w8 failed ({rc}): {_lib.strerror(rc)}")
    return out


def plan(a, a_scale, b, b_scale, layout="nt", user_kwargs: dict = {}, out_dtype=torch.bfloat16) -> dict:
    """What a call with these arguments would launch (tile, cluster split, grid, shared memory)."""
    raw = _arguments(a, a_scale, b, b_scale, 0, out_dtype, None, _layout(layout), user_kwargs, 148, 0)
    pl = _lib.Plan()
    rc = _lib.load().b200_gemm_a8w8_plan_query(C.byref(_lib.Args8.from_buffer_copy(raw)), C.byref(pl))
    if rc != 0:
        raise RuntimeError(f"b200_gemm_a8w8_plan_query failed ({rc}): {_lib.strerror(rc)}")
    return pl.as_dict()


# --------------------------------------------------------------------------------------------------------- quantizer
def _pitched(rows: int, cols: int, dtype: torch.dtype, device) -> torch.Tensor:
    """[rows, cols] with rows that start on 16-byte boundaries."""
    if cols % 16 == 0:
        return torch.empty(rows, cols, dtype=dtype, device=device)
    return torch.empty(rows, -(-cols // 16) * 16, dtype=dtype, device=device)[:, :cols]


def _is_row_major(x: torch.Tensor) -> bool:
    rows, cols = x.shape
    return (cols <= 1 or x.stride(1) == 1) and (rows <= 1 or x.stride(0) >= cols)


def _row_major(x: torch.Tensor) -> torch.Tensor:
    return x if _is_row_major(x) else x.contiguous()


_QUANT_ARGS = struct.Struct("@P3q4i" + "PqP2q" * 2 + "Pq")  # b200_gemm_quantize_args
_GROUPS = {"row": 1, "col": 2, "both": 3, "block": 4}


def _quantize(x, group, dtype, stream):
    if group not in _GROUPS:
        raise ValueError(f"unknown group {group!r}; expected one of {tuple(_GROUPS)}")
    if dtype not in _F8_ID:
        raise ValueError(f"quantize_a8 makes float8_e4m3fn or float8_e5m2, not {dtype}")
    if x.dtype not in _F_ID:
        raise ValueError(f"quantize_a8 takes float32, bfloat16 or float16, not {x.dtype}")
    assert x.ndim == 2, f"quantize_a8 takes a matrix, got {x.ndim} dimensions"
    rows, cols = x.shape
    if not _is_row_major(x):
        raise ValueError(f"x must be row-major: expected stride(1) == 1; got shape={tuple(x.shape)} and stride={x.stride()}")
    assert x.is_cuda, "quantize_a8 runs on CUDA tensors only (there is no CPU path)"
    device = x.device
    index = device.index
    mode = _GROUPS[group]
    got = []
    row = col = (0, 0, 0, 0, 0)
    with on_device(index, stream):
        if mode != 2:
            q = _pitched(rows, cols, dtype, device)
            # the product reads the scales of 128 rows at a time: rows are the contiguous dimension
            n_rows = _blocks(rows) if mode == 4 else rows
            s = torch.empty_strided((n_rows, _blocks(cols)), (1, n_rows), dtype=torch.float32, device=device)
            row = (q.data_ptr(), -(-cols // 16) * 16, s.data_ptr(), 1, n_rows)
            got += [q, s]
        if mode == 2 or mode == 3:
            q = _pitched(rows, cols, dtype, device)
            s = torch.empty(_blocks(rows), cols, dtype=torch.float32, device=device)
            col = (q.data_ptr(), -(-cols // 16) * 16, s.data_ptr(), cols, 1)
            got += [q, s]
        args = _QUANT_ARGS.pack(x.data_ptr(), rows, cols, x.stride(0) if rows > 1 else cols, _F_ID[x.dtype], _F8_ID[dtype], mode, 0,
                                *row, *col, 0, 0)
        rc = _lib.fast("b200_gemm_quantize_a8")(args, raw_stream(index))
    if rc != 0:
        raise RuntimeError(f"b200_gemm_quantize_a8 failed ({rc}): {_lib.strerror(rc)}")
    return tuple(got)


def quantize_a8(x: torch.Tensor, group: str = "row", dtype: torch.dtype = torch.float8_e4m3fn,
                stream: Optional[torch.cuda.Stream] = None) -> tuple:
    """8-bit values and scales of a row-major matrix x [R, C] (float32, bfloat16 or float16), in groups of 128.

    group: "row" -> (q [R, C], s [R, ceil(C / 128)]), the operand of a product over C; "col" -> (q [R, C], s [ceil(R / 128), C]),
    of one over R (used as `q.t()`, `s.t()`, or as B with `q`, `s`); "both" -> all four from one read of x; "block" ->
    (q, s [ceil(R / 128), ceil(C / 128)]), a weight's, which serves products over either dimension.

    A group's scale is the smallest power of two (at least 2^-126) that brings its largest finite magnitude to the format's
    largest value or below; 1 for a group of zeros. q is x / s rounded to nearest even, the only rounding. NaN stays NaN; an
    infinity becomes NaN in e4m3 and stays infinite in e5m2; neither changes its group's scale. Asynchronous on `stream`."""
    return _quantize(x, group, dtype, stream)


# ------------------------------------------------------------------------------------------------------ linear layer
# A step of the layer is eight launches, and a launch through the public calls costs the host more than the GPU needs for it at
# ordinary sizes. The layer checks its tensors once, keeps each pass's operands in one buffer and packs the argument blocks
# itself.
def _up(n: int, to: int) -> int:
    return -(-n // to) * to


class _Buffer:
    """Offsets of the pieces of one allocation, each on a 256-byte boundary."""

    __slots__ = ("at", "size")

    def __init__(self, *sizes: int):
        self.at, self.size = [], 0
        for n in sizes:
            self.at.append(self.size)
            self.size += _up(n, 256)


@functools.lru_cache(maxsize=1024)
def _quantized(rows: int, cols: int, row: bool, col: bool, block: bool) -> _Buffer:
    """Values (pitch a multiple of 16) and scales of each kind that is asked for, in this order."""
    values, sizes = rows * _up(cols, 16), []
    if row:
        sizes += [values, 4 * rows * _blocks(cols)]
    if col:
        sizes += [values, 4 * _blocks(rows) * cols]
    if block:
        sizes += [values, 4 * _blocks(rows) * _blocks(cols)]
    return _Buffer(*sizes)


def _check(rc: int, name: str) -> None:
    if rc != 0:
        raise RuntimeError(f"{name} failed ({rc}): {_lib.strerror(rc)}")


def _quantize_at(x, f8_id, row_at, col_at, block_at, sums, stream) -> None:
    """Quantizes a row-major matrix to device addresses (0: not wanted), laid out as `_quantized` has them."""
    rows, cols = x.shape
    if rows == 0 or cols == 0:
        return
    pitch = _up(cols, 16)
    mode = 4 if block_at else (1 if row_at else 0) + (2 if col_at else 0)
    q = rows * pitch
    row = (block_at or row_at, pitch, (block_at or row_at) + _up(q, 256), 1, _blocks(rows) if block_at else rows) if mode != 2 else (0,) * 5
    col = (col_at, pitch, col_at + _up(q, 256), cols, 1) if mode in (2, 3) else (0,) * 5
    args = _QUANT_ARGS.pack(x.data_ptr(), rows, cols, x.stride(0) if rows > 1 else cols, _F_ID[x.dtype], f8_id, mode, 0, *row, *col, *sums)
    _check(_lib.fast("b200_gemm_quantize_a8")(args, stream), "b200_gemm_quantize_a8")


def _gemm_at(pointers, m, n, k, lda, ldb, scale_strides, a_t, b_t, a_id, b_id, b_block, out_id, bias_id, index, status, stream) -> None:
    """b200_gemm_a8w8 on device addresses; pointers: a, b, a_scale, b_scale, out, bias."""
    if m == 0 or n == 0:
        return
    args = _ARGS.pack(*pointers, m, n, k, lda, ldb, n, *scale_strides, a_t, b_t, a_id, b_id, 0, b_block, out_id, bias_id,
                      *_policy(m, n, k, a_t, b_t, {}, device_sms(index)), status)
    _check(_lib.fast("b200_gemm_a8w8")(args, stream), "b200_gemm_a8w8")


class _Linear8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, grad_dtype):
        k, n = x.shape[-1], weight.shape[0]
        x2, w2 = _row_major(x.reshape(-1, k)), _row_major(weight)
        m = x2.shape[0]
        need_x, need_w = ctx.needs_input_grad[:2]
        index, device, e4 = x.get_device(), x.device, _lib.DTYPE_E4M3
        kp, mb, nb, kb = _up(k, 16), _blocks(m), _blocks(n), _blocks(k)
        with on_device(index, None):
            stream = raw_stream(index)
            y = torch.empty(m, n, dtype=x.dtype, device=device)
            rows, cols, blocks = _quantized(m, k, True, False, False), _quantized(m, k, False, True, False), _quantized(n, k, False, False, True)
            # what the backward pass reads: x by columns and the weight, as far as they are needed
            keep = _Buffer(cols.size if need_w else 0, blocks.size if need_x else 0)
            temp = torch.empty(rows.size + (0 if need_x else blocks.size), dtype=torch.uint8, device=device)
            saved = torch.empty(keep.size, dtype=torch.uint8, device=device)
            xr = temp.data_ptr()
            xc = saved.data_ptr() if need_w else 0
            wq = saved.data_ptr() + keep.at[1] if need_x else xr + rows.size
            if k == 0:
                y.copy_(0 if bias is None else bias.expand(m, n))
            else:
                _quantize_at(x2, e4, xr, xc, 0, (0, 0), stream)
                _quantize_at(w2, e4, 0, 0, wq, (0, 0), stream)
                _gemm_at((xr, wq, xr + rows.at[1], wq + blocks.at[1], y.data_ptr(), 0 if bias is None else bias.data_ptr()), m, n, k, kp, kp,
                         (1, m, 1, nb), False, True, e4, e4, 1, _F_ID[x.dtype], 0 if bias is None else _F_ID[bias.dtype], index,
                         _workspace_for(device, stream).status_ptr, stream)
        ctx.save_for_backward(saved)
        ctx.meta = (x.shape, x.dtype, weight.dtype, None if bias is None else bias.dtype, _F8_ID[grad_dtype], m, n, k, keep, cols, blocks)
        return y.view(*x.shape[:-1], n)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        (saved,) = ctx.saved_tensors
        shape, x_dtype, w_dtype, b_dtype, g_id, m, n, k, keep, cols, blocks = ctx.meta
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        g = _row_major(dy.reshape(m, n))  # an expanded gradient (of a sum) is spread out here
        index, device, e4 = dy.get_device(), dy.device, _lib.DTYPE_E4M3
        np_, kp, mb, nb = _up(n, 16), _up(k, 16), _blocks(m), _blocks(n)
        by_col = need_w or need_b
        dx = dw = db = None
        with on_device(index, None):
            stream = raw_stream(index)
            status = _workspace_for(device, stream).status_ptr
            grows, gcols = _quantized(m, n, True, False, False), _quantized(m, n, False, True, False)
            pitch = _up(n, 4)
            parts = _Buffer(grows.size if need_x else 0, gcols.size if by_col else 0, 4 * mb * pitch if need_b else 0)
            temp = torch.empty(parts.size, dtype=torch.uint8, device=device)
            gr, gc, sums = (temp.data_ptr() + at for at in parts.at)
            if by_col or need_x:
                _quantize_at(g, g_id, gr if need_x else 0, gc if by_col else 0, 0, (sums, pitch) if need_b else (0, 0), stream)
            if need_x:
                dx = torch.empty(m, k, dtype=x_dtype, device=device)
                if n == 0:
                    dx.zero_()
                elif k:
                    wq = saved.data_ptr() + keep.at[1]
                    _gemm_at((gr, wq, gr + grows.at[1], wq + blocks.at[1], dx.data_ptr(), 0), m, k, n, np_, kp, (1, m, nb, 1), False, False,
                             g_id, e4, 1, _F_ID[x_dtype], 0, index, status, stream)
                dx = dx.view(shape)
            if need_w:
                dw = torch.empty(n, k, dtype=w_dtype, device=device)
                if m == 0:
                    dw.zero_()
                elif k:
                    xc = saved.data_ptr()
                    _gemm_at((gc, xc, gc + gcols.at[1], xc + cols.at[1], dw.data_ptr(), 0), n, k, m, np_, kp, (1, n, 1, k), True, False,
                             g_id, e4, 0, _F_ID[w_dtype], 0, index, status, stream)
            if need_b:
                db = torch.empty(pitch, dtype=b_dtype, device=device)
                if m == 0:
                    db.zero_()
                elif n:  # the columns' sums over each 128 rows, added in order
                    _check(_lib.load().b200_gemm_reduce_slots(sums, pitch, mb, db.data_ptr(), None, 1, pitch, _F_ID[b_dtype], 0, stream),
                           "b200_gemm_reduce_slots")
                db = db[:n]
        return dx, dw, db, None


def linear_a8w8(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                grad_dtype: torch.dtype = torch.float8_e4m3fn) -> torch.Tensor:
    """y = x @ weight.T (+ bias) in 8-bit floating point, with its backward pass; x [..., K], weight [N, K], bias [N] of float32,
    bfloat16 or float16, y in x's type.

    Forward: x in groups of 128 along K, the weight in 128 x 128 blocks, both e4m3. Backward: the output's gradient is quantized
    to `grad_dtype` once along N (for dx, against the weight as it was quantized) and once along the rows (for dweight, against x
    quantized along the rows in the forward pass); dbias is the sum of the unquantized gradient in fp32, in a fixed order.
    Gradients have their tensor's type."""
    assert weight.ndim == 2 and x.ndim >= 1 and x.shape[-1] == weight.shape[1], f"x is {tuple(x.shape)}, weight {tuple(weight.shape)}"
    for name, t in (("x", x), ("weight", weight), ("bias", bias)):
        if t is not None and t.dtype not in _F_ID:
            raise ValueError(f"linear_a8w8 takes float32, bfloat16 or float16; {name} is {t.dtype}")
    if grad_dtype not in _F8_ID:
        raise ValueError(f"grad_dtype must be float8_e4m3fn or float8_e5m2, not {grad_dtype}")
    assert x.is_cuda, "linear_a8w8 runs on CUDA tensors only (there is no CPU path)"
    assert x.device == weight.device
    if bias is not None:
        assert bias.shape == (weight.shape[0],) and bias.device == x.device
        bias = bias.contiguous()
    return _Linear8.apply(x, weight, bias, grad_dtype)
