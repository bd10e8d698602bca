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
import math
import struct
from typing import Optional

import torch

from . import _lib
from ._launch import device_sms, is_current, on_device, raw_stream
from .gemm_a16w16 import _workspace_for

GROUP = 128
_F8_ID = {torch.float8_e4m3fn: _lib.DTYPE_E4M3, torch.float8_e5m2: _lib.DTYPE_E5M2}
_F_ID = {torch.float32: _lib.DTYPE_FP32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16}
_POLICY_KEYS = ("tile_n", "cta_group", "split_k", "group_m", "swap_ab", "max_ctas", "pdl", "wait_limit_us")


def _blocks(n: int) -> int:
    return -(-n // GROUP)


# ------------------------------------------------------------------------------------------------------------ policy
# Clusters of one CTA per SM that a B200 with its 148 SMs holds at a time, as its occupancy query answers: a cluster lies
# within one of its groups of SMs, so large ones leave some SMs over.
_HELD = {1: 148, 2: 74, 4: 33, 8: 15, 16: 7}


def _clusters(size: int, num_sms: int) -> int:
    return max(1, _HELD[size] * num_sms // 148)


@functools.lru_cache(maxsize=4096)
def _heuristic_items(m, n, k, a_t, b_t, num_sms) -> tuple:
    pol = heuristic_a8w8(m, n, k, a_t, b_t, num_sms)
    return pol["tile_n"], pol["cta_group"], pol["split_k"], pol.get("group_m", 0), int(pol["swap_ab"])


# Microseconds of a call by (tile_n, cta_group, swap_ab): of a wave of tiles, of a K block in it, of a cluster's reduction times
# its size (each CTA joins 1 / split of the tile), and of the SMs that all start together, times the part of them in use. Least
# squares over 5,800 times of 870 random problems (1 to 12288 rows and columns, 100 to 12288 deep, all layouts and scales).
_COST = {
    (16, 1, False): (2.3, 0.27, 3.4, 1.7),
    (16, 1, True): (2.1, 0.26, 3.9, 0.9),
    (32, 1, False): (2.9, 0.30, 3.3, 2.1),
    (32, 1, True): (2.8, 0.29, 5.1, 0.6),
    (64, 1, False): (3.2, 0.32, 6.6, 2.9),
    (64, 1, True): (4.3, 0.33, 6.2, 0.9),
    (128, 1, False): (3.7, 0.38, 13.8, 3.5),
    (128, 2, False): (4.2, 0.36, 0.0, 3.0),
    (256, 2, False): (5.5, 0.49, 0.0, 3.8),
}


def heuristic_a8w8(m: int, n: int, k: int, a_transposed: bool, b_transposed: bool, num_sms: int = 148) -> dict:
    """Tile, split and operand order for a call without a tiling of its own: the cheapest by a model of the call's time.

    A call takes whole waves of tiles; a cluster splits the K of a tile, down to a block of 128 per CTA, only as far as all
    clusters run at once (8 x 1024 x 2048: split 4 4.5 us, 8 4.0; 16, whose eighth cluster waits for one of the others, 7.5).
    Up to 64 rows of A the weights take the 128-row side (swap_ab) and the tokens fill a tile of 16 to 64 columns; small
    problems of any shape want small tiles as well (396 x 161 x 206: 128 wide 6.2 us, 16 wide 3.6), large ones CTA pairs."""
    kb = _blocks(k)
    best = pol = None
    for (tile, cg, swap), (wave, block, reduction, start) in _COST.items():
        if swap and m > 1024:
            continue  # a tile's columns are rows of the output here: stores of more rows than that cost more than they save
        if tile // cg != 128 and (a_transposed if swap else not b_transposed):
            continue  # an operand whose rows are contiguous along its own dimension arrives in boxes of 128 per CTA
        rows, cols = (n, m) if swap else (m, n)
        tiles = -(-rows // (128 * cg)) * -(-cols // tile)
        for split in (1, 2, 4, 8, 16) if cg == 1 else (1,):
            held = _clusters(split * cg, num_sms)
            if split > 1 and (tiles > held or split > kb):
                break
            cost = (-(-tiles // held) * (wave + -(-kb // split) * block) + (reduction / split if split > 1 else 0.0)
                    + start * min(1.0, tiles * split * cg / num_sms))
            if best is None or cost < best:
                best, pol = cost, {"tile_n": tile, "cta_group": cg, "swap_ab": swap, "split_k": split}
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
# b200_gemm_a8w8_args in parts; the last member is the status address
_POINTERS, _SIZES = struct.Struct("@6P"), struct.Struct("@10q8i16i")


def _leading(name: str, shape, stride, transposed: bool) -> int:
    """Leading stride of an operand; raises unless the contiguous dimension has stride 1 and rows start on 16 bytes."""
    n_lead, n_inner = shape
    lead, inner = stride
    if transposed:
        lead, inner, n_lead, n_inner = inner, lead, n_inner, n_lead
    if n_inner == 1:
        inner = 1  # a stride of a size-1 dimension is arbitrary in torch
    if n_lead == 1:
        lead = max(-(-n_inner // 16) * 16, 16)
    if inner != 1 or lead % 16 != 0 or lead < n_inner:
        raise ValueError(
            f"{name} does not satisfy the layout requirements for a {'column' if transposed else 'row'}-major input: expected "
            f"stride({0 if transposed else 1}) == 1 and a 16-byte-aligned data pointer and leading stride; "
            f"got shape={tuple(shape)} and stride={stride}"
        )
    return lead


def _check_scale(name: str, dtype, have_rows: int, have_kb: int, rows: int, kb: int) -> int:
    """1 when the scale is one per 128 rows, 0 when one per row."""
    if dtype is not torch.float32 or have_kb != kb or have_rows != rows and have_rows != _blocks(rows):
        raise ValueError(
            f"{name} must be a float32 tensor with one scale per block of {GROUP} along K and per row (column) or block of {GROUP}: "
            f"expected {rows} or {_blocks(rows)} and {kb}, got {have_rows} and {have_kb}, {dtype}"
        )
    return 0 if have_rows == rows else 1


@functools.lru_cache(maxsize=4096)
def _call_plan(a_shape, a_stride, a_dtype, b_shape, b_stride, b_dtype, sa_shape, sa_stride, sa_dtype, sb_shape, sb_stride, sb_dtype,
               out_dtype, bias_dtype, layout, kwargs, num_sms) -> tuple:
    """(m, n, k, sizes of the argument block) of a call with operands of these shapes, strides and types; raises what the call
    raises. Everything here follows from the sizes, so a repeated call pays for it once."""
    if layout not in _LAYOUTS:
        raise ValueError(f"unsupported GEMM layout: {layout!r}; expected 'nn', 'nt', 'tn', or 'tt'")
    a_t, b_t = _LAYOUTS[layout]
    assert len(a_shape) == len(b_shape) == len(sa_shape) == len(sb_shape) == 2, "operands and scales are matrices"
    (m, k), n = a_shape, b_shape[1]
    assert b_shape[0] == k, f"A is {tuple(a_shape)}, B is {tuple(b_shape)}"
    if a_dtype not in _F8_ID or b_dtype not in _F8_ID:
        raise ValueError(f"gemm_a8w8 takes float8_e4m3fn or float8_e5m2 operands, got {a_dtype} and {b_dtype}")
    if out_dtype not in _F_ID:
        raise ValueError(f"unsupported output dtype {out_dtype}; expected float32, bfloat16 or float16")
    if bias_dtype is not None and bias_dtype not in _F_ID:
        raise ValueError(f"unsupported bias dtype {bias_dtype}; expected float32, bfloat16 or float16")
    kb = _blocks(k)
    a_block = _check_scale("a_scale", sa_dtype, sa_shape[0], sa_shape[1], m, kb)
    b_block = _check_scale("b_scale", sb_dtype, sb_shape[1], sb_shape[0], n, kb)
    policy = _policy(m, n, k, a_t, b_t, dict(kwargs), num_sms)
    if not (m and n and k):
        return m, n, k, None
    sizes = _SIZES.pack(
        m, n, k, _leading("A", a_shape, a_stride, a_t), _leading("B", b_shape, b_stride, b_t), n, *sa_stride, sb_stride[1], sb_stride[0],
        a_t, b_t, _F8_ID[a_dtype], _F8_ID[b_dtype], a_block, b_block, _F_ID[out_dtype], 0 if bias_dtype is None else _F_ID[bias_dtype],
        *policy)
    return m, n, k, sizes


def _plan_of(a, a_scale, b, b_scale, out_dtype, bias_dtype, layout, user_kwargs, num_sms) -> tuple:
    return _call_plan(a.shape, a.stride(), a.dtype, b.shape, b.stride(), b.dtype, a_scale.shape, a_scale.stride(), a_scale.dtype,
                      b_scale.shape, b_scale.stride(), b_scale.dtype, out_dtype, bias_dtype, layout.lower(),
                      tuple(user_kwargs.items()) if user_kwargs else (), num_sms)


def _launch_gemm(a, a_scale, b, b_scale, out, bias, out_dtype, m, n, k, sizes, index) -> torch.Tensor:
    """On the current device and stream."""
    if out is None:
        out = torch.empty(m, n, dtype=out_dtype, device=a.device)
    elif out.shape != (m, n):
        out = out.view(m, n)
    if sizes is None:
        return out if m == 0 or n == 0 else out.zero_() if bias is None else out.copy_(bias.expand(m, n))
    bias_ptr = 0
    if bias is not None:
        if not bias.is_contiguous():
            bias = bias.contiguous()
        bias_ptr = bias.data_ptr()
    stream_ptr = raw_stream(index)
    args = (_POINTERS.pack(a.data_ptr(), b.data_ptr(), a_scale.data_ptr(), b_scale.data_ptr(), out.data_ptr(), bias_ptr) + sizes
            + _workspace_for(a.device, stream_ptr).status_bytes)
    rc = _lib.fast("b200_gemm_a8w8")(args, stream_ptr)
    if rc != 0:
        raise RuntimeError(f"b200_gemm_a8w8 failed ({rc}): {_lib.strerror(rc)}")
    return out


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
    [ceil(K / 128), ceil(N / 128)]; any strides. The product of the two scales of a block is rounded to float32 before it meets the
    block's sum: it should lie between 2^-126 and 2^128 (or be 0). `out` may be any contiguous tensor of M * N elements;
    `out_dtype` (default: out's, else bfloat16) and the bias are float32, bfloat16 or float16. Asynchronous on `stream`.

    user_kwargs: tile_n (16, 32, 64, 128; with cta_group 2: 128, 256), cta_group, split_k (K blocks of a tile over the CTAs of a
    cluster), swap_ab, group_m, max_ctas, pdl, wait_limit_us; without tile_n the tiling is chosen by `heuristic_a8w8`."""
    index = a.get_device()
    if out_dtype is None:
        out_dtype = torch.bfloat16 if out is None else out.dtype
    m, n, k, sizes = _plan_of(a, a_scale, b, b_scale, out_dtype, None if bias is None else bias.dtype, layout, user_kwargs,
                              device_sms(index) if index >= 0 else 148)
    if b.get_device() != index or a_scale.get_device() != index or b_scale.get_device() != index:
        raise ValueError(f"operands and scales are on different devices: {a.device}, {b.device}, {a_scale.device}, {b_scale.device}")
    if bias is not None:
        assert bias.ndim == 1 and bias.shape[0] == n and bias.get_device() == index
    if out is not None:
        assert out.dtype == out_dtype
        assert out.get_device() == index
        assert out.is_contiguous()
        assert out.numel() == m * n, f"out has {out.numel()} elements, the product {m * n}"
    if sizes is not None and (a.data_ptr() | b.data_ptr()) & 15:
        raise ValueError("A and B must start on a 16-byte-aligned address")
    assert index >= 0, "gemm_a8w8 runs on CUDA tensors only (there is no CPU path)"
    if stream is None and is_current(index):
        return _launch_gemm(a, a_scale, b, b_scale, out, bias, out_dtype, m, n, k, sizes, index)
    with on_device(index, stream):
        return _launch_gemm(a, a_scale, b, b_scale, out, bias, out_dtype, m, n, k, sizes, index)


def plan(a, a_scale, b, b_scale, layout="nt", user_kwargs: dict = {}, out_dtype=torch.bfloat16) -> dict:
    """What a call with these arguments would launch (tile, cluster split, grid, shared memory)."""
    sizes = _plan_of(a, a_scale, b, b_scale, out_dtype, None, layout, user_kwargs, 148)[3]
    raw = _POINTERS.pack(a.data_ptr(), b.data_ptr(), a_scale.data_ptr(), b_scale.data_ptr(), 0, 0) + (sizes or bytes(_SIZES.size)) + bytes(8)
    pl = _lib.Plan()
    rc = _lib.load().b200_gemm_a8w8_plan_query(C.byref(_lib.Args8.from_buffer_copy(raw)), C.byref(pl))
    if rc != 0:
        raise RuntimeError(f"b200_gemm_a8w8_plan_query failed ({rc}): {_lib.strerror(rc)}")
    return pl.as_dict()


# --------------------------------------------------------------------------------------------------------- quantizer
def _up(n: int, to: int) -> int:
    return -(-n // to) * to


def _row_major_strides(rows: int, cols: int, stride) -> bool:
    return (cols <= 1 or stride[1] == 1) and (rows <= 1 or stride[0] >= cols)


def _row_major(x: torch.Tensor) -> torch.Tensor:
    return x if _row_major_strides(*x.shape, x.stride()) else x.contiguous()


_QUANT_SIZES = struct.Struct("@10q4i")  # b200_gemm_quantize_args behind its six pointers
_GROUPS = {"row": 1, "col": 2, "both": 3, "block": 4}


def _quant_sizes(rows, cols, ld, in_id, out_id, mode, sums_pitch, packed=False) -> bytes:
    pitch = _up(cols, 16)
    row_groups, col_groups = (_blocks(rows), _blocks(cols)) if packed else (_blocks(rows) if mode == 4 else rows, cols)
    return _QUANT_SIZES.pack(rows, cols, ld, pitch, 1, row_groups, pitch, col_groups, 1, sums_pitch, in_id, out_id, mode, int(packed))


@functools.lru_cache(maxsize=4096)
def _quantize_plan(shape, stride, x_dtype, group, dtype) -> tuple:
    """(mode, shapes and strides of the outputs, parts of the argument block) for an input of this shape; raises what the call
    raises."""
    if group not in _GROUPS:
        raise ValueError(f"unknown group {group!r}; expected one of {tuple(_GROUPS)}")
    if dtype not in _F8_ID:
        raise ValueError(f"quantize_a8 makes float8_e4m3fn or float8_e5m2, not {dtype}")
    if x_dtype not in _F_ID:
        raise ValueError(f"quantize_a8 takes float32, bfloat16 or float16, not {x_dtype}")
    assert len(shape) == 2, f"quantize_a8 takes a matrix, got {len(shape)} dimensions"
    rows, cols = shape
    if not _row_major_strides(rows, cols, stride):
        raise ValueError(f"x must be row-major: expected stride(1) == 1; got shape={tuple(shape)} and stride={stride}")
    mode, pitch = _GROUPS[group], _up(cols, 16)
    n_rows = _blocks(rows) if mode == 4 else rows
    sizes = _quant_sizes(rows, cols, stride[0] if rows > 1 else cols, _F_ID[x_dtype], _F8_ID[dtype], mode, 0)
    # the product reads the scales of 128 rows at a time: rows are the contiguous dimension
    row = ((n_rows, _blocks(cols)), (1, n_rows)) if mode != 2 else None
    col = (_blocks(rows), cols) if mode in (2, 3) else None
    return rows, cols, pitch, sizes, row, col


def _launch_quantize(x, dtype, plan, index) -> tuple:
    """On the current device and stream."""
    rows, cols, pitch, sizes, row, col = plan
    device = x.device
    got = []
    q_row = s_row = q_col = s_col = 0
    if row is not None:
        q = torch.empty(rows, pitch, dtype=dtype, device=device)
        s = torch.empty_strided(*row, dtype=torch.float32, device=device)
        q_row, s_row = q.data_ptr(), s.data_ptr()
        got += [q if pitch == cols else q[:, :cols], s]
    if col is not None:
        q = torch.empty(rows, pitch, dtype=dtype, device=device)
        s = torch.empty(*col, dtype=torch.float32, device=device)
        q_col, s_col = q.data_ptr(), s.data_ptr()
        got += [q if pitch == cols else q[:, :cols], s]
    rc = _lib.fast("b200_gemm_quantize_a8")(_POINTERS.pack(x.data_ptr(), q_row, s_row, q_col, s_col, 0) + sizes, raw_stream(index))
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
    plan = _quantize_plan(x.shape, x.stride(), x.dtype, group, dtype)
    index = x.get_device()
    assert index >= 0, "quantize_a8 runs on CUDA tensors only (there is no CPU path)"
    if stream is None and is_current(index):
        return _launch_quantize(x, dtype, plan, index)
    with on_device(index, stream):
        return _launch_quantize(x, dtype, plan, index)


# ------------------------------------------------------------------------------------------------------ linear layer
# A step of the layer is six launches, seven with a bias, and a launch through the public calls costs the host more than the
# GPU needs for it at ordinary sizes. The layer checks its tensors once, keeps each pass's operands in one buffer, and works out
# sizes, offsets and argument blocks once per combination of sizes and types (`_forward_plan`, `_backward_plan`).
class _Pieces:
    """Offsets of the pieces of one allocation, each on a 256-byte boundary."""

    def __init__(self):
        self.size = 0

    def add(self, nbytes: int) -> int:
        at = self.size
        self.size += _up(nbytes, 256)
        return at

    def quantized(self, rows: int, cols: int, by_col: bool = False) -> tuple:
        """(values, exponent tiles for 128 rows and four groups of columns, or the other way round) of a matrix; the values'
        pitch is a multiple of 16."""
        return self.add(rows * _up(cols, 16)), self.tiles(cols, rows) if by_col else self.tiles(rows, cols)

    def tiles(self, rows: int, k: int) -> int:
        return self.add(512 * _blocks(rows) * -(-_blocks(k) // 4))


# The layer's launches leave in one call: records of b200_gemm_sequence, whose constant parts are worked out once.
_QUANT_RECORD, _GEMM_RECORD, _REDUCE_RECORD = "q6P96s", "q6P176s8s", "q3P40s"
_REDUCE_SIZES = struct.Struct("@3q4i")


def _run(records: bytes, stream) -> None:
    rc = _lib.fast("b200_gemm_sequence")(records, stream)
    if rc != 0:
        raise RuntimeError(f"b200_gemm_sequence failed ({rc}): {_lib.strerror(rc)}")


def _packed_policy(m, n, k, num_sms) -> tuple:
    """Tiling of a product whose scales are exponent tiles, as the fields of b200_gemm_policy: CTA pairs with 256 x 256 tiles or
    CTAs with 128 x 128, by whole waves times the microseconds of a tile and of a K block in it (1024 x 2048 x 4096: pairs 16.5
    us, single CTAs 14.2; 2048 x 4096 x 4096: 30.1 and 46.2; 4096 x 4096 x 128: 13.1 and 10.3)."""
    pairs = -(-(-(-m // 256) * -(-n // 256)) // max(1, num_sms // 2)) * (2.2 + _blocks(k) * 0.36)
    single = -(-(-(-m // 128) * -(-n // 128)) // num_sms) * (0.9 + _blocks(k) * 0.31)
    return (256 if pairs < single else 128, 0, 1, 8 if m > 1024 else 0, 0, 2 if pairs < single else 1) + (0,) * 10


def _gemm_sizes(m, n, k, lda, ldb, scale_strides, a_t, b_t, a_id, b_id, out_id, bias_id, num_sms) -> bytes:
    return _SIZES.pack(m, n, k, lda, ldb, n, *scale_strides, a_t, b_t, a_id, b_id, 2, 2, out_id, bias_id, *_packed_policy(m, n, k, num_sms))


class _ForwardPlan:
    def __init__(self, m, n, k, x_ld, x_dtype, w_ld, w_dtype, bias_dtype, need_x, need_w, num_sms):
        e4 = _lib.DTYPE_E4M3
        temp, keep = _Pieces(), _Pieces()
        self.xr = temp.quantized(m, k)
        # what the backward pass reads: x by columns and the weight, as far as they are needed
        self.xc = keep.quantized(m, k, True) if need_w else None
        self.wq = (keep if need_x else temp).quantized(n, k)
        self.wt = keep.tiles(k, n) if need_x else None  # the weight's scales as dx needs them, with K = n
        self.temp_size, self.keep_size = temp.size, keep.size
        self.quant_x = _quant_sizes(m, k, x_ld, _F_ID[x_dtype], e4, 3 if need_w else 1, 0, True)
        self.quant_w = _quant_sizes(n, k, w_ld, _F_ID[w_dtype], e4, 4, 0, True)
        kp = _up(k, 16)
        self.gemm = _gemm_sizes(m, n, k, kp, kp, (1, _blocks(m), 1, _blocks(n)), False, True, e4, e4, _F_ID[x_dtype],
                                0 if bias_dtype is None else _F_ID[bias_dtype], num_sms) if m and n and k else None
        self.records = struct.Struct("@" + 2 * _QUANT_RECORD + _GEMM_RECORD + "q")


class _BackwardPlan:
    def __init__(self, m, n, k, g_ld, g_dtype, g_id, x_dtype, w_dtype, b_dtype, need_x, need_w, need_b, num_sms):
        e4 = _lib.DTYPE_E4M3
        temp = _Pieces()
        by_col = need_w or need_b
        self.gr = temp.quantized(m, n) if need_x else None
        self.gc = temp.quantized(m, n, True) if by_col else None
        self.pitch = _up(n, 4)
        self.sums = temp.add(4 * _blocks(m) * self.pitch) if need_b else None
        self.temp_size = temp.size
        self.quant = (_quant_sizes(m, n, g_ld, _F_ID[g_dtype], g_id, 3 if need_x and by_col else 2 if by_col else 1, self.pitch, True)
                      if m and n else None)
        np_, kp, full = _up(n, 16), _up(k, 16), m and n and k
        self.dx = _gemm_sizes(m, k, n, np_, kp, (1, _blocks(m), 1, _blocks(k)), False, False, g_id, e4, _F_ID[x_dtype], 0, num_sms) if full else None
        self.dw = _gemm_sizes(n, k, m, np_, kp, (1, _blocks(n), 1, _blocks(k)), True, False, g_id, e4, _F_ID[w_dtype], 0, num_sms) if full else None
        self.reduce = _REDUCE_SIZES.pack(self.pitch, 1, self.pitch, _blocks(m), _F_ID[b_dtype], 0, 0) if need_b else None
        self.records = struct.Struct("@" + _QUANT_RECORD + (_GEMM_RECORD if need_x and full else "") + (_GEMM_RECORD if need_w and full else "")
                                     + (_REDUCE_RECORD if need_b else "") + "q") if m and n else None


_forward_plan = functools.lru_cache(maxsize=1024)(_ForwardPlan)
_backward_plan = functools.lru_cache(maxsize=1024)(_BackwardPlan)


def _at(base: int, offsets) -> tuple:
    return (0, 0) if offsets is None else (base + offsets[0], base + offsets[1])


class _Linear8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, grad_dtype, grad_enabled):
        shape, (n, k) = x.shape, weight.shape
        m = math.prod(shape[:-1])
        x2, w2 = _row_major(x if x.ndim == 2 else x.reshape(m, k)), _row_major(weight)
        # needs_input_grad says what the tensors require, also where no backward pass can follow
        need_x, need_w = ctx.needs_input_grad[:2] if grad_enabled else (False, False)
        index, device = x.get_device(), x.device
        bias_dtype = None if bias is None else bias.dtype
        plan = _forward_plan(m, n, k, x2.stride(0) if m > 1 else k, x.dtype, w2.stride(0) if n > 1 else k, weight.dtype, bias_dtype, need_x,
                             need_w, device_sms(index))
        with on_device(index, None):
            stream = raw_stream(index)
            y = torch.empty(*shape[:-1], n, dtype=x.dtype, device=device)
            keep = torch.empty(plan.keep_size, dtype=torch.uint8, device=device)
            if plan.gemm is not None:
                temp = torch.empty(plan.temp_size, dtype=torch.uint8, device=device)
                temp_ptr, keep_ptr = temp.data_ptr(), keep.data_ptr()
                xr, wq = _at(temp_ptr, plan.xr), _at(keep_ptr if need_x else temp_ptr, plan.wq)
                _run(plan.records.pack(
                    2, x2.data_ptr(), *xr, *_at(keep_ptr, plan.xc), 0, plan.quant_x,
                    2, w2.data_ptr(), *wq, 0, keep_ptr + plan.wt if need_x else 0, 0, plan.quant_w,
                    1, xr[0], wq[0], xr[1], wq[1], y.data_ptr(), 0 if bias is None else bias.data_ptr(), plan.gemm,
                    _workspace_for(device, stream).status_bytes, 0), stream)
            elif k == 0:
                y.zero_() if bias is None else y.copy_(bias.expand_as(y))
        ctx.save_for_backward(keep)
        ctx.plan = plan
        ctx.meta = (shape, m, n, k, x.dtype, weight.dtype, bias_dtype, _F8_ID[grad_dtype])
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        (keep,) = ctx.saved_tensors
        shape, m, n, k, x_dtype, w_dtype, b_dtype, g_id = ctx.meta
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        g = _row_major(dy if dy.ndim == 2 else dy.reshape(m, n))  # an expanded gradient (of a sum) is spread out here
        index, device = dy.get_device(), dy.device
        plan = _backward_plan(m, n, k, g.stride(0) if m > 1 else n, g.dtype, g_id, x_dtype, w_dtype, b_dtype, need_x, need_w, need_b,
                              device_sms(index))
        dx = dw = db = None
        with on_device(index, None):
            stream = raw_stream(index)
            status = _workspace_for(device, stream).status_bytes
            temp = torch.empty(plan.temp_size, dtype=torch.uint8, device=device)
            base, keep_ptr = temp.data_ptr(), keep.data_ptr()
            gr, gc = _at(base, plan.gr), _at(base, plan.gc)
            records = [2, g.data_ptr(), *gr, *gc, base + plan.sums if need_b else 0, plan.quant]
            if need_x:
                dx = torch.empty(shape, dtype=x_dtype, device=device)
                if plan.dx is not None:
                    records += (1, gr[0], keep_ptr + ctx.plan.wq[0], gr[1], keep_ptr + ctx.plan.wt, dx.data_ptr(), 0, plan.dx, status)
                else:
                    dx.zero_()
            if need_w:
                dw = torch.empty(n, k, dtype=w_dtype, device=device)
                if plan.dw is not None:
                    xc = _at(keep_ptr, ctx.plan.xc)
                    records += (1, gc[0], xc[0], gc[1], xc[1], dw.data_ptr(), 0, plan.dw, status)
                else:
                    dw.zero_()
            if need_b:
                db = torch.empty(plan.pitch, dtype=b_dtype, device=device)
                if plan.records is not None:  # the columns' sums over each 128 rows, added in order
                    records += (3, base + plan.sums, db.data_ptr(), 0, plan.reduce)
                else:
                    db.zero_()
                if plan.pitch != n:
                    db = db[:n]
            if plan.records is not None and (need_x or need_w or need_b):
                _run(plan.records.pack(*records, 0), stream)
        return dx, dw, db, None, None


def linear_a8w8(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                grad_dtype: torch.dtype = torch.float8_e4m3fn) -> torch.Tensor:
    """y = x @ weight.T (+ bias) in 8-bit floating point, with its backward pass; x [..., K], weight [N, K], bias [N] of float32,
    bfloat16 or float16, y in x's type.

    Forward: x in groups of 128 along K, the weight in 128 x 128 blocks, both e4m3. Backward: the output's gradient is quantized
    to `grad_dtype` once along N (for dx, against the weight as it was quantized) and once along the rows (for dweight, against x
    quantized along the rows in the forward pass, unless gradients are disabled). The tensor cores apply the scales and sum
    32 groups, whose sums are added in fp32. dbias is the sum of the unquantized gradient in fp32, in a fixed order.
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
    return _Linear8.apply(x, weight, bias, grad_dtype, torch.is_grad_enabled())
