"""The 8-bit block-scaled product, its quantizer and the linear layer against plain 64-bit forms.

Bounds. An 8-bit product is exact in fp32. With S = sum |a| |b| times the scales, a K block's sum on the tensor core is off
by a few units of 2^-23 of its S (four accumulating instructions; 8 units are allowed), each fp32 addition of the running
sum and each product of scales adds at most 2^-24 of S: |error| <= (8 + blocks) * 2^-23 * S, plus half a step of the output type.
"""
import ctypes as C
import functools

import pytest
import torch

from flydsl_examples_b200 import _lib
from flydsl_examples_b200.gemm_a16w16 import _workspace_for, check_status
from flydsl_examples_b200.gemm_a8w8 import gemm_a8w8, linear_a8w8, plan, quantize_a8

pytestmark = pytest.mark.gpu

DEV = "cuda"
E4, E5 = torch.float8_e4m3fn, torch.float8_e5m2
LARGEST = {E4: 448.0, E5: 57344.0}


def blocks(n):
    return -(-n // 128)


def operand(g, rows, k, dtype, block, transposed, pad=0):
    """[rows, k] 8-bit values, `transposed`: rows contiguous, with rows padded to 16 bytes + pad, and random scales. The padding
    and everything around the matrix is NaN."""
    r, c = (k, rows) if transposed else (rows, k)
    pitch = -(-c // 16) * 16 + pad
    buf = torch.full((r, pitch), 0x7F, dtype=torch.uint8, device=DEV)
    vals = torch.randn(r, c, generator=g, device=DEV) * 2
    buf[:, :c] = vals.to(dtype).view(torch.uint8)
    q = buf.view(dtype)[:, :c]
    q = q.t() if transposed else q
    nb = blocks(rows) if block else rows
    s = torch.rand(nb, blocks(k), generator=g, device=DEV) + 0.25
    return q, s


def values(q, s):
    """64-bit values of an operand [rows, k]."""
    rows, k = q.shape
    wide = s.double().repeat_interleave(128, 1)[:, :k]
    if s.shape[0] != rows:
        wide = wide.repeat_interleave(128, 0)[:rows]
    return q.float().double() * wide


def check(got, a, sa, b, sb, bias=None):
    """got against A @ B^T (+ bias); a [M, K], b [N, K]."""
    va, vb = values(a, sa), values(b, sb)
    ref, mag = va @ vb.t(), va.abs() @ vb.abs().t()
    if bias is not None:
        ref = ref + bias.double()
        mag = mag + bias.double().abs()
    bound = (8 + blocks(a.shape[1])) * 2.0 ** -23 * mag + torch.finfo(got.dtype).eps / 2 * ref.abs()
    bound = bound * (1 + 1e-6) + (2.0 ** -25 if got.dtype == torch.float16 else 0)  # half a step among fp16 subnormals
    bad = (got.double() - ref).abs() > bound
    bad |= ~got.isfinite()
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), got[bad][:4].tolist(), ref[bad][:4].tolist())


def run(m, n, k, layout="nt", ad=E4, bd=E4, a_block=False, b_block=True, out_dtype=torch.bfloat16, bias=False, kw={}, seed=0, pad=0,
        repeats=1):
    g = torch.Generator(device=DEV).manual_seed(seed + m + 7 * n + 13 * k)
    a, sa = operand(g, m, k, ad, a_block, layout[0] == "t", pad)
    b, sb = operand(g, n, k, bd, b_block, layout[1] == "n", pad)
    bv = torch.randn(n, generator=g, device=DEV).to(torch.bfloat16) if bias else None
    out = torch.full((m, n), float("nan"), dtype=out_dtype, device=DEV)
    for _ in range(repeats):
        got = gemm_a8w8(a, sa, b.t(), sb.t(), out, bias=bv, user_kwargs=kw, layout=layout)
    check_status()
    assert got.data_ptr() == out.data_ptr()
    check(got, a, sa, b, sb, bv)
    return got


VARIANTS = [
    {"tile_n": 128}, {"tile_n": 128, "cta_group": 2}, {"tile_n": 256, "cta_group": 2}, {"tile_n": 64}, {"tile_n": 32}, {"tile_n": 16},
]


@pytest.mark.parametrize("kw", VARIANTS, ids=str)
@pytest.mark.parametrize("b_block", [True, False])
def test_variants_small(kw, b_block):
    run(200, 264, 328, kw=kw, b_block=b_block)


@pytest.mark.parametrize("kw", VARIANTS, ids=str)
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.float16])
def test_variants_outputs_and_bias(kw, out_dtype):
    run(300, 520, 1000, kw=kw, out_dtype=out_dtype, bias=True)
    run(300, 520, 1000, kw=kw, out_dtype=out_dtype, bias=True, a_block=True, b_block=False)


@pytest.mark.parametrize("layout", ["nn", "nt", "tn", "tt"])
@pytest.mark.parametrize("kw", [{"tile_n": 128}, {"tile_n": 256, "cta_group": 2}, {"tile_n": 128, "swap_ab": True}, {}], ids=str)
@pytest.mark.parametrize("types", [(E4, E4), (E5, E4), (E4, E5), (E5, E5)], ids=["44", "54", "45", "55"])
def test_layouts_and_types(layout, kw, types):
    run(272, 400, 656, layout, *types, a_block=False, b_block=False, kw=kw, pad=32)


@pytest.mark.parametrize("tile", [16, 32, 64, 128])
@pytest.mark.parametrize("split", [1, 2, 4, 8, 16])
@pytest.mark.parametrize("swap", [True, False])
def test_cluster_split(tile, split, swap):
    # 17 K blocks: uneven slices; ragged against every tile
    m, n = (tile - 3, 390) if swap else (390, tile * 2 - 3)
    kw = {"tile_n": tile, "split_k": split, "swap_ab": swap}
    x = run(m, n, 2100, kw=kw, out_dtype=torch.float32, bias=True, b_block=swap, repeats=3)
    y = run(m, n, 2100, kw=kw, out_dtype=torch.float32, bias=True, b_block=swap)
    assert torch.equal(x, y)  # summed in a fixed order


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 33, 64, 65, 127, 129, 255, 513])
@pytest.mark.parametrize("n,k", [(128, 128), (130, 4096), (1000, 16), (7, 1), (2050, 129)])
def test_default_policy_odd_sizes(m, n, k):
    run(m, n, k)
    run(m, n, k, b_block=False, a_block=True, out_dtype=torch.float32, bias=True)


@pytest.mark.parametrize("m,n,k", [(2048, 4096, 4096), (1000, 3000, 4100), (4096, 2304, 1152), (20000, 130, 260), (130, 20000, 260)])
@pytest.mark.parametrize("layout", ["nt", "nn", "tn"])
def test_ordinary_sizes(m, n, k, layout):
    run(m, n, k, layout, b_block=layout != "tn", repeats=2)


def test_unaligned_output_rows_and_storage_offset():
    # an odd N leaves C's rows off 16-byte boundaries: no TMA stores
    for kw in ({"tile_n": 256, "cta_group": 2}, {"tile_n": 128}, {}):
        run(300, 517, 400, kw=kw, bias=True)
    g = torch.Generator(device=DEV).manual_seed(5)
    a, sa = operand(g, 70, 300, E4, False, False)
    b, sb = operand(g, 90, 300, E4, True, False)
    flat = torch.full((70 * 90 + 9,), 7.0, dtype=torch.bfloat16, device=DEV)
    got = gemm_a8w8(a, sa, b.t(), sb.t(), flat[3:-6])
    check(got.view(70, 90), a, sa, b, sb)
    assert (flat[:3] == 7).all() and (flat[-6:] == 7).all()


def test_scale_strides_and_extremes():
    g = torch.Generator(device=DEV).manual_seed(6)
    m, n, k = 260, 300, 520
    a, sa = operand(g, m, k, E4, False, False)
    b, sb = operand(g, n, k, E4, True, False)
    want = gemm_a8w8(a, sa, b.t(), sb.t(), out_dtype=torch.float32)
    wide = torch.full((m * 2, blocks(k) * 3), float("nan"), device=DEV)
    wide[::2, ::3] = sa
    assert torch.equal(want, gemm_a8w8(a, wide[::2, ::3], b.t(), sb.t(), out_dtype=torch.float32))
    assert torch.equal(want, gemm_a8w8(a, sa.t().contiguous().t(), b.t(), sb.t().contiguous(), out_dtype=torch.float32))
    # one scale for everything: a broadcast tensor of strides 0
    one = torch.full((1, 1), 0.5, device=DEV)
    got = gemm_a8w8(a, one.expand(m, blocks(k)), b.t(), one.expand(blocks(k), blocks(n)), out_dtype=torch.float32)
    check(got, a, one.expand(m, blocks(k)), b, one.expand(blocks(n), blocks(k)))
    # scales at the ends of fp32: the two of a block are multiplied in fp32 and stay finite here
    check(gemm_a8w8(a, sa * 2.0 ** 60, b.t(), sb.t() * 2.0 ** -60, out_dtype=torch.float32), a, sa * 2.0 ** 60, b, sb * 2.0 ** -60)


def test_nan_stays_in_its_row_and_column():
    g = torch.Generator(device=DEV).manual_seed(7)
    for kw in ({"tile_n": 128}, {"tile_n": 256, "cta_group": 2}, {"tile_n": 64, "swap_ab": True, "split_k": 2}):
        a, sa = operand(g, 140, 300, E4, False, False)
        b, sb = operand(g, 150, 300, E4, True, False)
        a.view(torch.uint8)[5, 299] = 0x7F
        b.view(torch.uint8)[149, 0] = 0xFF
        got = gemm_a8w8(a, sa, b.t(), sb.t(), user_kwargs=kw, out_dtype=torch.float32)
        bad = got.isnan()
        assert bad[5].all() and bad[:, 149].all() and int(bad.sum()) == 140 + 150 - 1


def test_other_stream_graph_and_two_callers():
    g = torch.Generator(device=DEV).manual_seed(8)
    a, sa = operand(g, 33, 1024, E4, False, False)
    b, sb = operand(g, 640, 1024, E4, True, False)
    want = gemm_a8w8(a, sa, b.t(), sb.t())
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    got = gemm_a8w8(a, sa, b.t(), sb.t(), stream=s)
    s.synchronize()
    assert torch.equal(want, got)
    # captured and replayed on changed inputs
    out = torch.empty_like(want)
    gemm_a8w8(a, sa, b.t(), sb.t(), out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, qs = quantize_a8(want, "row")
        gemm_a8w8(a, sa, b.t(), sb.t(), out)
    a.view(torch.uint8).copy_(a.view(torch.uint8).flip(0).contiguous())
    sa.copy_(sa.flip(0).contiguous())
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want.flip(0))
    # two streams at once
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.empty_like(want) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for st, o in zip(streams, outs):
            with torch.cuda.stream(st):
                gemm_a8w8(a, sa, b.t(), sb.t(), o)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], want.flip(0))
    check_status()


# --------------------------------------------------------------------------------------------------------- quantizer
def groups64(x, rg, cg, dtype):
    """Scales by comparison and exact quotients in fp64; torch's conversion of the exact fp32 quotient."""
    big = LARGEST[dtype]
    r, c = x.shape
    v = torch.where(x.isfinite(), x, torch.zeros_like(x)).double().abs()
    v = torch.nn.functional.pad(v, (0, -c % cg, 0, -r % rg)).view(-(-r // rg), rg, -(-c // cg), cg).amax((1, 3))
    e = torch.full_like(v, -126.0)
    for p in range(-126, 128):  # smallest power of two that suffices
        e = torch.where(v / 2.0 ** (p - 1) > big, torch.full_like(e, float(p)), e) if p > -126 else e
    s = torch.where(v > 0, torch.exp2(e), torch.ones_like(v))
    wide = s.repeat_interleave(rg, 0)[:r].repeat_interleave(cg, 1)[:, :c]
    return (x.double() / wide).float().to(dtype), s.float()


def same8(q, want):
    nan = q.float().isnan()
    return torch.equal(nan, want.float().isnan()) and torch.equal(q.float()[~nan], want.float()[~nan])


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 130), (128, 128), (129, 257), (32, 7168), (300, 1000), (1000, 72)])
@pytest.mark.parametrize("x_dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("dtype", [E4, E5])
def test_quantize(rows, cols, x_dtype, dtype):
    g = torch.Generator(device=DEV).manual_seed(rows * 1000 + cols)
    x = (torch.randn(rows, cols, generator=g, device=DEV) * torch.exp2(torch.randint(-12, 13, (rows, cols), generator=g, device=DEV))).to(x_dtype)
    for group, sizes in (("row", [(1, 128)]), ("col", [(128, 1)]), ("both", [(1, 128), (128, 1)]), ("block", [(128, 128)])):
        got = quantize_a8(x, group, dtype)
        for i, (rg, cg) in enumerate(sizes):
            q, s = groups64(x, rg, cg, dtype)
            assert got[2 * i].dtype == dtype and same8(got[2 * i], q), group
            assert torch.equal(got[2 * i + 1], s), group


@pytest.mark.parametrize("dtype", [E4, E5])
def test_quantize_borders_and_specials(dtype):
    x = torch.zeros(256, 256, device=DEV)
    x[1, :] = torch.tensor([448.0, 448.00003, 447.9, 57344.0, 57344.004, 1e-38, 1e-45, 3e38] * 32, device=DEV)
    x[2, 3], x[2, 4], x[2, 5], x[2, 6] = float("inf"), float("-inf"), float("nan"), 3.0
    x[3, :128] = 2.0 ** -120
    x[4, :128] = 1.1754944e-38  # smallest normal
    x[5, :128] = 1e-45          # smallest subnormal
    x[6, :] = float("nan")
    x[7, 0], x[7, 1:9] = 448.0, torch.tensor([8.5, 9.5, 0.0009765625, 0.0029296875, -8.5, 17.0, 19.0, 2.0 ** -10], device=DEV)  # ties
    for group, (rg, cg) in (("row", (1, 128)), ("col", (128, 1)), ("block", (128, 128))):
        q, s = groups64(x, rg, cg, dtype)
        got, gs = quantize_a8(x, group, dtype)
        assert torch.equal(gs, s) and same8(got, q)


def test_quantize_strides_offsets_and_neighbours():
    g = torch.Generator(device=DEV).manual_seed(9)
    big = torch.randn(140, 701, generator=g, device=DEV).to(torch.bfloat16)
    for x in (big[3:133, 5:330], big[:, 1:], big[::2, 8:264], big[:1, :5], big[7:8].expand(1, 701)):
        for group in ("row", "col", "block"):
            got, want = quantize_a8(x, group), quantize_a8(x.contiguous(), group)
            assert same8(got[0], want[0]) and torch.equal(got[1], want[1])


def test_quantize_feeds_the_product():
    g = torch.Generator(device=DEV).manual_seed(10)
    x = torch.randn(77, 500, generator=g, device=DEV).to(torch.bfloat16)
    w = torch.randn(333, 500, generator=g, device=DEV).to(torch.bfloat16)
    dy = torch.randn(77, 333, generator=g, device=DEV).to(torch.bfloat16)
    xr, sxr, xc, sxc = quantize_a8(x, "both")
    wq, sw = quantize_a8(w, "block")
    gr, sgr, gc, sgc = quantize_a8(dy, "both", E5)
    check(gemm_a8w8(xr, sxr, wq.t(), sw.t(), out_dtype=torch.float32), xr, sxr, wq, sw)
    check(gemm_a8w8(gr, sgr, wq, sw, layout="nn", out_dtype=torch.float32), gr, sgr, wq.t(), sw.t())
    check(gemm_a8w8(gc.t(), sgc.t(), xc, sxc, layout="tn", out_dtype=torch.float32), gc.t(), sgc.t(), xc.t(), sxc.t())


# ------------------------------------------------------------------------------------------------------ linear layer
def reference_linear(x, w, b, dy, grad_dtype):
    """(value, magnitude, blocks) of y, dx, dw in fp64 by the definition."""
    def val(t, rg, cg, dtype):
        q, s = groups64(t.float(), rg, cg, dtype)
        return q.float().double() * s.double().repeat_interleave(rg, 0)[: t.shape[0]].repeat_interleave(cg, 1)[:, : t.shape[1]]
    wq = val(w, 128, 128, E4)
    pairs = ((val(x, 1, 128, E4), wq.t()), (val(dy, 1, 128, grad_dtype), wq), (val(dy, 128, 1, grad_dtype).t(), val(x, 128, 1, E4)))
    got = [(p @ q, p.abs() @ q.abs(), blocks(p.shape[1])) for p, q in pairs]
    if b is not None:
        got[0] = (got[0][0] + b.double(), got[0][1] + b.double().abs(), got[0][2])
    return got


def near(got, ref):
    want, mag, nb = ref
    eps = torch.finfo(got.dtype).eps / 2
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 0
    return bool(((got.double() - want).abs() <= (8 + nb) * 2.0 ** -23 * mag + eps * 1.000001 * want.abs() + tiny).all())


@pytest.mark.parametrize("m,n,k", [(1, 8, 16), (100, 72, 200), (300, 513, 260), (512, 384, 640)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("grad_dtype", [E4, E5])
def test_linear_and_its_gradients(m, n, k, dtype, grad_dtype):
    g = torch.Generator(device=DEV).manual_seed(m + n + k)
    x = torch.randn(m, k, generator=g, device=DEV).to(dtype).requires_grad_()
    w = (torch.randn(n, k, generator=g, device=DEV) / k ** 0.5).to(dtype).requires_grad_()
    b = torch.randn(n, generator=g, device=DEV).to(dtype).requires_grad_()
    dy = torch.randn(m, n, generator=g, device=DEV).to(dtype)
    y = linear_a8w8(x, w, b, grad_dtype)
    y.backward(dy)
    ref = reference_linear(x.detach(), w.detach(), b.detach(), dy, grad_dtype)
    assert y.dtype == x.grad.dtype == w.grad.dtype == b.grad.dtype == dtype
    for got, want in zip((y.detach(), x.grad, w.grad), ref):
        assert near(got, want)
    want, mag = dy.double().sum(0), dy.double().abs().sum(0)
    assert ((b.grad.double() - want).abs() <= (m + 1) * 2.0 ** -24 * mag + torch.finfo(dtype).eps / 2 * 1.000001 * want.abs()).all()
    check_status()


def test_linear_gradient_against_differences():
    # quantization is piecewise constant, so differences are taken on operands that 8 bits hold exactly: small integers whose
    # groups all have the same scale; the layer is then the exact bilinear product
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randint(-4, 5, (6, 256), generator=g, device=DEV).float()
    w = torch.randint(-4, 5, (5, 256), generator=g, device=DEV).float()
    x[:, ::128], w[:, ::128] = 7.0, 7.0
    dy = torch.randint(-2, 3, (6, 5), generator=g, device=DEV).float()
    xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
    linear_a8w8(xl, wl).backward(dy)
    loss = lambda x_, w_: (linear_a8w8(x_, w_) * dy).sum().item()  # noqa: E731
    for i, j in ((0, 1), (3, 77), (5, 255)):
        up, down = x.clone(), x.clone()
        up[i, j] += 1
        down[i, j] -= 1
        assert (loss(up, w) - loss(down, w)) / 2 == xl.grad[i, j].item()
    for i, j in ((0, 1), (4, 200)):
        up, down = w.clone(), w.clone()
        up[i, j] += 1
        down[i, j] -= 1
        assert (loss(x, up) - loss(x, down)) / 2 == wl.grad[i, j].item()


def test_linear_partial_gradients_shapes_and_broadcast_gradient():
    g = torch.Generator(device=DEV).manual_seed(4)
    x = torch.randn(2, 3, 160, generator=g, device=DEV).to(torch.bfloat16)
    w = torch.randn(96, 160, generator=g, device=DEV).to(torch.bfloat16)
    b = torch.randn(96, generator=g, device=DEV).to(torch.bfloat16)
    dy = torch.ones(1, 1, 1, device=DEV, dtype=torch.bfloat16).expand(2, 3, 96)
    full = None
    for need in ((1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1)):
        leaves = [t.clone().requires_grad_(bool(f)) for t, f in zip((x, w, b), need)]
        y = linear_a8w8(*leaves)
        assert y.shape == (2, 3, 96)
        y.backward(dy)
        got = [t.grad for t in leaves]
        full = full or got
        for f, a_, b_ in zip(need, got, full):
            assert (a_ is None) if not f else torch.equal(a_, b_)
    with torch.no_grad():
        assert linear_a8w8(x[:0], w, b).shape == (0, 3, 96)
    leaves = [t.clone().requires_grad_() for t in (x[:0], w, b)]
    linear_a8w8(*leaves).sum().backward()
    assert leaves[0].grad.shape == (0, 3, 160) and not leaves[1].grad.any() and not leaves[2].grad.any()
    xt = x.view(6, 160).t().contiguous().t()  # column-major input
    assert torch.equal(linear_a8w8(xt, w, b), linear_a8w8(x.view(6, 160), w, b))


def test_no_offset_over_32_bits_wraps():
    # 2^31 bytes of output: the last rows lie past a signed 32-bit offset
    m, n, k = 270000, 4096, 128
    g = torch.Generator(device=DEV).manual_seed(11)
    a, sa = operand(g, m, k, E4, False, False)
    b, sb = operand(g, n, k, E4, True, False)
    got = gemm_a8w8(a, sa, b.t(), sb.t())
    for lo in (0, 131000, m - 300):
        check(got[lo:lo + 300], a[lo:lo + 300], sa[lo:lo + 300], b, sb)
    q, s = quantize_a8(got, "both")[:2]
    q2, s2 = quantize_a8(got[m - 256:].contiguous(), "row")
    assert same8(q[m - 256:], q2) and torch.equal(s[m - 256:], s2)


def test_linear_captured_with_its_backward_and_changed_in_place():
    g = torch.Generator(device=DEV).manual_seed(12)
    x = torch.randn(130, 256, generator=g, device=DEV).to(torch.bfloat16)
    w = torch.randn(200, 256, generator=g, device=DEV).to(torch.bfloat16)
    b = torch.randn(200, generator=g, device=DEV).to(torch.bfloat16)
    dy = torch.randn(130, 200, generator=g, device=DEV).to(torch.bfloat16)

    def step(x_, w_, b_):
        leaves = [t.detach().requires_grad_() for t in (x_, w_, b_)]
        y = linear_a8w8(*leaves)
        return (y.detach(),) + torch.autograd.grad(y, leaves, dy)
    want = step(x, w, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, w, b)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(x, w, b)
    for t in got:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    x.copy_(x.flip(0).contiguous())
    dy.copy_(dy.flip(0).contiguous())
    graph.replay()
    again = step(x, w, b)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, again))
    xl = x.clone().requires_grad_()
    y = linear_a8w8(xl, w, b)
    y.relu_()  # the output is no view, so it may be changed in place
    y.sum().backward()
    assert xl.grad.isfinite().all()
    check_status()


def test_threads_share_the_calls():
    import threading

    g = torch.Generator(device=DEV).manual_seed(13)
    a, sa = operand(g, 50, 512, E4, False, False)
    b, sb = operand(g, 300, 512, E4, True, False)
    x = torch.randn(50, 512, generator=g, device=DEV)
    want, want_q = gemm_a8w8(a, sa, b.t(), sb.t()), quantize_a8(x, "both")
    torch.cuda.synchronize()
    bad = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                got, q = gemm_a8w8(a, sa, b.t(), sb.t()), quantize_a8(x, "both")
                torch.cuda.current_stream().synchronize()
                if not torch.equal(got, want) or not all(torch.equal(p.float(), r.float()) for p, r in zip(q, want_q)):
                    bad.append(1)
    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
    check_status()


@pytest.mark.parametrize("kw", [{"tile_n": 256, "cta_group": 2}, {"tile_n": 64}, {"tile_n": 16, "swap_ab": True, "split_k": 2}], ids=str)
@pytest.mark.parametrize("bias_dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_bias_types_and_offsets(kw, bias_dtype):
    g = torch.Generator(device=DEV).manual_seed(14)
    a, sa = operand(g, 150, 300, E4, False, False)
    b, sb = operand(g, 277, 300, E4, False, False)
    wide = torch.randn(600, generator=g, device=DEV).to(bias_dtype)
    for bias in (wide[:277], wide[3:280], wide[:554:2]):  # aligned, off 16 bytes, strided
        check(gemm_a8w8(a, sa, b.t(), sb.t(), bias=bias, user_kwargs=kw, out_dtype=torch.float32), a, sa, b, sb, bias)


# ------------------------------------------------------------------------------------------------------ exponent tiles
# Every element of a block carries its scales into the tensor core, whose accumulator then holds the sum over all blocks: four
# accumulating instructions per block instead of four in all, so |error| <= (8 * blocks) * 2^-23 * S.
def tiles_of(s, fill):
    """[K groups of four, row tiles, 512] bytes of power-of-two scales s [rows, K blocks]; bytes of no scale are `fill`."""
    rows, nb = s.shape
    out = torch.full((-(-nb // 4), blocks(rows), 512), fill, dtype=torch.uint8, device=s.device)
    r = torch.arange(rows, device=s.device)
    at = r % 32 * 16 + r % 128 // 32 * 4
    for b in range(nb):
        out[b // 4, r // 128, at + b % 4] = (s[:, b].contiguous().view(torch.int32) >> 23).to(torch.uint8)
    return out


def quantize_packed(x, mode, dtype, fill):
    rows, cols = x.shape
    pitch = -(-cols // 16) * 16
    q = [torch.zeros(rows, pitch, dtype=torch.uint8, device=DEV) for _ in range(2)]
    by_row = torch.full((-(-blocks(cols) // 4), blocks(rows), 512), fill, dtype=torch.uint8, device=DEV)
    by_col = torch.full((-(-blocks(rows) // 4), blocks(cols), 512), fill, dtype=torch.uint8, device=DEV)
    a = _lib.QuantizeArgs()
    for key, v in dict(x=x.data_ptr(), q_row=q[0].data_ptr(), s_row=by_row.data_ptr(), q_col=q[1].data_ptr(), s_col=by_col.data_ptr(), rows=rows,
                       cols=cols, ldx=x.stride(0), ldq_row=pitch, sr_group=blocks(rows), ldq_col=pitch, sc_group=blocks(cols),
                       in_dtype={torch.float32: 1, torch.bfloat16: 2, torch.float16: 3}[x.dtype], out_dtype=4 if dtype == E4 else 5, mode=mode,
                       packed=1).items():
        setattr(a, key, v)
    assert _lib.load().b200_gemm_quantize_a8(C.byref(a), torch.cuda.current_stream().cuda_stream) == 0
    return [t[:, :cols].view(dtype) for t in q], by_row, by_col


@pytest.mark.parametrize("rows,cols", [(1, 1), (128, 128), (130, 700), (517, 140), (640, 1100)])
@pytest.mark.parametrize("mode", [1, 2, 3, 4])
def test_quantizer_writes_the_same_scales_as_tiles(rows, cols, mode):
    g = torch.Generator(device=DEV).manual_seed(rows + cols)
    for x_dtype, dtype in ((torch.bfloat16, E4), (torch.float32, E5), (torch.float16, E4)):
        x = (torch.randn(rows, cols, generator=g, device=DEV) * torch.exp2(torch.randint(-9, 5, (rows, cols), generator=g, device=DEV))).to(x_dtype)
        x[rows // 2] = 0
        (q_row, q_col), by_row, by_col = quantize_packed(x, mode, dtype, 0xAB)
        if mode == 4:
            q, s = quantize_a8(x, dtype=dtype, group="block")
            assert torch.equal(by_row, tiles_of(s.repeat_interleave(128, 0)[:rows], 0xAB))
            assert torch.equal(by_col, tiles_of(s.t().repeat_interleave(128, 0)[:cols], 0xAB))
            assert torch.equal(q.view(torch.uint8), q_row.view(torch.uint8))
            continue
        if mode & 1:
            q, s = quantize_a8(x, dtype=dtype, group="row")
            assert torch.equal(by_row, tiles_of(s, 0xAB)) and torch.equal(q.view(torch.uint8), q_row.view(torch.uint8))
        else:
            assert (by_row == 0xAB).all()
        if mode & 2:
            q, s = quantize_a8(x, dtype=dtype, group="col")
            assert torch.equal(by_col, tiles_of(s.t(), 0xAB)) and torch.equal(q.view(torch.uint8), q_col.view(torch.uint8))
        else:
            assert (by_col == 0xAB).all()


def run_packed(m, n, k, layout, tile_n, ad=E4, bd=E4, out_dtype=torch.bfloat16, bias=False, spread=12, shift=0):
    g = torch.Generator(device=DEV).manual_seed(m + 3 * n + 5 * k)
    a, _ = operand(g, m, k, ad, False, layout[0] == "t")
    b, _ = operand(g, n, k, bd, False, layout[1] == "n")
    sa, sb = (torch.exp2(torch.randint(-spread, spread + 1, (r, blocks(k)), generator=g, device=DEV).float() + d) for r, d in ((m, shift), (n, -shift)))
    ta, tb = tiles_of(sa, 0xFF), tiles_of(sb, 0xFF)  # 0xFF is NaN: what belongs to no row must not matter
    bv = torch.randn(n, generator=g, device=DEV) if bias else None
    guard = torch.full((m * n + 64,), 7.0, dtype=out_dtype, device=DEV)
    args = _lib.Args8()
    for key, v in dict(a=a.data_ptr(), b=b.data_ptr(), a_scale=ta.data_ptr(), b_scale=tb.data_ptr(), out=guard.data_ptr(), bias=bv.data_ptr() if bias else None,
                       m=m, n=n, k=k, lda=a.stride(0) if layout[0] == "n" else a.stride(1), ldb=b.stride(0) if layout[1] == "t" else b.stride(1),
                       ldo=n, sa_row=1, sa_kb=ta.shape[1], sb_col=1, sb_kb=tb.shape[1], a_trans=int(layout[0] == "t"), b_trans=int(layout[1] == "t"),
                       a_dtype=4 if ad == E4 else 5, b_dtype=4 if bd == E4 else 5, a_block=2, b_block=2, bias_dtype=1 if bias else 0,
                       out_dtype={torch.float32: 1, torch.bfloat16: 2, torch.float16: 3}[out_dtype],
                       status=_workspace_for(torch.device(DEV, torch.cuda.current_device()), torch.cuda.current_stream().cuda_stream).status_ptr).items():
        setattr(args, key, v)
    args.policy.tile_n, args.policy.cta_group, args.policy.group_m = tile_n, 2 if tile_n == 256 else 1, 8 if m > 1024 else 0
    assert _lib.load().b200_gemm_a8w8(C.byref(args), torch.cuda.current_stream().cuda_stream) == 0
    check_status()
    assert (guard[m * n:] == 7).all()
    got = guard[: m * n].view(m, n)
    va, vb = values(a, sa), values(b, sb)
    ref, mag = va @ vb.t(), va.abs() @ vb.abs().t()
    if bias:
        ref, mag = ref + bv.double(), mag + bv.double().abs()
    bound = (8 * blocks(k) + 1) * 2.0 ** -23 * mag + torch.finfo(out_dtype).eps / 2 * 1.000001 * ref.abs()
    bad = ~((got.double() - ref).abs() <= bound)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), got[bad][:4].tolist(), ref[bad][:4].tolist())


@pytest.mark.parametrize("tile_n", [128, 256])
@pytest.mark.parametrize("layout", ["nt", "nn", "tn", "tt"])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (128, 128, 128), (256, 256, 512), (129, 257, 513), (300, 140, 1700), (1100, 530, 640), (2600, 2700, 150)])
def test_product_with_exponent_tiles(m, n, k, layout, tile_n):
    run_packed(m, n, k, layout, tile_n)
    run_packed(m, n, k, layout, tile_n, E5, E4, torch.float32, bias=True)


def test_product_with_exponent_tiles_of_extreme_scales():
    run_packed(200, 300, 700, "nt", 256, out_dtype=torch.float32, spread=20, shift=100)
    run_packed(200, 300, 700, "tn", 128, E4, E5, torch.float32, spread=20, shift=-100)


def test_linear_of_tiny_by_huge_values():
    g = torch.Generator(device=DEV).manual_seed(9)
    x = (torch.randn(150, 600, generator=g, device=DEV) * torch.exp2(torch.randint(-110, -89, (150, 1), generator=g, device=DEV).float())).requires_grad_()
    w = (torch.randn(200, 600, generator=g, device=DEV) * 2.0 ** 100).requires_grad_()
    dy = torch.randn(150, 200, generator=g, device=DEV) * 2.0 ** -20
    y = linear_a8w8(x, w)
    y.backward(dy)
    for got, (want, mag, nb) in zip((y.detach(), x.grad, w.grad), reference_linear(x.detach(), w.detach(), None, dy, E4)):
        bound = (8 * nb + 1) * 2.0 ** -23 * mag + 2.0 ** -24 * 1.000001 * want.abs() + 2.0 ** -149
        assert ((got.double() - want).abs() <= bound).all()
    check_status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("grad_dtype", [E4, E5])
def test_bias_gradient_of_infinities_and_nan(dtype, grad_dtype):
    # the sum of the gradient as it is, whatever the 8-bit copy makes of an infinity
    inf, nan = float("inf"), float("nan")
    g = torch.Generator(device=DEV).manual_seed(15)
    x = torch.randn(300, 64, generator=g, device=DEV).to(dtype)
    w = torch.randn(140, 64, generator=g, device=DEV).to(dtype)
    dy = torch.randint(-4, 5, (300, 140), generator=g, device=DEV).to(dtype)  # finite sums are exact
    for i, j, v in ((3, 1, inf), (299, 2, -inf), (5, 3, inf), (250, 3, -inf), (6, 4, nan), (7, 5, inf), (7, 6, inf), (8, 6, nan), (130, 139, -inf)):
        dy[i, j] = v
    want = dy.double().sum(0).to(dtype)
    for need in ((0, 0, 1), (1, 0, 1), (1, 1, 1)):  # columns alone, and with rows
        x_, w_, b = x.clone().requires_grad_(bool(need[0])), w.clone().requires_grad_(bool(need[1])), torch.zeros(140, dtype=dtype, device=DEV, requires_grad=True)
        linear_a8w8(x_, w_, b, grad_dtype).backward(dy)
        assert torch.equal(b.grad.isnan(), want.isnan()) and torch.equal(b.grad[~want.isnan()], want[~want.isnan()])
        if need[0]:  # the quantized copy has them as before
            q, s = groups64(dy.float(), 1, 128, grad_dtype)
            odd = ~q.float().isfinite().all(1)
            assert odd.any() and not x_.grad[odd].isfinite().all(1).any() and x_.grad[~odd].isfinite().all()
    check_status()


@pytest.mark.parametrize("kw", [{"tile_n": 128}, {"tile_n": 256, "cta_group": 2}, {"tile_n": 64, "swap_ab": True}], ids=str)
@pytest.mark.parametrize("group", [1, 3, 1 << 30, (1 << 31) - 1])
def test_groups_of_tile_rows(kw, group):
    run(700, 1100, 300, kw={**kw, "group_m": group}, repeats=2)


@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
def test_linear_without_gradients_does_only_the_forward_work(monkeypatch, mode):
    from flydsl_examples_b200 import gemm_a8w8 as module

    g = torch.Generator(device=DEV).manual_seed(16)
    x = torch.randn(70, 300, generator=g, device=DEV)
    w, b = (torch.nn.Parameter(torch.randn(*s, generator=g, device=DEV)) for s in ((90, 300), (90,)))
    plans = []
    forward_plan = module._forward_plan
    monkeypatch.setattr(module, "_forward_plan", lambda *a: plans.append(forward_plan(*a)) or plans[-1])
    want = linear_a8w8(x, w, b)
    assert plans[0].xc is not None and plans[0].keep_size > 0
    with mode():
        got = linear_a8w8(x.clone().requires_grad_(), w, b)
    assert not got.requires_grad and torch.equal(got, want)
    assert plans[1].xc is plans[1].wt is None and plans[1].keep_size == 0  # x by rows only, nothing kept
    xl = x.clone().requires_grad_()  # and with them enabled again
    linear_a8w8(xl, w, b).sum().backward()
    assert xl.grad is not None and w.grad is not None and b.grad is not None
    check_status()


@pytest.mark.parametrize("shape,n", [((2, 3, 0), 5), ((0,), 5), ((0, 3, 0), 5), ((2, 3, 0), 0), ((0, 4), 5), ((3, 4), 0)])
def test_linear_of_empty_dimensions(shape, n):
    k = shape[-1]
    for bias in (True, False):
        leaves = [torch.ones(*s, device=DEV, requires_grad=True) for s in (shape, (n, k), (n,))]
        y = linear_a8w8(leaves[0], leaves[1], leaves[2] if bias else None)
        assert y.shape == (*shape[:-1], n) and (k or (y == float(bias)).all())
        y.sum().backward()
        assert leaves[0].grad.shape == shape and leaves[1].grad.shape == (n, k) and not leaves[1].grad.any()
        if bias:
            assert (leaves[2].grad == y.numel() // max(n, 1)).all()
    check_status()


@pytest.mark.parametrize("positive", [False, True])
@pytest.mark.parametrize("k", [4096, 4100, 8200, 16384, 65536])
def test_long_sums_do_not_drift(k, positive):
    # The tensor core cuts its sums off instead of rounding them, so values of one sign drift by up to a unit per instruction; 32
    # blocks of 128 at most are summed that way (8 units of 2^-23 for each block, as above), their sums in fp32: half a unit for each.
    g = torch.Generator(device=DEV).manual_seed(k)
    draw = torch.rand if positive else torch.randn
    units = 8 * min(blocks(k), 32) + -(-blocks(k) // 32) / 2
    for long in ("features", "tokens"):
        if long == "features":
            x, w = (draw(*s, generator=g, device=DEV) for s in ((130, k), (140, k)))
            got = linear_a8w8(x, w)
            (q, s), (p, t) = quantize_a8(x, "row"), quantize_a8(w, "block")
        else:
            x, dy = (draw(*s, generator=g, device=DEV) for s in ((k, 130), (k, 140)))
            w = torch.zeros(140, 130, device=DEV, requires_grad=True)
            linear_a8w8(x, w).backward(dy)
            got = w.grad
            (q, s), (p, t) = quantize_a8(dy, "col"), quantize_a8(x, "col")
            q, s, p, t = q.t(), s.t(), p.t(), t.t()
        a, b = values(q, s), values(p, t)
        want, mag = a @ b.t(), a.abs() @ b.abs().t()
        bound = units * 2.0 ** -23 * mag + 2.0 ** -24 * want.abs()
        assert ((got.double() - want).abs() <= bound).all()
    check_status()


@pytest.mark.parametrize("tile_n", [128, 256])
@pytest.mark.parametrize("layout", ["nt", "nn", "tn", "tt"])
@pytest.mark.parametrize("m,n,k", [(129, 257, 4096), (129, 257, 4097), (300, 530, 8300), (2600, 2700, 4200), (40, 50, 12288)])
def test_product_with_exponent_tiles_of_many_blocks(m, n, k, layout, tile_n):
    run_packed(m, n, k, layout, tile_n, out_dtype=torch.float32)
