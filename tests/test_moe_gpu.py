"""The few-token mixture-of-experts layer against its formula in 64 bits.

Bounds, from the roundings that happen: the first product's fp32 sums (H / 16 accumulating instructions, 2^-23 of the sum of
magnitudes each), the exponentials and the softmax (32 units of 2^-23, and 2 |g| more for the SiLU's), half a step of half a
step of the 16-bit type for each h (a value and a remainder), the second product's fp32 sums, and half a step for the
result. They are propagated entry by entry.
"""
import pytest
import torch

from flydsl_examples_b200.gemm_a16w16 import check_status, gemm_a16w16
from flydsl_examples_b200.moe_a16w16 import moe_a16w16

pytestmark = pytest.mark.gpu

DEV = "cuda"
U23 = 2.0 ** -23


def inputs(t, e, h, i, dtype, seed=0, logits_dtype=torch.float32):
    g = torch.Generator(device=DEV).manual_seed(seed + t * 3 + e * 5 + h * 7 + i)
    x = torch.randn(t, h, generator=g, device=DEV).to(dtype)
    logits = torch.randn(t, e, generator=g, device=DEV).to(logits_dtype)
    w13 = (torch.randn(e, 2 * i, h, generator=g, device=DEV) * h ** -0.5).to(dtype)
    w2 = (torch.randn(e, h, i, generator=g, device=DEV) * i ** -0.5).to(dtype)
    return x, logits, w13, w2


def routing(logits, top_k, renorm):
    """{token: [(expert, weight)]} by plain comparison; a zero weight is no choice."""
    got = {}
    for t, row in enumerate(logits.double().cpu().tolist()):
        ids = sorted(range(len(row)), key=lambda j: (-row[j], j))[:top_k]
        top = row[ids[0]]
        if top == float("-inf"):
            got[t] = []
            continue
        p = torch.tensor(row, dtype=torch.float64).sub(top).exp()
        total = p[ids].sum() if renorm else p.sum()
        got[t] = [(j, float(p[j] / total)) for j in ids if float(p[j]) > 0]
    return got


def reference(x, logits, w13, w2, top_k, renorm):
    """Value and bound of every output."""
    t_n, h_n = x.shape
    i_n = w2.shape[2]
    eps = torch.finfo(x.dtype).eps / 2
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 0.0  # half a step among fp16 subnormals
    y = torch.zeros(t_n, h_n, dtype=torch.float64, device=DEV)
    err, mag = torch.zeros_like(y), torch.zeros_like(y)
    for t, chosen in routing(logits, top_k, renorm).items():
        for e, p in chosen:
            a, b, v = w13[e].double(), w2[e].double(), x[t].double()
            gu, s = a @ v, (a.abs() @ v.abs()) * (h_n / 16 + 8) * U23
            g, u = gu[:i_n], gu[i_n:]
            silu = g / (1 + torch.exp(-g))
            hv = p * silu * u
            d = p * (1.1 * u.abs() * s[:i_n] + (silu.abs() + 1.1 * s[:i_n]) * s[i_n:]) + hv.abs() * (32 + 2 * g.abs()) * U23
            d = d + (hv.abs() + d) * eps * eps + tiny
            y[t] += b @ hv
            err[t] += b.abs() @ d
            mag[t] += b.abs() @ (hv.abs() + d)
    err += mag * (top_k * i_n / 16 + 24) * U23
    return y, err + (y.abs() + err) * eps + tiny


def check(got, x, logits, w13, w2, top_k, renorm=True):
    y, bound = reference(x, logits, w13, w2, top_k, renorm)
    bad = ~((got.double() - y).abs() <= bound * (1 + 1e-6))
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), got[bad][:4].tolist(), y[bad][:4].tolist(), bound[bad][:4].tolist())


def run(t, e, h, i, top_k, dtype=torch.bfloat16, renorm=True, **kw):
    x, logits, w13, w2 = inputs(t, e, h, i, dtype, **kw)
    out = torch.full((t, h), float("nan"), dtype=dtype, device=DEV)
    got = moe_a16w16(x, logits, w13, w2, top_k, out, renormalize=renorm)
    check_status()
    assert got.data_ptr() == out.data_ptr()
    check(got, x, logits, w13, w2, top_k, renorm)
    return got


@pytest.mark.parametrize("t", [1, 2, 15, 16, 17, 32, 33, 64])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_tokens(t, dtype):
    run(t, 8, 256, 192, 2, dtype)


@pytest.mark.parametrize("e,top_k", [(1, 1), (2, 2), (5, 3), (16, 16), (33, 1), (128, 8), (200, 6), (512, 16)])
@pytest.mark.parametrize("renorm", [True, False])
def test_experts(e, top_k, renorm):
    run(5, e, 128, 72, top_k, renorm=renorm)
    run(40, e, 72, 128, top_k, torch.float16, renorm=renorm)


@pytest.mark.parametrize("h,i", [(8, 8), (8, 200), (200, 8), (1000, 520), (136, 64), (128, 1032), (2048, 768), (7168, 256)])
def test_widths(h, i):
    run(3, 6, h, i, 2)
    run(20, 4, h, i, 3, torch.float16)


@pytest.mark.parametrize("logits_dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_logit_types_and_ties(logits_dtype):
    run(9, 24, 128, 64, 4, logits_dtype=logits_dtype)
    x, _, w13, w2 = inputs(4, 12, 128, 64, torch.bfloat16)
    logits = torch.zeros(4, 12, device=DEV, dtype=logits_dtype)
    logits[1, 3:9] = 1.0
    logits[2, ::2] = -0.0  # equal to 0: the lowest indices win
    logits[3, 11] = 5.0
    check(moe_a16w16(x, logits, w13, w2, 3), x, logits, w13, w2, 3)


def test_masked_experts():
    x, logits, w13, w2 = inputs(6, 10, 256, 128, torch.bfloat16)
    inf = float("inf")
    logits[0, :] = -inf                       # nothing left
    logits[1, 1:] = -inf                      # fewer than top_k left
    logits[2, :5] = torch.finfo(torch.float32).min
    logits[3, :] = torch.finfo(torch.float32).min  # the type's lowest value everywhere: equal shares
    logits[4, 3] = 1e30
    w13[9] = float("nan")                     # an expert that no token may choose
    w2[9] = inf
    logits[:, 9] = -inf
    logits[3, 9] = -inf
    for renorm in (True, False):
        got = moe_a16w16(x, logits, w13, w2, 4, renormalize=renorm)
        assert not got[0].any()
        check(got, x, logits, w13, w2, 4, renorm)
    all_masked = moe_a16w16(x, torch.full_like(logits, -inf), w13, w2, 4, torch.full_like(x, 3.0))
    assert not all_masked.any()
    check_status()


def test_nan_stays_with_its_token():
    x, logits, w13, w2 = inputs(7, 10, 256, 128, torch.bfloat16)
    want = moe_a16w16(x, logits, w13, w2, 3)
    logits2 = logits.clone()
    logits2[2, 4] = float("nan")
    logits2[5, 0] = float("inf")
    x2 = x.clone()
    x2[3, 100] = float("nan")
    x2[6, 0] = float("inf")
    got = moe_a16w16(x2, logits2, w13, w2, 3)
    assert got[2].isnan().all() and got[5].isnan().all() and got[3].isnan().all() and not got[6].isfinite().all()
    for t in (0, 1, 4):
        assert torch.equal(got[t], want[t])


def test_strides():
    x, logits, w13, w2 = inputs(6, 5, 128, 72, torch.float16)
    want = moe_a16w16(x, logits, w13, w2, 2)
    nan = float("nan")

    def inside(t, before, after):
        big = torch.full([n + a + b for n, a, b in zip(t.shape, before, after)], nan, dtype=t.dtype, device=DEV)
        view = big[tuple(slice(a, a + n) for n, a in zip(t.shape, before))]
        view.copy_(t)
        return view
    got = moe_a16w16(inside(x, (1, 8), (0, 16)), inside(logits, (0, 3), (2, 0)), inside(w13, (1, 2, 8), (0, 1, 0)), inside(w2, (0, 1, 16), (1, 0, 8)), 2)
    assert torch.equal(got, want)
    assert torch.equal(moe_a16w16(x, logits.t().contiguous().t(), w13, w2, 2), want)
    assert torch.equal(moe_a16w16(x[:1].expand(1, 128), logits[:1], w13, w2, 2), want[:1])
    same = moe_a16w16(x, logits[:1].expand(6, 5), w13, w2, 2)  # broadcast logits
    check(same, x, logits[:1].expand(6, 5), w13, w2, 2)


def test_behind_the_router_and_beside_split_k():
    # the layer as it is used: the router's product, then the experts; a ticket split-K GEMM shares the stream's workspace
    g = torch.Generator(device=DEV).manual_seed(2)
    t, e, h, i = 32, 384, 512, 64
    x, _, w13, w2 = inputs(t, e, h, i, torch.bfloat16)
    wr = (torch.randn(e, h, generator=g, device=DEV) * h ** -0.5).to(torch.bfloat16)
    out = torch.empty(t, h, dtype=torch.bfloat16, device=DEV)
    logits = torch.empty(t, e, device=DEV)
    for _ in range(3):
        gemm_a16w16(x, wr.t(), logits, user_kwargs={"tile_n": 128, "split_k": 4}, out_dtype=torch.float32)
        moe_a16w16(x, logits, w13, w2, 8, out)
    check_status()
    assert torch.allclose(logits.double(), x.double() @ wr.double().t(), atol=1e-4)
    check(out, x, logits, w13, w2, 8)


def test_repeats_streams_and_two_graphs():
    x, logits, w13, w2 = inputs(24, 16, 512, 264, torch.bfloat16)
    out = torch.empty_like(x)
    want = moe_a16w16(x, logits, w13, w2, 4).clone()
    for _ in range(5):
        assert torch.equal(moe_a16w16(x, logits, w13, w2, 4, out), want)  # the same bits every time
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = moe_a16w16(x, logits, w13, w2, 4, stream=s)
    s.synchronize()
    assert torch.equal(got, want)
    x2, logits2 = x.flip(0).contiguous(), logits.flip(0).contiguous()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for a, b in ((x, logits), (x2, logits2)):
        gr = torch.cuda.CUDAGraph()
        o = torch.empty_like(x)
        with torch.cuda.graph(gr):
            moe_a16w16(a, b, w13, w2, 4, o)
        graphs.append(gr)
        outs.append(o)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(20):  # replayed at once on two streams, with eager calls between
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        moe_a16w16(x, logits, w13, w2, 4, out)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want.flip(0)) and torch.equal(out, want)
    check_status()


def test_growing_workspace_and_no_tokens():
    small = inputs(1, 4, 64, 64, torch.bfloat16)
    big = inputs(64, 64, 64, 2048, torch.bfloat16)
    o1, o2 = torch.empty_like(small[0]), torch.empty_like(big[0])
    for _ in range(2):
        moe_a16w16(*small, 2, o1)
        moe_a16w16(*big, 8, o2)
    check(o1, *small, 2)
    check(o2, *big, 8)
    assert moe_a16w16(small[0][:0], small[1][:0], *small[2:], 2).shape == (0, 64)


def test_weights_past_32_bit_offsets():
    # 2^31 elements of gate/up weights: the last expert's lie past a 32-bit element offset (and 2^32 bytes)
    e, h, i = 40, 7168, 4096
    g = torch.Generator(device=DEV).manual_seed(1)
    w13 = torch.zeros(e, 2 * i, h, dtype=torch.bfloat16, device=DEV)
    w2 = torch.zeros(e, h, i, dtype=torch.bfloat16, device=DEV)
    for k in (0, e - 1):
        w13[k].normal_(generator=g).mul_(h ** -0.5)
        w2[k].normal_(generator=g).mul_(i ** -0.5)
    x = torch.randn(2, h, generator=g, device=DEV).to(torch.bfloat16)
    logits = torch.full((2, e), -5.0, device=DEV)
    logits[0, e - 1], logits[1, 0], logits[1, e - 1] = 4.0, 2.0, 3.0
    check(moe_a16w16(x, logits, w13, w2, 2), x, logits, w13, w2, 2)


def test_threads_on_one_stream():
    # torch's default stream is one for all threads: layers of different sizes and inputs from several threads, with ticket split-K
    # GEMMs between, each thread's results as when it is alone
    import threading

    layers = [(inputs(t, e, 256, i, torch.bfloat16, seed=t), k) for t, e, i, k in ((3, 40, 264, 4), (17, 8, 512, 2), (64, 24, 64, 6), (9, 12, 1032, 3))]
    want = [moe_a16w16(*a, k) for a, k in layers]
    g = torch.Generator(device=DEV).manual_seed(5)
    a = torch.randn(96, 4096, generator=g, device=DEV).to(torch.bfloat16)
    b = torch.randn(256, 4096, generator=g, device=DEV).to(torch.bfloat16)
    product = torch.empty(96, 256, device=DEV)
    kw = {"tile_n": 128, "split_k": 8}
    gemm_a16w16(a, b.t(), product, user_kwargs=kw, out_dtype=torch.float32)
    want_product = product.clone()
    torch.cuda.synchronize()
    bad, go = [], threading.Barrier(len(layers) + 1)

    def thread(body):
        def work():
            try:
                go.wait()
                for _ in range(200):
                    body()
            except Exception as e:
                bad.append(e)
        return threading.Thread(target=work)

    got = [[] for _ in layers]
    threads = [thread(lambda i=i: got[i].append(moe_a16w16(*layers[i][0], layers[i][1]))) for i in range(len(layers))]
    threads.append(thread(lambda: gemm_a16w16(a, b.t(), product, user_kwargs=kw, out_dtype=torch.float32)))
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not bad and torch.equal(product, want_product)
    for y, of_thread in zip(want, got):
        assert len(of_thread) == 200 and all(torch.equal(y, v) for v in of_thread)
    check_status()


# In fp16 the second product's operand h = p * silu(g) * u is a value rounded at h / 16 and a remainder kept 2^11 times as large: half a
# step of half a step, (2^-11)^2 of h, or half of the remainder's smallest step, 2^-25 * 2^-11 * 16 = 2^-32. The error of the SiLU's
# exponential grows with |g| only where g is negative; from -40 on h itself is below 2^-32 (40 e^-40 |u| < 2e-13 for |u| < 1000).
@pytest.mark.parametrize("x_size,w2_size", [(1, 1), (100, 1e-3), (200, 1e-4), (0.1, 4), (0.02, 30), (0.004, 200), (0.001, 1000)])
def test_small_and_large_activations_in_fp16(x_size, w2_size):
    x, logits, w13, w2 = inputs(5, 3, 256, 320, torch.float16)
    x, w2 = (x * x_size).half(), (w2.float() * w2_size).half()
    got = moe_a16w16(x, logits, w13, w2, 2)
    check_status()
    y = torch.zeros(5, 256, dtype=torch.float64, device=DEV)
    err, mag = torch.zeros_like(y), torch.zeros_like(y)
    for t, chosen in routing(logits, 2, True).items():
        for e, p in chosen:
            a, b, v = w13[e].double(), w2[e].double(), x[t].double()
            gu, s = a @ v, (a.abs() @ v.abs()) * (256 / 16 + 8) * U23
            g, u = gu[:320], gu[320:]
            silu = g / (1 + torch.exp(-g))
            hv = p * silu * u
            assert hv.abs().max() < 2 ** 20 * 0.99
            d = p * (1.1 * u.abs() * s[:320] + (silu.abs() + 1.1 * s[:320]) * s[320:]) + hv.abs() * (32 + 2 * g.abs().clamp(max=40)) * U23
            d = d + (hv.abs() + d) * 2.0 ** -22 + 2.0 ** -32
            y[t] += b @ hv
            err[t] += b.abs() @ d
            mag[t] += b.abs() @ (hv.abs() + d)
    err += mag * (2 * 320 / 16 + 24) * U23
    bound = err + (y.abs() + err) * 2.0 ** -11 + 2.0 ** -25
    assert y.abs().max() < 65504
    assert ((got.double() - y).abs() <= bound * (1 + 1e-6)).all()
