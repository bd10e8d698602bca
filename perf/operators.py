"""The 8-bit and mixture-of-experts operators as measured cases: inputs, plain forms, and the calls a user makes.

Four operators, `op` in a case:

* ``gemm``: C[M, N] = A[M, K] @ B[K, N] (+ bias[N]) with 8-bit floating-point operands and one fp32 scale for each block of
  128 along K (a vector of scales per row / column, or one per 128 x 128 block), fp32 accumulation, one rounding.
* ``quantize``: 16-bit or fp32 rows to 8-bit values and scales, in groups of 128 along a row, along a column, both in one
  pass, or in 128 x 128 blocks. The scale of a group is the smallest power of two that brings its largest finite
  magnitude down to the format's largest value, so dividing by it is exact and one rounding remains.
* ``linear``: one training step of a linear layer on the two operators above: output, and the gradients of input, weight
  and bias for a given output gradient.
* ``moe``: a mixture-of-experts layer for a few tokens from the router's logits: top-k, softmax, gate/up product, SiLU,
  down product, weighted sum.

With `own` false, `run` computes the plain form from elementary torch operations; with `own` true it calls the package.
"""
import math

import torch

own = False

_F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
_F8_MAX = {torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0}  # both 1.75 * 2^n
_F = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
GROUP = 128


# ------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one token of decoding against a square projection: streams 16.8 MB of weights, latency counts
        {"name": "gemm 1 token", "op": "gemm", "m": 1, "n": 4096, "k": 4096, "layout": "nt", "a": "e4m3", "b": "e4m3",
         "a_scale": "vector", "b_scale": "block", "out": "bf16", "bias": False},
        # a decoding batch of 32 against a wide feed-forward projection
        {"name": "gemm 32 tokens", "op": "gemm", "m": 32, "n": 14336, "k": 4096, "layout": "nt", "a": "e4m3", "b": "e4m3",
         "a_scale": "vector", "b_scale": "block", "out": "fp16", "bias": False},
        # an input gradient of odd sizes: e5m2 gradient rows against the weight as it is stored, K tail, ragged edges
        {"name": "gemm odd dgrad", "op": "gemm", "m": 1000, "n": 3000, "k": 4100, "layout": "nn", "a": "e5m2", "b": "e4m3",
         "a_scale": "vector", "b_scale": "block", "out": "bf16", "bias": True},
        # prefill / training forward of the largest square
        {"name": "gemm 8192", "op": "gemm", "m": 8192, "n": 8192, "k": 8192, "layout": "nt", "a": "e4m3", "b": "e4m3",
         "a_scale": "vector", "b_scale": "block", "out": "bf16", "bias": False},
        # activations of a decoding batch on their way into a product
        {"name": "quantize 32 tokens", "op": "quantize", "rows": 32, "cols": 7168, "x": "bf16", "to": "e4m3", "group": "row"},
        # activations of a training step: rows for the forward and input-gradient product, columns for the weight gradient
        {"name": "quantize both 16384", "op": "quantize", "rows": 16384, "cols": 8192, "x": "bf16", "to": "e4m3", "group": "both"},
        # one training step of a linear layer at an ordinary size
        {"name": "linear 2048", "op": "linear", "m": 2048, "n": 4096, "k": 4096, "x": "bf16", "bias": True},
        # the same with odd sizes, fp16, no bias
        {"name": "linear odd", "op": "linear", "m": 1000, "n": 3000, "k": 4100, "x": "fp16", "bias": False},
        # one token through a layer of many small experts: eight of 128 are read
        {"name": "moe 1 token", "op": "moe", "t": 1, "e": 128, "top_k": 8, "h": 2048, "i": 768, "x": "bf16", "renorm": True},
        # a decoding batch of 8 through few wide experts
        {"name": "moe 8 tokens", "op": "moe", "t": 8, "e": 16, "top_k": 2, "h": 4096, "i": 3584, "x": "bf16", "renorm": True},
        # a decoding batch of 32 through a wide hidden size: nearly every expert is read
        {"name": "moe 32 tokens", "op": "moe", "t": 32, "e": 32, "top_k": 8, "h": 7168, "i": 2048, "x": "bf16", "renorm": True},
        # odd token count, expert count and widths, fp16, weights not renormalised
        {"name": "moe odd", "op": "moe", "t": 13, "e": 10, "top_k": 3, "h": 1000, "i": 520, "x": "fp16", "renorm": False},
    ]


def _log(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(step, int(round(v / step)) * step)


def draw(rng):
    op = rng.choice(["gemm", "gemm", "quantize", "linear", "moe", "moe"])
    if op == "gemm":
        wgrad = rng.random() < 0.25
        return {"op": op, "m": _log(rng, 1, 8192), "n": _log(rng, 100, 8192), "k": _log(rng, 100, 8192),
                "layout": "tn" if wgrad else rng.choice(["nt", "nt", "nn", "tt", "tn"]), "a": rng.choice(["e4m3", "e4m3", "e5m2"]),
                "b": rng.choice(["e4m3", "e4m3", "e5m2"]), "a_scale": "vector",
                "b_scale": "vector" if wgrad else rng.choice(["block", "block", "vector"]),
                "out": rng.choice(["bf16", "fp16"]), "bias": rng.random() < 0.3}
    if op == "quantize":
        return {"op": op, "rows": _log(rng, 1, 16384), "cols": _log(rng, 64, 8192), "x": rng.choice(["bf16", "fp16", "fp32"]),
                "to": rng.choice(["e4m3", "e4m3", "e5m2"]), "group": rng.choice(["row", "col", "both", "block"])}
    if op == "linear":
        return {"op": op, "m": _log(rng, 16, 4096), "n": _log(rng, 128, 4096), "k": _log(rng, 128, 4096),
                "x": rng.choice(["bf16", "fp16"]), "bias": rng.random() < 0.5}
    e = _log(rng, 4, 128)
    h, i = _log(rng, 256, 7168, 8), _log(rng, 256, 4096, 8)
    while 6 * e * h * i > 2.8e9:  # the largest listed layer holds 2.8 GB of weights
        e = max(4, e // 2)
        if e == 4:
            i = max(256, i // 16 * 8)
    return {"op": op, "t": _log(rng, 1, 64), "e": e, "top_k": rng.randint(1, min(8, e)), "h": h, "i": i,
            "x": rng.choice(["bf16", "fp16"]), "renorm": rng.random() < 0.7}


# ------------------------------------------------------------------------------------------------------------ inputs
def _activations(gen, rows, cols, dtype):
    """Normal values with a few columns that are 16 times as large, as activations have them."""
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    x[:, torch.randperm(cols, generator=gen, device="cuda")[: max(1, cols // 200)]] *= 16
    return x.to(dtype)


def _spread(s, dim, n):
    """Each group's value for each of its 128 members along `dim`, cut to n."""
    return s.repeat_interleave(GROUP, dim).narrow(dim, 0, n)


def _pow2_scale(amax, largest):
    """The smallest power of two s >= 2^-126 with amax / s <= largest = 1.75 * 2^n; 1 for a group of zeros."""
    m, e = torch.frexp(amax)  # amax = m * 2^e, 0.5 <= m < 1
    n = math.frexp(largest)[1] - 1
    p = e - 1 - n + (m > 0.875).to(e.dtype)
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), p.clamp(min=-126)), torch.ones_like(amax))


def _amax(x, rows_per_group, cols_per_group):
    """Largest finite magnitude of each group."""
    r, c = x.shape
    a = torch.where(x.isfinite(), x, torch.zeros_like(x)).abs()
    a = torch.nn.functional.pad(a, (0, -c % cols_per_group, 0, -r % rows_per_group))
    return a.view(a.shape[0] // rows_per_group, rows_per_group, a.shape[1] // cols_per_group, cols_per_group).amax((1, 3))


def _quantize(x, to, rows_per_group, cols_per_group):
    """(8-bit values, scales) in the working precision of x (fp32 or fp64)."""
    s = _pow2_scale(_amax(x, rows_per_group, cols_per_group), _F8_MAX[to])
    wide = s.repeat_interleave(rows_per_group, 0)[: x.shape[0]].repeat_interleave(cols_per_group, 1)[:, : x.shape[1]]
    return (x / wide).float().to(to), s


def _padded(q):
    """The same values with rows that start on 16-byte boundaries, as the 8-bit product wants them."""
    pitch = -(-q.shape[1] // 16) * 16
    buf = torch.zeros(q.shape[0], pitch, dtype=torch.uint8, device=q.device)
    buf[:, : q.shape[1]] = q.view(torch.uint8)
    return buf.view(q.dtype)[:, : q.shape[1]]


def _operand(gen, rows, k, to, kind, transposed):
    """An 8-bit operand [rows, K] with its scales [rows or blocks of rows, blocks of K]; `transposed`: stored with the rows'
    index contiguous. Weights (blocks) carry scales that are no powers of two, as published checkpoints do."""
    g = 1 if kind == "vector" else GROUP
    q, s = _quantize(_activations(gen, rows, k, torch.float32), to, g, GROUP)
    if kind == "block":
        s = s * torch.rand(s.shape, generator=gen, device="cuda").add_(0.5)
    q = _padded(q.view(torch.uint8).t().contiguous().view(to)).t() if transposed else _padded(q)
    return q, s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    st = {"case": case}
    if op == "gemm":
        m, n, k, lay = case["m"], case["n"], case["k"], case["layout"]
        a, sa = _operand(gen, m, k, _F8[case["a"]], case["a_scale"], lay[0] == "t")
        b, sb = _operand(gen, n, k, _F8[case["b"]], case["b_scale"], lay[1] == "n")
        out_t = _F[case["out"]]
        # outputs of a product of K terms around 1: keep fp16 in range as a trained model's scales do
        sa = sa / math.sqrt(k)
        # sa [M, blocks]: stored with the tokens contiguous, the layout the quantizer leaves
        st.update(a=a, sa=sa.t().contiguous().t(), b=b.t(), sb=sb.t(),
                  bias=torch.randn(n, generator=gen, device="cuda").to(out_t) if case["bias"] else None,
                  out=torch.empty(m, n, dtype=out_t, device="cuda"))
    elif op == "quantize":
        st.update(x=_activations(gen, case["rows"], case["cols"], _F[case["x"]]))
    elif op == "linear":
        dt = _F[case["x"]]
        st.update(x=_activations(gen, case["m"], case["k"], dt).requires_grad_(),
                  w=(torch.randn(case["n"], case["k"], generator=gen, device="cuda") / math.sqrt(case["k"])).to(dt).requires_grad_(),
                  b=torch.randn(case["n"], generator=gen, device="cuda").to(dt).requires_grad_() if case["bias"] else None,
                  dy=(torch.randn(case["m"], case["n"], generator=gen, device="cuda") / 16).to(dt))
    else:
        t, e, h, i, dt = case["t"], case["e"], case["h"], case["i"], _F[case["x"]]
        st.update(x=torch.randn(t, h, generator=gen, device="cuda").to(dt),
                  logits=torch.randn(t, e, generator=gen, device="cuda"),
                  w13=torch.randn(e, 2 * i, h, generator=gen, device="cuda", dtype=dt).mul_(h ** -0.5),
                  w2=torch.randn(e, h, i, generator=gen, device="cuda", dtype=dt).mul_(i ** -0.5),
                  out=torch.empty(t, h, dtype=dt, device="cuda"))
    return st


# ------------------------------------------------------------------------------------------------------- plain forms
def _plain_gemm(a, sa, b, sb, bias, out_dtype):
    """A [M, K], B [K, N] with scales [M or blocks, blocks of K] and [blocks of K, N or blocks]."""
    m, k = a.shape
    n = b.shape[1]
    sa = _spread(sa, 1, k) if sa.shape[0] == m else _spread(_spread(sa, 1, k), 0, m)
    sb = _spread(sb, 0, k) if sb.shape[1] == n else _spread(_spread(sb, 0, k), 1, n)
    c = (a.float() * sa) @ (b.float() * sb)
    return (c if bias is None else c + bias.float()).to(out_dtype)


def _plain_quantize(x, to, group):
    x = x.float()
    if group == "both":
        return _quantize(x, to, 1, GROUP) + _quantize(x, to, GROUP, 1)
    return _quantize(x, to, *{"row": (1, GROUP), "col": (GROUP, 1), "block": (GROUP, GROUP)}[group])


def _plain_linear(x, w, b, dy):
    f8 = torch.float8_e4m3fn
    xr, sxr, xc, sxc = _plain_quantize(x, f8, "both")
    gr, sgr, gc, sgc = _plain_quantize(dy, f8, "both")
    wq, sw = _plain_quantize(w, f8, "block")
    y = _plain_gemm(xr, sxr, wq.t(), sw.t(), b, x.dtype)
    dx = _plain_gemm(gr, sgr, wq, sw, None, x.dtype)
    dw = _plain_gemm(gc.t(), sgc.t(), xc, sxc, None, w.dtype)
    return y, dx, dw, None if b is None else dy.float().sum(0).to(b.dtype)


def _plain_moe(x, logits, w13, w2, top_k, renorm):
    e, i2, h = w13.shape
    x, t = x.float(), x.shape[0]
    p = torch.softmax(logits.float(), 1)
    ids = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :top_k]  # ties go to the lowest index
    p = p.gather(1, ids)
    if renorm:
        p = p / p.sum(1, keepdim=True)
    if t * top_k < e:  # the chosen experts of each token
        g = (w13[ids].float() @ x.view(t, 1, h, 1)).squeeze(3)
        a = torch.nn.functional.silu(g[..., : i2 // 2]) * g[..., i2 // 2:]
        y = (w2[ids].float() @ a.unsqueeze(3)).squeeze(3)
        return (y * p.unsqueeze(2)).sum(1)
    g = x @ w13.float().transpose(1, 2)  # every expert for every token
    a = torch.nn.functional.silu(g[..., : i2 // 2]) * g[..., i2 // 2:]
    weight = torch.zeros(t, e, device=x.device).scatter_(1, ids, p)
    y = (a * weight.t().unsqueeze(2)) @ w2.float().transpose(1, 2)
    return y.sum(0)


def run(st):
    case = st["case"]
    op = case["op"]
    if own:
        from flydsl_examples_b200.gemm_a8w8 import gemm_a8w8, linear_a8w8, quantize_a8
        from flydsl_examples_b200.moe_a16w16 import moe_a16w16

        if op == "gemm":
            return gemm_a8w8(st["a"], st["sa"], st["b"], st["sb"], st["out"], bias=st["bias"], layout=case["layout"])
        if op == "quantize":
            return quantize_a8(st["x"], case["group"], _F8[case["to"]])
        if op == "linear":
            y = linear_a8w8(st["x"], st["w"], st["b"])
            leaves = (st["x"], st["w"]) + (() if st["b"] is None else (st["b"],))
            return (y.detach(),) + torch.autograd.grad(y, leaves, st["dy"])
        return moe_a16w16(st["x"], st["logits"], st["w13"], st["w2"], case["top_k"], st["out"], renormalize=case["renorm"])
    with torch.no_grad():
        if op == "gemm":
            return _plain_gemm(st["a"], st["sa"], st["b"], st["sb"], st["bias"], st["out"].dtype)
        if op == "quantize":
            return _plain_quantize(st["x"], _F8[case["to"]], case["group"])
        if op == "linear":
            got = _plain_linear(st["x"], st["w"], st["b"], st["dy"])
            return got if st["b"] is not None else got[:3]
        return _plain_moe(st["x"], st["logits"], st["w13"], st["w2"], case["top_k"], case["renorm"]).to(st["x"].dtype)


# -------------------------------------------------------------------------------------------------------------- work
def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    op = case["op"]
    blocks = lambda v: -(-v // GROUP)  # noqa: E731
    if op == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        scales = 4 * blocks(k) * (m + (n if case["b_scale"] == "vector" else blocks(n)))
        return {"bytes": m * k + n * k + scales + size[case["out"]] * (m * n + (n if case["bias"] else 0)), "flops": 2 * m * n * k}
    if op == "quantize":
        r, c, g = case["rows"], case["cols"], case["group"]
        scales = {"row": r * blocks(c), "col": blocks(r) * c, "both": r * blocks(c) + blocks(r) * c, "block": blocks(r) * blocks(c)}[g]
        return {"bytes": r * c * (size[case["x"]] + (2 if g == "both" else 1)) + 4 * scales, "flops": 3 * r * c}
    if op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        # x, w, dy in; y, dx, dw out (the 8-bit copies are the method's own)
        return {"bytes": 2 * (m * k + n * k + m * n) * 2, "flops": 6 * m * n * k}
    t, e, h, i = case["t"], case["e"], case["h"], case["i"]
    # each expert that a token chose is read once: the expected number of them for choices at random
    read = e * (1 - (1 - case["top_k"] / e) ** t)
    return {"bytes": int(read * 3 * h * i * 2 + 4 * t * h + 4 * t * e), "flops": 6 * t * case["top_k"] * h * i}


# ------------------------------------------------------------------------------------- the definitions in 64 bits
def _exact_groups(x, to, rg, cg):
    """Quantised values and scales by the definition: group by group in fp64, powers of two found by comparison."""
    big = _F8_MAX[to]
    r, c = x.shape
    pad = torch.zeros(-(-r // rg) * rg, -(-c // cg) * cg, dtype=torch.float64, device=x.device)
    pad[:r, :c] = x.double()
    v = pad.reshape(pad.shape[0] // rg, rg, pad.shape[1] // cg, cg)
    top = v.abs().amax(dim=(1, 3), keepdim=True)
    s = torch.exp2(torch.ceil(torch.log2(torch.where(top > 0, top, torch.ones_like(top)) / big)))
    s = torch.where(top / s > big, 2 * s, s)
    s = torch.where(top / (s / 2) <= big, s / 2, s)
    s = torch.where(top > 0, s.clamp(min=2.0 ** -126), torch.ones_like(s))
    # round to the format: 2^-mantissa steps of the value's own binade, no finer than the smallest subnormal
    man, low = (3, -6) if to == torch.float8_e4m3fn else (2, -14)
    z = v / s
    step = torch.exp2(torch.frexp(z)[1].double().sub(1).clamp(min=low) - man)
    q = torch.round(z / step) * step  # half to even
    return q.reshape(pad.shape)[:r, :c], s[:, 0, :, 0], (q * s).reshape(pad.shape)[:r, :c]


def _exact_value(q, s, rows):
    """8-bit values [rows, K] times their scales in fp64."""
    k = q.shape[1]
    row = torch.arange(rows, device=q.device) // (1 if s.shape[0] == rows else GROUP)
    return q.to(torch.float32).double() * s.double()[row][:, torch.arange(k, device=q.device) // GROUP]


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    with torch.no_grad():
        if op == "gemm":
            a = _exact_value(st["a"], st["sa"], case["m"])
            b = _exact_value(st["b"].t(), st["sb"].t(), case["n"])
            c = torch.mm(a, b.t())
            return c if st["bias"] is None else c.add_(st["bias"].double())
        if op == "quantize":
            to, got = _F8[case["to"]], []
            for rg, cg in {"row": [(1, GROUP)], "col": [(GROUP, 1)], "both": [(1, GROUP), (GROUP, 1)], "block": [(GROUP, GROUP)]}[case["group"]]:
                got += _exact_groups(st["x"], to, rg, cg)[:2]
            return tuple(got)
        if op == "linear":
            f8 = torch.float8_e4m3fn
            x, w, dy = st["x"].detach(), st["w"].detach(), st["dy"]
            wq = _exact_groups(w, f8, GROUP, GROUP)[2]
            y = _exact_groups(x, f8, 1, GROUP)[2] @ wq.t()
            dx = _exact_groups(dy, f8, 1, GROUP)[2] @ wq
            dw = _exact_groups(dy, f8, GROUP, 1)[2].t() @ _exact_groups(x, f8, GROUP, 1)[2]
            if st["b"] is None:
                return y, dx, dw
            return y + st["b"].detach().double(), dx, dw, dy.double().sum(0)
        x, logits = st["x"].double(), st["logits"].double().cpu()
        y = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
        chosen = {}
        for t in range(case["t"]):
            row = logits[t].tolist()
            ids = sorted(range(len(row)), key=lambda j: (-row[j], j))[: case["top_k"]]
            top = row[ids[0]]
            p = [math.exp(row[j] - top) for j in ids]
            total = sum(p) if case["renorm"] else sum(math.exp(v - top) for v in row)
            for j, v in zip(ids, p):
                chosen.setdefault(j, []).append((t, v / total))
        for j, pairs in chosen.items():
            rows = torch.tensor([t for t, _ in pairs], device=x.device)
            weight = torch.tensor([v for _, v in pairs], dtype=torch.float64, device=x.device)
            g = x[rows] @ st["w13"][j].double().t()
            gate, up = g[:, : case["i"]], g[:, case["i"]:]
            y[rows] += weight[:, None] * ((gate / (1 + torch.exp(-gate)) * up) @ st["w2"][j].double().t())
        return y
