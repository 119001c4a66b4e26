"""Cases, plain forms and exact values of the 8-bit path: the residual RMSNorm with an 8-bit output, the block quantiser,
the block-scaled matrix product and its form grouped by expert.

8-bit values are e4m3 (largest 448) or e5m2 (largest 57344); a block of 128 values (1 x 128 along the contraction, or a
128 x 128 tile of a weight) shares the scale 2^e with the smallest integer e that brings the block's largest magnitude to at
most that number."""
import math

import torch
import torch.nn.functional as F

own = False

E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2
FMT = {"e4m3": E4M3, "e5m2": E5M2}
TYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-5


def listed():
    return [
        # one token of a decoding step through the norm before a projection of a 4096-wide layer: latency
        {"name": "norm, one token", "op": "norm", "rows": 1, "cols": 4096, "dtype": "bf16", "fmt": "e4m3", "backward": False},
        # the norm of a layer over a training chunk, forward and backward (the benchmark's 8192 x 4096 chunk)
        {"name": "norm, training chunk", "op": "norm", "rows": 8192, "cols": 4096, "dtype": "bf16", "fmt": "e4m3", "backward": True},
        # an upstream gradient quantised for both of its products: by rows (input gradient), by columns (weight gradient)
        {"name": "quantise gradient both ways", "op": "quant", "rows": 8192, "cols": 14336, "dtype": "bf16", "fmt": "e5m2", "mode": "both"},
        # a weight of odd size in 128 x 128 tiles, as it is and transposed
        {"name": "quantise odd weight", "op": "quant", "rows": 1000, "cols": 2056, "dtype": "bf16", "fmt": "e4m3", "mode": "tiles"},
        # expert-sorted gradients, columns quantised per expert for the expert weight gradients
        {"name": "quantise expert columns", "op": "quant_grouped", "rows": 65536, "cols": 1536, "experts": 128, "dtype": "bf16", "fmt": "e5m2"},
        # one token through an up projection: bound by the weight's bytes
        {"name": "product, one token", "op": "matmul", "m": 1, "n": 14336, "k": 4096, "fmt": "e4m3", "b_tiles": True, "add": False, "out": "bf16"},
        # a short ragged batch, nothing a multiple of a tile
        {"name": "product, ragged batch", "op": "matmul", "m": 333, "n": 1000, "k": 2056, "fmt": "e4m3", "b_tiles": True, "add": False, "out": "fp16"},
        # the up projection of a training chunk
        {"name": "product, training chunk", "op": "matmul", "m": 8192, "n": 14336, "k": 4096, "fmt": "e4m3", "b_tiles": True, "add": False, "out": "bf16"},
        # the weight gradient of that projection, added to the gradient so far; both operands scaled along the tokens
        {"name": "product, weight gradient", "op": "matmul", "m": 14336, "n": 4096, "k": 8192, "fmt": "e5m2", "b_tiles": False, "add": True, "out": "bf16"},
        # four tokens through the up projection of a 128-expert block, top 8: most experts have no row
        {"name": "experts, four tokens", "op": "grouped", "tokens": 4, "top": 8, "experts": 128, "n": 1536, "k": 2048, "fmt": "e4m3", "gather": True},
        # the up projection of the benchmark's routed block: 8192 tokens, top 8 of 128, rows gathered from the unsorted tokens
        {"name": "experts, training chunk", "op": "grouped", "tokens": 8192, "top": 8, "experts": 128, "n": 1536, "k": 2048, "fmt": "e4m3", "gather": True},
        # its weight gradient, added to the gradient so far
        {"name": "experts, weight gradient", "op": "grouped_wgrad", "rows": 65536, "experts": 128, "m": 1536, "n": 2048, "fmt": "e5m2"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "quant", "quant", "quant_grouped", "matmul", "matmul", "matmul", "grouped", "grouped", "grouped_wgrad"])
    fmt = rng.choice(["e4m3", "e5m2"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "norm":
        cols = rng.choice([_log(rng, 64, 8192), 8 * _log(rng, 8, 1024), 128 * _log(rng, 1, 64)])
        return {"op": op, "rows": _log(rng, 1, min(16384, (1 << 25) // cols)), "cols": cols, "dtype": dtype, "fmt": fmt, "backward": rng.random() < 0.5}
    if op == "quant":
        cols = rng.choice([_log(rng, 1, 14336), 16 * _log(rng, 1, 896)])
        return {"op": op, "rows": _log(rng, 1, min(16384, (1 << 26) // cols)), "cols": cols, "dtype": dtype, "fmt": fmt, "mode": rng.choice(["rows", "both", "tiles"])}
    if op == "quant_grouped":
        return {"op": op, "rows": _log(rng, 1, 32768), "cols": 8 * _log(rng, 1, 256), "experts": _log(rng, 1, 256), "dtype": rng.choice(["bf16", "fp16"]), "fmt": fmt}
    if op == "matmul":
        n, k = _log(rng, 16, 14336), _log(rng, 16, 14336)
        m = _log(rng, 1, max(1, min(16384, (1 << 37) // (n * k))))
        return {"op": op, "m": m, "n": n, "k": k, "fmt": fmt, "b_tiles": rng.random() < 0.6, "add": rng.random() < 0.4, "out": rng.choice(["bf16", "bf16", "fp16"])}
    experts = _log(rng, 1, 128)
    n, k = 8 * _log(rng, 8, 256), 8 * _log(rng, 8, 256)
    if op == "grouped":
        top = min(experts, rng.choice([1, 2, 8]))
        return {"op": op, "tokens": _log(rng, 1, 8192 // top), "top": top, "experts": experts, "n": n, "k": k, "fmt": fmt, "gather": rng.random() < 0.5}
    return {"op": op, "rows": _log(rng, 1, 16384), "experts": experts, "m": n, "n": k, "fmt": fmt}


# ---------------------------------------------------------------- inputs

def _values(g, rows, cols, dtype, sigma=1.0):
    """Activations: normal, with a few channels an order of magnitude larger than the rest, as layers have them."""
    x = torch.randn(rows, cols, generator=g, device="cuda") * sigma
    loud = torch.rand(cols, generator=g, device="cuda") < 0.01
    return (x * torch.where(loud, 16.0, 1.0)).to(dtype)


def _counts(g, rows, experts, top=1):
    """Rows per expert of a routing with unequal popularity (the last experts may well get none)."""
    if top > 1:
        score = torch.rand(rows // top, experts, generator=g, device="cuda") + 0.25 * torch.rand(experts, generator=g, device="cuda")
        pick = score.topk(top, dim=1).indices.reshape(-1)
    else:
        pick = (torch.rand(rows, generator=g, device="cuda") ** 1.25 * experts).long().clamp_(max=experts - 1)
    order = torch.argsort(pick, stable=True)
    return torch.bincount(pick, minlength=experts).to(torch.int32), (order // top).to(torch.int32)


def _padded(t, mult):
    """A copy whose rows start at multiples of `mult` values in memory, as operands of the product have to."""
    ld = (t.shape[-1] + mult - 1) // mult * mult
    return F.pad(t.view(torch.uint8), (0, ld - t.shape[-1])).view(t.dtype)[..., : t.shape[-1]]


def _operand(x, fmt, tiles=False):
    """(values, scales) as the quantiser lays them out: scales have the block index of the contraction outermost in memory."""
    q, s = _quantise(x, fmt, 128 if tiles else 1)
    return _padded(q, 16), s.transpose(-1, -2).contiguous().transpose(-1, -2)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, state = case["op"], dict(case)
    fmt = FMT[case["fmt"]]
    if op == "norm":
        t = TYPE[case["dtype"]]
        r, c = case["rows"], case["cols"]
        state |= {"x": _values(g, r, c, t), "res": _values(g, r, c, t, 2.0), "w": (1 + 0.1 * torch.randn(c, generator=g, device="cuda")).to(t)}
        if case["backward"]:
            state |= {"dy": _values(g, r, c, t, 0.01), "dh": _values(g, r, c, t, 0.01)}
    elif op == "quant":
        state["x"] = _values(g, case["rows"], case["cols"], TYPE[case["dtype"]], 1e-3 if fmt is E5M2 else 1.0)
    elif op == "quant_grouped":
        state["x"] = _values(g, case["rows"], case["cols"], TYPE[case["dtype"]], 1e-3)
        state["counts"], _ = _counts(g, case["rows"], case["experts"])
    elif op == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        state["a"], state["sa"] = _operand(_values(g, m, k, torch.bfloat16, 1e-3 if fmt is E5M2 else 1.0), fmt)
        state["b"], state["sb"] = _operand(_values(g, n, k, torch.bfloat16, k ** -0.5), E4M3, case["b_tiles"])
        state["c"] = _values(g, m, n, TYPE[case["out"]], 1e-3 if fmt is E5M2 else 1.0) if case["add"] else None
    elif op == "grouped":
        e, n, k = case["experts"], case["n"], case["k"]
        state["counts"], source = _counts(g, case["tokens"] * case["top"], e, case["top"])
        x = _values(g, case["tokens"], k, torch.bfloat16, 1e-3 if fmt is E5M2 else 1.0)
        if not case["gather"]:
            x = x[source.long()]
        state["source"] = source if case["gather"] else None
        state["a"], state["sa"] = _operand(x, fmt)
        w = (torch.randn(e, n, k, generator=g, device="cuda") * k ** -0.5).to(torch.bfloat16)
        state["b"], state["sb"] = _operand(w, E4M3, True)
    else:
        e, m, n = case["experts"], case["m"], case["n"]
        state["counts"], _ = _counts(g, case["rows"], e)
        a = _columns(_values(g, case["rows"], m, torch.bfloat16, 1e-3 if fmt is E5M2 else 1.0), state["counts"], fmt)
        b = _columns(_values(g, case["rows"], n, torch.bfloat16), state["counts"], E4M3)
        state |= {"a": a[0], "sa": a[1].t().contiguous().t(), "b": b[0], "sb": b[1].t().contiguous().t()}
        state["c"] = (torch.randn(e, m, n, generator=g, device="cuda") * 0.01).to(torch.bfloat16)
    return state


# ---------------------------------------------------------------- plain forms

def _exponent(amax, fmt):
    """Smallest e with amax <= F 2^e; F is 0.875 of a power of two. A block of zeros has e = 0."""
    frac, p = torch.frexp(amax)
    e = p - (9 if fmt is E4M3 else 16) + (frac > 0.875).to(p.dtype)
    return torch.where(amax == 0, torch.zeros_like(e), e.clamp(-127, 127))


def _quantise(x, fmt, rows=1):
    """(values, scales) of x (..., R, C) in blocks of `rows` x 128."""
    x = x.float()
    r, c = x.shape[-2:]
    br, bc = -(-r // rows), -(-c // 128)
    v = F.pad(x, (0, bc * 128 - c, 0, br * rows - r)).reshape(x.shape[:-2] + (br, rows, bc, 128))
    mag = torch.where(torch.isfinite(v), v.abs(), torch.zeros_like(v))
    e = _exponent(mag.amax(dim=(-3, -1)), fmt)
    inverse = ((127 - e) << 23).view(torch.float32)  # 2^-e by its bits: the library's powers are an ulp off
    q = (v * inverse[..., :, None, :, None]).to(fmt)
    s = (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)
    q = q.view(torch.uint8).reshape(x.shape[:-2] + (br * rows, bc * 128))[..., :r, :c].contiguous().view(fmt)
    return q, s


def _places(counts):
    """Of every expert-sorted row: its place when each expert's rows start at a multiple of 128."""
    padded = (counts + 127) // 128 * 128
    expert = torch.repeat_interleave(torch.arange(counts.numel(), device=counts.device), counts)
    start, pstart = counts.cumsum(0) - counts, padded.cumsum(0) - padded
    return torch.arange(expert.numel(), device=counts.device) - start[expert] + pstart[expert], expert


def _capacity(rows, experts):
    return (rows + 127 * experts) // 128 * 128


def _columns(x, counts, fmt):
    """Expert-sorted x (R, C) -> transposed values (C, capacity) whose experts start at multiples of 128, and scales (C, capacity / 128)."""
    wide = torch.zeros(_capacity(x.shape[0], counts.numel()), x.shape[1], device=x.device, dtype=torch.float32)
    wide[_places(counts.long())[0]] = x.float()
    return _quantise(wide.t(), fmt)


def _values_of(q, s, rows):
    """What 8-bit values with scales (blocks of `rows` x 128) stand for, in 32 bits."""
    n, k = q.shape[-2:]
    scale = s.float()
    if rows > 1:
        scale = scale.repeat_interleave(rows, -2)[..., :n, :]
    return q.float() * scale.repeat_interleave(128, -1)[..., :k]


def _plain(st):
    op, fmt = st["op"], FMT[st["fmt"]]
    if op == "norm":
        t = TYPE[st["dtype"]]
        h = (st["x"].float() + st["res"].float()).to(t)
        hf, w = h.float(), st["w"].float()
        rstd = (hf.square().mean(1, keepdim=True) + EPS).rsqrt()
        q, s = _quantise(hf * rstd * w, fmt)
        out = {"q": q, "s": s, "h": h, "rstd": rstd}
        if st["backward"]:
            xh, dyw = hf * rstd, st["dy"].float() * w
            dx = st["dh"].float() + rstd * (dyw - xh * (dyw * xh).mean(1, keepdim=True))
            out |= {"dx": dx.to(t), "dw": (st["dy"].float() * xh).sum(0, dtype=torch.float64).float()}
        return out
    if op == "quant":
        rows = 128 if st["mode"] == "tiles" else 1
        q, s = _quantise(st["x"], fmt, rows)
        if st["mode"] == "rows":
            return {"q": q, "s": s}
        qt, s_t = _quantise(st["x"].t(), fmt, rows)
        return {"q": q, "s": s, "qt": qt, "st": s_t}
    if op == "quant_grouped":
        qt, s_t = _columns(st["x"], st["counts"], fmt)
        return {"qt": qt, "st": s_t}
    if op == "matmul":
        d = _values_of(st["a"], st["sa"], 1) @ _values_of(st["b"], st["sb"], 128 if st["b_tiles"] else 1).t()
        return (d if st["c"] is None else d + st["c"].float()).to(TYPE[st["out"]])
    counts = st["counts"].long()
    if op == "grouped":
        # every expert's rows padded to the longest, one batched product
        a = _values_of(st["a"], st["sa"], 1)
        if st["source"] is not None:
            a = a[st["source"].long()]
        rows, longest = a.shape[0], int(counts.max())
        expert = torch.repeat_interleave(torch.arange(counts.numel(), device=a.device), counts)
        at = torch.arange(rows, device=a.device) - (counts.cumsum(0) - counts)[expert]
        wide = torch.zeros(counts.numel(), longest, a.shape[1], device=a.device)
        wide[expert, at] = a
        w = _values_of(st["b"], st["sb"], 128).transpose(1, 2).contiguous()
        return torch.bmm(wide, w)[expert, at].to(torch.bfloat16)
    place, expert = _places(counts)
    a, b = _values_of(st["a"], st["sa"], 1)[:, place], _values_of(st["b"], st["sb"], 1)[:, place]
    longest = max(1, int(counts.max()))
    at = torch.arange(place.numel(), device=a.device) - (counts.cumsum(0) - counts)[expert]
    wa = torch.zeros(counts.numel(), longest, a.shape[0], device=a.device)
    wb = torch.zeros(counts.numel(), longest, b.shape[0], device=a.device)
    wa[expert, at], wb[expert, at] = a.t(), b.t()
    return (torch.bmm(wa.transpose(1, 2).contiguous(), wb) + st["c"].float()).to(torch.bfloat16)


# ---------------------------------------------------------------- the framework's calls

def _ours(st):
    from flextrain_amd import ops

    op, fmt = st["op"], FMT[st["fmt"]]
    if op == "norm":
        q, s, h, rstd = ops.flextrain_add_rmsnorm_fwd(st["x"], st["res"], st["w"], output_dtype=fmt, rms_norm_eps=EPS)
        out = {"q": q, "s": s, "h": h, "rstd": rstd}
        if st["backward"]:
            out["dx"], out["dw"] = ops.flextrain_add_rmsnorm_bwd(st["dy"], h, st["w"], rstd, dH=st["dh"])
        return out
    if op == "quant":
        if st["mode"] == "rows":
            q, s = ops.flextrain_fp8_quantize(st["x"], dtype=fmt)
            return {"q": q, "s": s}
        q, s, qt, s_t = ops.flextrain_fp8_quantize_both(st["x"], dtype=fmt, tiles=st["mode"] == "tiles")
        return {"q": q, "s": s, "qt": qt, "st": s_t}
    if op == "quant_grouped":
        qt, s_t = ops.flextrain_fp8_quantize_grouped_cols(st["x"], st["counts"], dtype=fmt)
        return {"qt": qt, "st": s_t}
    if op == "matmul":
        return ops.flextrain_fp8_matmul(st["a"], st["sa"], st["b"], st["sb"], C=st["c"], out_dtype=TYPE[st["out"]])
    if op == "grouped":
        return ops.flextrain_fp8_grouped_matmul(st["a"], st["sa"], st["b"], st["sb"], st["counts"], row_sources=st["source"])
    return ops.flextrain_fp8_grouped_wgrad(st["a"], st["sa"], st["b"], st["sb"], st["counts"], C=st["c"])


def run(state):
    return _ours(state) if own else _plain(state)


# ---------------------------------------------------------------- work

def work(case):
    op = case["op"]
    if op == "norm":
        n, z = case["rows"] * case["cols"], SIZE[case["dtype"]]
        b = n * (3 * z + 1) + n / 128 + 4 * case["rows"] + z * case["cols"]
        if case["backward"]:
            b += n * 4 * z + 4 * case["cols"]  # dy, h, dh read, dx written
        return {"bytes": b, "flops": n * (18 if case["backward"] else 8)}
    if op in ("quant", "quant_grouped"):
        n = case["rows"] * case["cols"]
        copies = 2 if case.get("mode", "rows") != "rows" else 1
        return {"bytes": n * (SIZE[case["dtype"]] + copies * (1 + 1 / 128)), "flops": 3 * copies * n}
    if op == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": (m + n) * k + m * n * 2 * (2 if case["add"] else 1), "flops": 2.0 * m * n * k}
    if op == "grouped":
        rows = case["tokens"] * case["top"]
        live = min(case["experts"], rows)
        return {"bytes": case["tokens"] * case["k"] + live * case["n"] * case["k"] + 2 * rows * case["n"], "flops": 2.0 * rows * case["n"] * case["k"]}
    m, n, rows = case["m"], case["n"], case["rows"]
    return {"bytes": rows * (m + n) + 4 * case["experts"] * m * n, "flops": 2.0 * rows * m * n}


# ---------------------------------------------------------------- exact values (64 bits, from the definitions)

def _two_to(e):
    """2^e in 64 bits, for whole numbers e held as such or as 64-bit floats (by its bits: the library's powers are an ulp off)."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _block_scales(x, fmt, rows, cols):
    """Exponents of the blocks of `rows` x `cols` of a 64-bit matrix, from the definition by logarithms and two comparisons."""
    top = 448.0 if fmt is E4M3 else 57344.0
    r, c = x.shape
    pad = torch.zeros(-(-r // rows) * rows, -(-c // cols) * cols, dtype=torch.float64, device=x.device)
    pad[:r, :c] = x.abs()
    amax = pad.unflatten(0, (-1, rows)).unflatten(2, (-1, cols)).amax(dim=(1, 3))
    e = torch.ceil(torch.log2(amax.clamp(min=1e-60) / top))
    e = torch.where(amax > top * _two_to(e), e + 1, e)
    e = torch.where(amax <= top * _two_to(e - 1), e - 1, e)
    return torch.where(amax == 0, torch.zeros_like(e), e.clamp(-127, 127))


def _spread(e, rows, cols, r, c):
    return _two_to(e).repeat_interleave(rows, 0).repeat_interleave(cols, 1)[:r, :c]


def _round8(v, fmt):
    """64-bit values of magnitude at most the type's largest, rounded to it (ties to even)."""
    bits, low = (3, -6) if fmt is E4M3 else (2, -14)
    step = _two_to(torch.frexp(v.abs().clamp(min=2.0 ** low))[1] - 1 - bits)
    return torch.round(v / step) * step


def _exact_quant(x, fmt, rows):
    e = _block_scales(x, fmt, rows, 128)
    return _round8(x / _spread(e, rows, 128, *x.shape), fmt), _two_to(e)


def _exact_values(q, s, rows):
    n, k = q.shape
    scale = _two_to(s.view(torch.uint8).to(torch.int64) - 127)
    row = torch.arange(n, device=q.device) // rows
    col = torch.arange(k, device=q.device) // 128
    return q.double() * scale[row][:, col]


def exact(case, seed):
    st = prepare(case, seed)
    op, fmt = st["op"], FMT[st["fmt"]]
    if op == "norm":
        h = (st["x"].double() + st["res"].double()).to(TYPE[st["dtype"]]).double()
        w = st["w"].double()
        rstd = 1 / torch.sqrt((h * h).sum(1, keepdim=True) / h.shape[1] + EPS)
        q, s = _exact_quant(h * rstd * w, fmt, 1)
        out = {"q": q, "s": s, "h": h, "rstd": rstd}
        if st["backward"]:
            dy = st["dy"].double()
            n = h * rstd
            inner = (dy * w * n).sum(1, keepdim=True) / h.shape[1]
            out |= {"dx": st["dh"].double() + rstd * (dy * w - n * inner), "dw": (dy * n).sum(0)}
        return out
    if op == "quant":
        x, rows = st["x"].double(), 128 if st["mode"] == "tiles" else 1
        q, s = _exact_quant(x, fmt, rows)
        if st["mode"] == "rows":
            return {"q": q, "s": s}
        qt, s_t = _exact_quant(x.t().contiguous(), fmt, rows)
        return {"q": q, "s": s, "qt": qt, "st": s_t}
    if op == "quant_grouped":
        x = st["x"].double()
        cap = _capacity(x.shape[0], case["experts"])
        wide = torch.zeros(x.shape[1], cap, dtype=torch.float64, device=x.device)
        at, to = 0, 0
        for c in st["counts"].tolist():
            wide[:, to:to + c] = x[at:at + c].t()
            at, to = at + c, to + -(-c // 128) * 128
        q, s = _exact_quant(wide, fmt, 1)
        return {"qt": q, "st": s}
    if op == "matmul":
        d = _exact_values(st["a"], st["sa"], 1) @ _exact_values(st["b"], st["sb"], 128 if st["b_tiles"] else 1).t()
        return d if st["c"] is None else d + st["c"].double()
    if op == "grouped":
        a = _exact_values(st["a"], st["sa"], 1)
        rows = sum(st["counts"].tolist())
        d = torch.empty(rows, case["n"], dtype=torch.float64, device=a.device)
        at = 0
        for i, c in enumerate(st["counts"].tolist()):
            if c:
                x = a[st["source"][at:at + c].long()] if st["source"] is not None else a[at:at + c]
                d[at:at + c] = x @ _exact_values(st["b"][i], st["sb"][i], 128).t()
                at += c
        return d
    a, b = _exact_values(st["a"], st["sa"], 1), _exact_values(st["b"], st["sb"], 1)
    g = st["c"].double()
    to = 0
    for i, c in enumerate(st["counts"].tolist()):
        g[i] += a[:, to:to + c] @ b[:, to:to + c].t()
        to += -(-c // 128) * 128
    return g
