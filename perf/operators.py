"""The 8-bit block-scaled products and the gradient-norm operators as measured workloads.

Five operators, each over listed cases and over ranges (``draw``):

``quantize``  a matrix as 8-bit floating point with one power-of-two scale per block of 128, row-wise, per 128 x 128 tile,
              transposed, or row-wise and transposed at once (what a training step keeps);
``matmul``    out = A B^T of two such matrices (feature maps against filters, weights against activations);
``linear``    a layer's forward pass from 16- / 32-bit activations: quantise, then multiply with the resident weight;
``backward``  the layer's two gradient products from the output gradient;
``clip``      the global norm over a list of gradient tensors and the clipped gradients.

``run`` computes the plain form (elementary torch operations in 32 bits) unless ``own`` is set, then it calls the
framework. ``exact`` states each operator once more in 64 bits.
"""
import math

import torch

own = False

FMT = {"e4m3": (torch.float8_e4m3fn, 8, 3, -6), "e5m2": (torch.float8_e5m2, 15, 2, -14)}   # dtype, max exponent (1.75 2^x), mantissa bits, min exponent
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}

# the 16 convolutions of VGG-19 (weight and bias): the parameter list of the feature stack this framework trains through
VGG_CONVS = ([(64, 3), (64, 64), (128, 64), (128, 128), (256, 128)] + [(256, 256)] * 3 + [(512, 256)] + [(512, 512)] * 7)


def listed():
    return [
        # one activation row against a resident weight: single-token serving, the latency end
        dict(name="linear_token", op="linear", m=1, n=4096, k=4096, x="bf16", out="bf16"),
        # a ragged handful of rows, an output width that ends inside a tile and a depth that ends inside a block
        dict(name="linear_rows", op="linear", m=37, n=8200, k=5001, x="bf16", out="bf16"),
        # relu3_1 of a 256 x 341 view (64 x 85 positions) against the 256 x (9 * 256) filters of conv3_2 as a plain product
        dict(name="matmul_features", op="matmul", m=5440, n=256, k=2304, b="rows", scale="e8m0", a_fmt="e4m3", out="f32"),
        # weights that come with arbitrary fp32 scales per tile (pre-quantised elsewhere)
        dict(name="matmul_f32_scales", op="matmul", m=4096, n=4096, k=4096, b="tiles", scale="f32", a_fmt="e4m3", out="f16"),
        # a large square product, the throughput end
        dict(name="matmul_large", op="matmul", m=8192, n=8192, k=8192, b="tiles", scale="e8m0", a_fmt="e4m3", out="bf16"),
        # a small training layer with nothing divisible by anything
        dict(name="backward_odd", op="backward", m=1029, n=517, k=1283, x="f32", g_fmt="e5m2"),
        # a layer of ordinary size, 4096 rows per step
        dict(name="backward_layer", op="backward", m=4096, n=4096, k=4096, x="bf16", g_fmt="e4m3"),
        # the activations of a decoding step
        dict(name="quantize_small", op="quantize", m=16, k=4096, x="f32", mode="rows", fmt="e4m3"),
        # a training step's activations: row-wise for the forward product, transposed for the weight gradient
        dict(name="quantize_both", op="quantize", m=8192, k=8192, x="bf16", mode="both", fmt="e4m3"),
        # the weights and biases of VGG-19's sixteen convolutions: 32 tensors from 64 to 2.4 M elements
        dict(name="clip_vgg", op="clip", kind="vgg", x="f32", out="f32", norm=2.0, max_norm=1.0),
        # gradients of a many-tensor model in bf16, the list handed over anew every step
        dict(name="clip_many", op="clip", kind="many", count=161, size=99991, x="bf16", out="bf16", norm=2.0, max_norm=0.5),
        # the four layers of a 4096 x 4096 hierarchical texture
        dict(name="clip_texture", op="clip", kind="texture", side=4096, x="f32", out="f32", norm=2.0, max_norm=1.0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quantize", "matmul", "linear", "backward", "clip"])
    x = rng.choice(["bf16", "bf16", "f32", "f16"])
    if op == "quantize":
        return dict(op=op, m=_log(rng, 1, 8192), k=_log(rng, 16, 8192), x=x,
                    mode=rng.choice(["rows", "tiles", "rows_t", "tiles_t", "both"]), fmt=rng.choice(["e4m3", "e5m2"]))
    if op == "matmul":
        return dict(op=op, m=_log(rng, 1, 8192), n=_log(rng, 16, 8192), k=_log(rng, 16, 8192), b=rng.choice(["rows", "tiles"]),
                    scale=rng.choice(["e8m0", "e8m0", "f32"]), a_fmt=rng.choice(["e4m3", "e4m3", "e5m2"]),
                    out=rng.choice(["f32", "bf16", "f16"]))
    if op == "linear":
        return dict(op=op, m=_log(rng, 1, 512), n=_log(rng, 64, 8192), k=_log(rng, 64, 8192), x=x, out=x)
    if op == "backward":
        return dict(op=op, m=_log(rng, 64, 4096), n=_log(rng, 64, 4096), k=_log(rng, 64, 4096), x=x, g_fmt=rng.choice(["e4m3", "e5m2"]))
    norm = rng.choice([2.0, 2.0, math.inf])
    if rng.random() < 0.4:
        return dict(op=op, kind="texture", side=rng.choice([256, 512, 1000, 1024, 2048, 4096]), x="f32", out="f32", norm=norm, max_norm=1.0)
    count = _log(rng, 1, 400)
    size = _log(rng, 1, min(4 << 20, (48 << 20) // count))
    return dict(op=op, kind="many", count=count, size=size, x=x, out=x, norm=norm, max_norm=0.5)


# ---- inputs ------------------------------------------------------------------------------------------------------
def _shapes(case):
    """Shapes of a ``clip`` case's tensors."""
    if case["kind"] == "vgg":
        return [s for co, ci in VGG_CONVS for s in ((co, ci, 3, 3), (co,))]
    if case["kind"] == "texture":
        return [(3, case["side"] >> i, case["side"] >> i) for i in range(4)]
    # sizes spread around the mean, as layers differ: 1/2, 1, 3/2 of it in turn, each odd by another remainder
    return [(max(1, case["size"] * (1 + i % 3) // 2 - i % 7),) for i in range(case["count"])]


def _inputs(case, seed):
    """What the operator reads, made from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")
    op = case["op"]
    if op == "clip":
        dt = TYPES[case["x"]]
        out = []
        for i, s in enumerate(_shapes(case)):
            # layers' gradients differ in size by orders of magnitude; a texture's data-term gradient is mostly small
            out.append((rand(*s) * 10.0 ** (-1 - i % 4)).to(dt))
        return {"grads": out}
    m, k = case["m"], case["k"]
    # activations: channels of very different size, as after a ReLU or a norm's gain
    x = rand(m, k) * torch.exp(1.5 * rand(1, k))
    if op == "quantize":
        return {"x": x.to(TYPES[case["x"]])}
    n = case["n"]
    w = rand(n, k) / math.sqrt(k)
    if op == "matmul":
        a, sa = _quantize(x, "rows", case["a_fmt"])
        b, sb = _quantize(w, case["b"], "e4m3")
        if case["scale"] == "f32":      # scales as foreign checkpoints have them: any fp32 value
            sa = _pow2(sa) * (1 + torch.rand(sa.shape, generator=g, device="cuda"))
            sb = _pow2(sb) * (1 + torch.rand(sb.shape, generator=g, device="cuda"))
        return {"a": a, "sa": sa, "b": b, "sb": sb}
    x = x.to(TYPES[case["x"]])
    w8, sw = _quantize(w, "tiles", "e4m3")
    if op == "linear":
        return {"x": x, "w8": w8, "sw": sw}
    # output gradients: a few rows carry most of it
    dy = (rand(m, n) * 1e-3 * torch.exp(rand(m, 1))).to(TYPES[case["x"]])
    return {"x": x, "w8": w8, "sw": sw, "dy": dy}


# ---- the plain form ----------------------------------------------------------------------------------------------
def _pow2(e):
    """2^e of whole exponents -127 ... 127 as fp32, from the bits (no transcendental function)."""
    e = e.to(torch.int32)
    return ((e.clamp(-126, 127) + 127) << 23).view(torch.float32) * torch.where(e < -126, 0.5, 1.0)


def _blocks(x, kind):
    """[R, C] padded with zeros to whole blocks, as [.., .., ..] with the block's elements on the last axis / axes."""
    r, c = x.shape
    x = torch.nn.functional.pad(x, (0, -c % 128, 0, (-r % 128) if kind == "tiles" else 0))
    if kind == "rows":
        return x.view(r, -1, 128)
    return x.view((r + 127) // 128, 128, -1, 128)


def _quantize(x, kind, fmt):
    """Codes [R, C padded to 128] (8-bit floats) and exponents of the blocks ([R or R / 128][C / 128], int32): the smallest
    power of two that brings the block's largest magnitude into the format's range."""
    dt, top, _, _ = FMT[fmt]
    r = x.shape[0]
    b = _blocks(x.float(), kind)
    amax = b.abs().amax(dim=-1) if kind == "rows" else b.abs().amax(dim=(1, 3))
    mant, ex = torch.frexp(amax)                      # amax = mant 2^ex, mant in [1/2, 1)
    e = ex - 1 - top + (2 * mant > 1.75).to(torch.int32)
    e = torch.where(amax > 0, e.clamp(-127, 127), torch.zeros_like(e))
    scaled = b * _pow2(-(e[:, :, None] if kind == "rows" else e[:, None, :, None]))
    codes = scaled.reshape(-1, b.shape[-1] * b.shape[-2])[:r].to(dt)
    return codes, e


def _dequantize(codes, e, kind, cols):
    """The values the codes stand for, fp32 [R, cols]; ``e``: exponents (whole) or fp32 scales."""
    s = e if e.is_floating_point() else _pow2(e)
    b = _blocks(codes.float(), kind)
    v = b * (s[:, :, None] if kind == "rows" else s[:, None, :, None])
    return v.reshape(-1, b.shape[-1] * b.shape[-2])[:codes.shape[0], :cols]


def _stored(e):
    """Exponents [R][KB] as the framework keeps them: bytes (exponent + 127), four blocks of a row together,
    [KB / 4][R][4], blocks behind the last one 127."""
    e = torch.nn.functional.pad(e + 127, (0, -e.shape[1] % 4), value=127)
    return e.view(e.shape[0], -1, 4).permute(1, 0, 2).to(torch.uint8).contiguous()


MODES = {"rows": [("rows", False)], "tiles": [("tiles", False)], "rows_t": [("rows", True)], "tiles_t": [("tiles", True)],
         "both": [("rows", False), ("rows", True)]}


def _plain(case, s):
    op = case["op"]
    if op == "quantize":
        out = {}
        for kind, t in MODES[case["mode"]]:
            codes, e = _quantize(s["x"].t() if t else s["x"], kind, case["fmt"])
            out["t" if t else "n"] = (codes, _stored(e))
        return out
    if op == "matmul":
        a = _dequantize(s["a"], s["sa"], "rows", case["k"])
        b = _dequantize(s["b"], s["sb"], case["b"], case["k"])
        return (a @ b.t()).to(TYPES[case["out"]])
    if op == "linear":
        x = _dequantize(*_quantize(s["x"], "rows", "e4m3"), "rows", case["k"])
        w = _dequantize(s["w8"], s["sw"], "tiles", case["k"])
        return (x @ w.t()).to(TYPES[case["out"]])
    if op == "backward":
        dy, fmt = s["dy"], case["g_fmt"]
        w = _dequantize(s["w8"], s["sw"], "tiles", case["k"])
        dx = _dequantize(*_quantize(dy, "rows", fmt), "rows", case["n"]) @ w
        xt = _dequantize(*_quantize(s["x"].t(), "rows", "e4m3"), "rows", case["m"])
        dyt = _dequantize(*_quantize(dy.t(), "rows", fmt), "rows", case["m"])
        return {"dx": dx.to(dy.dtype), "dw": dyt @ xt.t()}
    norm = _norm(s["grads"], case["norm"])
    coef = (case["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    grads = [(g.float() * coef.float()).to(g.dtype) for g in s["grads"]]
    return {"norm": norm.float(), "grads": torch.cat(grads) if case["kind"] == "many" else grads}


def _norm(grads, kind):
    if kind == math.inf:
        return torch.stack([g.abs().amax().double() for g in grads]).amax()
    return torch.stack([g.double().square().sum() for g in grads]).sum().sqrt()


# ---- the framework's calls -----------------------------------------------------------------------------------------
def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    op = case["op"]
    if op == "backward":
        # the forward pass left the transposed activations in 8 bits; the weight's transpose is made once per update
        s["xt8"], s["sxt"] = _quantize(s["x"].t(), "rows", "e4m3")
    if not own:
        return s
    from stylemesh_amd.runtime import fp8, gradclip
    if op == "matmul":
        keep = (lambda e: e.t().contiguous()) if case["scale"] == "f32" else _stored
        s["a8"] = fp8.Fp8Matrix(s["a"], keep(s["sa"]), case["k"], "rows")
        s["b8"] = fp8.Fp8Matrix(s["b"], keep(s["sb"]), case["k"], case["b"])
    if op in ("linear", "backward"):
        s["weight"] = fp8.Fp8Matrix(s["w8"], _stored(s["sw"]), case["k"], "tiles")
    if op == "backward":
        s["weight_t"] = s["weight"].transposed()
        s["x_t"] = fp8.Fp8Matrix(s["xt8"], _stored(s["sxt"]), case["m"], "rows")
    if op == "clip":
        if case["kind"] == "many":       # the clipped gradients go, tightly packed, into the bucket that travels to the other ranks
            s["bucket"] = torch.empty(sum(g.numel() for g in s["grads"]), dtype=TYPES[case["out"]], device="cuda")
            s["out"] = list(s["bucket"].split([g.numel() for g in s["grads"]]))
        else:                            # gradient buffers that stay where they are: the program keeps the plan
            s["out"] = [torch.empty_like(g) for g in s["grads"]]
            s["plan"] = gradclip.GradClip(s["grads"], out=s["out"])
    return s


def run(state):
    return _own(state["case"], state) if own else _plain(state["case"], state)


def _own(case, s):
    from stylemesh_amd.runtime import fp8, gradclip
    op = case["op"]
    if op == "quantize":
        if case["mode"] == "both":
            n, t = fp8.fp8_quantize_both(s["x"], fmt=case["fmt"])
            return {"n": (n.data, n.scale), "t": (t.data, t.scale)}
        kind, t = MODES[case["mode"]][0]
        q = fp8.fp8_quantize(s["x"], block=kind, fmt=case["fmt"], transpose=t)
        return {"t" if t else "n": (q.data, q.scale)}
    if op == "matmul":
        return fp8.matmul_fp8(s["a8"], s["b8"], out_dtype=TYPES[case["out"]])
    if op == "linear":
        return fp8.linear_fp8_fwd(s["x"], s["weight"], out_dtype=TYPES[case["out"]])
    if op == "backward":
        dx, dw = fp8.linear_fp8_bwd(s["dy"], s["x_t"], s["weight_t"], fmt=case["g_fmt"])
        return {"dx": dx, "dw": dw}
    if "plan" in s:
        return {"norm": s["plan"].clip(case["max_norm"], norm_type=case["norm"]), "grads": s["out"]}
    norm = gradclip.clip_grad_norm(s["grads"], case["max_norm"], norm_type=case["norm"], out=s["out"])
    return {"norm": norm, "grads": s["bucket"]}


def work(case):
    op = case["op"]
    size = lambda t: TYPES[t].itemsize
    if op == "clip":
        n = sum(math.prod(s) for s in _shapes(case))
        return {"bytes": n * (size(case["x"]) + size(case["out"])) + 4, "flops": 3 * n}
    m, k = case["m"], case["k"]
    kb = -(-k // 128)
    if op == "quantize":
        copies = len(MODES[case["mode"]])
        return {"bytes": m * k * (size(case["x"]) + copies), "flops": 2 * copies * m * k}
    n = case["n"]
    if op == "matmul":
        sc = 4 if case["scale"] == "f32" else 1
        scales = sc * kb * (m + (n if case["b"] == "rows" else -(-n // 128)))
        return {"bytes": m * k + n * k + scales + m * n * size(case["out"]), "flops": 2 * m * n * k}
    if op == "linear":
        return {"bytes": m * k * size(case["x"]) + n * k + m * n * size(case["out"]), "flops": 2 * m * n * k}
    return {"bytes": m * n * size(case["x"]) + m * k + n * k + m * k * size(case["x"]) + 4 * n * k, "flops": 4 * m * n * k}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------
def _exp2(e):
    """2^e of whole numbers (held in double), from the bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _round64(v, e, fmt):
    """v / 2^e on the format's grid, ties to even, in double arithmetic: the step at magnitude 2^q is 2^(q - mantissa bits)."""
    _, _, bits, low = FMT[fmt]
    y = v * _exp2(-e)
    q = torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -60)))
    q = torch.where(_exp2(q + 1) <= y.abs(), q + 1, torch.where(_exp2(q) > y.abs(), q - 1, q)).clamp_min(low)
    step = _exp2(q - bits)
    return torch.round(y / step) * step


def _quant64(x, kind, fmt):
    """(grid values, exponents) blockwise: loops over the blocks of a row / tile, no reshaping shared with the plain form."""
    x = x.double()
    r, c = x.shape
    limit = 1.75 * 2.0 ** FMT[fmt][1]
    cb = -(-c // 128)
    rb = r if kind == "rows" else -(-r // 128)
    exps = torch.zeros(rb, cb, dtype=torch.float64, device=x.device)
    vals = torch.zeros(r, cb * 128, dtype=torch.float64, device=x.device)
    for j in range(cb):
        part = x[:, 128 * j:128 * (j + 1)]
        top = part.abs().amax(dim=1)
        if kind == "tiles":
            top = torch.stack([top[128 * i:128 * (i + 1)].amax() for i in range(rb)])
        e = torch.ceil(torch.log2(top.clamp_min(2.0 ** -140) / limit))
        e = torch.where(limit * _exp2(e - 1) >= top, e - 1, torch.where(limit * _exp2(e) < top, e + 1, e))
        e = torch.where(top > 0, e.clamp(-127, 127), torch.zeros_like(e))
        exps[:, j] = e
        rows = e if kind == "rows" else e.repeat_interleave(128)[:r]
        vals[:, 128 * j:128 * j + part.shape[1]] = _round64(part, rows[:, None], fmt)
    return vals, exps


def _value64(vals, s, kind, cols):
    """grid values times the blocks' scales (exact in double for powers of two)."""
    f = s.repeat_interleave(128, dim=1)
    if kind == "tiles":
        f = f.repeat_interleave(128, dim=0)[:vals.shape[0]]
    return (vals * f[:, :vals.shape[1]])[:, :cols]


def _bytes64(exps):
    r, cb = exps.shape
    out = torch.full((-(-cb // 4), r, 4), 127, dtype=torch.uint8, device=exps.device)
    for j in range(cb):
        out[j // 4, :, j % 4] = (exps[:, j] + 127).to(torch.uint8)
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    scale64 = lambda e: e.double() if e.is_floating_point() else _exp2(e.double())
    if op == "quantize":
        out = {}
        for kind, t in MODES[case["mode"]]:
            vals, e = _quant64(s["x"].t() if t else s["x"], kind, case["fmt"])
            out["t" if t else "n"] = (vals, _bytes64(e))
        return out
    if op == "matmul":
        a = _value64(s["a"].double(), scale64(s["sa"]), "rows", case["k"])
        b = _value64(s["b"].double(), scale64(s["sb"]), case["b"], case["k"])
        return torch.mm(a, b.t())
    if op in ("linear", "backward"):
        q = lambda t, fmt, cols: (lambda v, e: _value64(v, _exp2(e), "rows", cols))(*_quant64(t, "rows", fmt))
        w = _value64(s["w8"].double(), scale64(s["sw"]), "tiles", case["k"])
        if op == "linear":
            return torch.mm(q(s["x"], "e4m3", case["k"]), w.t())
        dx = torch.mm(q(s["dy"], case["g_fmt"], case["n"]), w)
        dw = torch.mm(q(s["dy"].t(), case["g_fmt"], case["m"]), q(s["x"].t(), "e4m3", case["m"]).t())
        return {"dx": dx, "dw": dw}
    total = torch.zeros((), dtype=torch.float64, device="cuda")
    for g in s["grads"]:
        v = g.double()
        total = torch.maximum(total, v.abs().max()) if case["norm"] == math.inf else total + (v * v).sum()
    norm = total if case["norm"] == math.inf else torch.sqrt(total)
    coef = torch.clamp(case["max_norm"] / (norm + 1e-6), max=1.0)
    grads = [g.double() * coef for g in s["grads"]]
    return {"norm": norm, "grads": torch.cat(grads) if case["kind"] == "many" else grads}
