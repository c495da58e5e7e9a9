"""The operators of a deep residual model beside the graph layers, as cases that can be timed.

  norm      h = x + residual; y = h / rms(h) * weight: forward (y in 32, 16 or 8 bits), or forward and backward
  ffn       y = (act(x Wg) * (x Wu)) Wo: forward, forward and backward, or forward with the first product in 8 bits
  adamw     one step over every tensor of a model, moments in 32 or in 8 bits

run() computes them in plain torch operations in 32 bits, or (``own``) through graphcuda_b200.  Widths and row counts are
those of the graph configurations (synth.py: 2708, 169,343 vertices; widths 64 to 256) and, beyond them, powers of two.
"""
import math

import torch

own = False
DEV = "cuda"
EPS = 1e-6
BLOCK = 256  # elements that share a scale of an 8-bit moment
LR, BETAS, ADAM_EPS, DECAY = 1e-3, (0.9, 0.999), 1e-8, 0.01
FIRST_STEP = 1000
SEED = 7
BF16, F32, F8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
TYPES = {"bf16": BF16, "fp32": F32}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # One vertex asked for by a server: the norm in front of its feed-forward block.  All latency.
        dict(name="norm_row", op="norm", rows=1, width=256, x="bf16", stream="bf16", out="bf16", mode="forward"),
        # A training step at citation-graph size: the feed-forward block's bf16 output joins an fp32 stream.
        dict(name="norm_train_arxiv", op="norm", rows=169_343, width=256, x="bf16", stream="fp32", out="bf16", mode="train"),
        # Raw features of the small citation graph: an odd width, everything in fp32.
        dict(name="norm_train_odd", op="norm", rows=2708, width=1433, x="fp32", stream="fp32", out="fp32", mode="train"),
        # Serving a wide model: the operand of an 8-bit product.
        dict(name="norm_fp8_wide", op="norm", rows=8192, width=4096, x="bf16", stream="bf16", out="fp8", mode="forward"),
        # One row through a wide block: every weight is read once.
        dict(name="ffn_row", op="ffn", rows=1, width=2048, hidden=8192, out=2048, act="silu", mode="forward"),
        # A training step of the block at citation-graph size: short products, much to read and write.
        dict(name="ffn_train_arxiv", op="ffn", rows=169_343, width=256, hidden=1024, out=256, act="silu", mode="train"),
        # A wide block: long products.
        dict(name="ffn_train_wide", op="ffn", rows=8192, width=2048, hidden=8192, out=2048, act="gelu", mode="train"),
        # Odd widths on a small graph: class counts and feature counts as they fall.
        dict(name="ffn_train_odd", op="ffn", rows=2708, width=100, hidden=267, out=47, act="silu", mode="train"),
        # Evaluation of every vertex with the first product in 8 bits.
        dict(name="ffn_fp8_arxiv", op="ffn", rows=169_343, width=256, hidden=1024, out=256, act="silu", mode="fp8"),
        # A small model: ten tensors, all latency.
        dict(name="adamw_small", op="adamw", layers=2, width=64, hidden=171, bits=32, params="fp32"),
        # A deep narrow model: 480 tensors, most of them small.
        dict(name="adamw_many", op="adamw", layers=96, width=256, hidden=1024, bits=32, params="fp32"),
        # A wide model in mixed precision: bf16 parameters with fp32 masters, moments in 8 bits.
        dict(name="adamw_wide_8bit", op="adamw", layers=4, width=2048, hidden=8192, bits=8, params="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """Half of them as users choose widths (multiples of 8), half as they fall."""
    n = _log(rng, lo, hi)
    return max(8, n // 8 * 8) if rng.random() < 0.5 else n


def draw(rng):
    op = rng.choice(("norm", "ffn", "ffn", "adamw"))
    if op == "norm":
        width = _size(rng, 16, 8192)
        rows = _log(rng, 1, min(400_000, 40_000_000 // width))
        out = rng.choice(("bf16", "fp32", "fp8"))
        x, stream = rng.choice((("bf16", "bf16"), ("bf16", "fp32"), ("fp32", "fp32")))
        return dict(op=op, rows=rows, width=width, x=x, stream=stream, out=out,
                    mode="forward" if out == "fp8" else rng.choice(("forward", "train", "train")))
    if op == "adamw":
        while True:
            case = dict(op=op, layers=_log(rng, 1, 100), width=_size(rng, 16, 2048), hidden=_size(rng, 16, 8192),
                        bits=rng.choice((8, 32)), params=rng.choice(("fp32", "bf16")))
            if sum(n for n in _sizes(case)) <= 2.1e8:
                return case
    while True:
        mode = rng.choice(("forward", "train", "train", "fp8"))
        case = dict(op=op, rows=_log(rng, 1, 200_000), width=_size(rng, 16, 4096), hidden=_size(rng, 16, 8192),
                    out=_size(rng, 16, 4096), act=rng.choice(("silu", "gelu", "relu")), mode=mode)
        if work(case)["flops"] <= 2.4e12 and work(case)["bytes"] <= 2e9 and case["rows"] * case["hidden"] <= 2e8:
            return case


def _sizes(case):
    """Tensor sizes of a model of `layers` blocks: graph transform, two norms, feed-forward block."""
    d, h = case["width"], case["hidden"]
    return [d * d, d, d, d * 2 * h, h * d] * case["layers"]


def work(case):
    op = case["op"]
    if op == "norm":
        n, d = case["rows"] * case["width"], case["width"]
        size = {"bf16": 2, "fp32": 4, "fp8": 1}
        x, s, y = size[case["x"]], size[case["stream"]], size[case["out"]]
        b = n * (x + 2 * s + y) + 4 * d + (4 * case["rows"] if case["out"] == "fp8" else 0)
        if case["mode"] == "train":  # gradients of y and of the stream in, of x and of the residual out
            b += n * (y + s + x + (s if s != x else 0)) + 4 * d
        return {"bytes": b, "flops": n * (17 if case["mode"] == "train" else 6)}
    if op == "ffn":
        m, d, h, o = case["rows"], case["width"], case["hidden"], case["out"]
        weights = d * 2 * h + h * o
        flops = 2 * m * weights
        if case["mode"] == "fp8":
            return {"bytes": m * (d + 4 + 2 * o) + d * 2 * h + 8 * h + 2 * h * o, "flops": flops}
        if case["mode"] == "train":
            return {"bytes": 2 * (2 * m * d + 2 * m * o + 2 * weights), "flops": 3 * flops}
        return {"bytes": 2 * (m * d + m * o + weights), "flops": flops}
    n = sum(_sizes(case))
    p = 12  # parameter in and out, gradient in; or master in and out, gradient and parameter of 16 bits
    if case["bits"] == 32:
        return {"bytes": n * (p + 16), "flops": 14 * n}
    # codes in and out, and the moments as values, which the pass returns
    return {"bytes": n * (p + 4 + 8) + n // BLOCK * 16, "flops": 60 * n}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, generator=g, device=DEV)  # noqa: E731
    op = case["op"]
    if op == "norm":
        shape = case["rows"], case["width"]
        tx, ts = TYPES[case["x"]], TYPES[case["stream"]]
        s = dict(case=case, x=randn(*shape).to(tx), residual=(2 * randn(*shape)).to(ts), weight=1 + 0.1 * randn(shape[1]))
        if case["mode"] == "train":
            s["dy"], s["dstream"] = randn(*shape).to(TYPES[case["out"]]), randn(*shape).to(ts)
        return s
    if op == "ffn":
        m, d, h, o = case["rows"], case["width"], case["hidden"], case["out"]
        s = dict(case=case, w_in=(randn(d, 2 * h) / math.sqrt(d)).to(BF16), w_out=(randn(h, o) / math.sqrt(h)).to(BF16))
        x = randn(m, d)
        if case["mode"] == "fp8":  # a row of x and a column of w_in have a scale each; w_in laid out along its inputs
            top = x.abs().amax(1, keepdim=True)
            s["x_scale"] = (top / 448.0).squeeze(1)
            s["x8"] = (x / s["x_scale"][:, None]).to(F8)
            w = s.pop("w_in").float()
            s["w_scale"] = w.abs().amax(0) / 448.0
            s["w8"] = (w / s["w_scale"]).t().contiguous().to(F8)
        else:
            s["x"] = x.to(BF16)
        if case["mode"] == "train":
            s["dy"] = randn(m, o).to(BF16)
        return s
    # every tensor a view of one buffer per kind, at a multiple of BLOCK elements
    sizes = _sizes(case)
    blocks = [-(-n // BLOCK) for n in sizes]
    starts = [0]
    for b in blocks:
        starts.append(starts[-1] + b)
    total = starts[-1]
    tensor = torch.repeat_interleave(torch.arange(len(sizes), device=DEV), torch.tensor(blocks, device=DEV))
    within = torch.arange(total, device=DEV) - torch.tensor(starts, device=DEV)[tensor]
    live = within[:, None] * BLOCK + torch.arange(BLOCK, device=DEV) < torch.tensor(sizes, device=DEV)[tensor][:, None]
    # gradients differ in size by tensor, moments are those of a run in progress
    scale = torch.exp(randn(len(sizes)) - 7.0)[tensor][:, None] * live
    spread = torch.exp(0.7 * randn(total, BLOCK)) * scale
    grad = spread * randn(total, BLOCK)
    s = dict(case=case, tensor=tensor, within=within, live=live, step=FIRST_STEP)
    s["master"] = (0.02 * randn(total, BLOCK)) * live
    m, v = 0.3 * spread * randn(total, BLOCK), spread.square()
    if case["params"] == "bf16":
        s["p"], grad = s["master"].to(BF16), grad.to(BF16)
    s["g"] = grad
    if case["bits"] == 8:
        s["m"], s["m_scale"], s["v"], s["v_scale"] = _pack(m, v, torch.full_like(m, 0.5), torch.full_like(v, 0.5), live)
        s["m_values"], s["v_values"] = torch.zeros_like(m), torch.zeros_like(v)
    else:
        s["m"], s["v"] = m, v
    # the lists of tensors that an optimizer keeps
    s["device_step"] = torch.tensor([FIRST_STEP, 0], dtype=torch.int64, device=DEV)
    views = lambda key: [s[key].view(-1)[starts[i] * BLOCK:starts[i] * BLOCK + n] for i, n in enumerate(sizes)]  # noqa: E731
    s["views"] = {k: views(k) for k in ("p", "master", "g", "m", "v", "m_values", "v_values") if k in s}
    for k in ("m_scale", "v_scale"):
        if k in s:
            s["views"][k] = [s[k][starts[i]:starts[i + 1]] for i in range(len(sizes))]
    return s


# ------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    return {"norm": _norm, "ffn": _ffn, "adamw": _adamw}[case["op"]](state, case)


def _norm(s, case):
    x, r, w = s["x"], s["residual"], s["weight"]
    out = F8 if case["out"] == "fp8" else TYPES[case["out"]]
    if own:
        import graphcuda_b200 as gc
        if case["out"] == "fp8":
            y, scale, stream = gc.rms_norm_fp8(x, w, residual=r, eps=EPS)
            return {"y": y, "scale": scale, "stream": stream}
        if case["mode"] == "forward":
            with torch.no_grad():
                y, stream = gc.rms_norm(x, w, residual=r, eps=EPS, out_dtype=out)
            return {"y": y, "stream": stream}
        x, r, w = (t.detach().requires_grad_() for t in (x, r, w))
        y, stream = gc.rms_norm(x, w, residual=r, eps=EPS, out_dtype=out)
        dx, dr, dw = torch.autograd.grad((y, stream), (x, r, w), (s["dy"], s["dstream"]))
        return {"y": y, "stream": stream, "dx": dx, "dresidual": dr, "dweight": dw}
    h = x.float() + r.float()
    rstd = torch.rsqrt(h.square().mean(1, keepdim=True) + EPS)
    hat = h * rstd
    y = hat * w
    if case["out"] == "fp8":
        scale = y.abs().amax(1, keepdim=True) / 448.0
        return {"y": (y / scale).to(F8), "scale": scale.squeeze(1), "stream": h.to(r.dtype)}
    got = {"y": y.to(out), "stream": h.to(r.dtype)}
    if case["mode"] == "train":
        dy = s["dy"].float()
        dw_y = dy * w
        dh = rstd * (dw_y - hat * (dw_y * hat).mean(1, keepdim=True)) + s["dstream"].float()
        got.update(dx=dh.to(x.dtype), dresidual=dh.to(r.dtype), dweight=(dy * hat).sum(0))
    return got


def _act(name, g):
    """(act(g), its derivative)."""
    if name == "silu":
        sig = torch.sigmoid(g)
        return g * sig, sig * (1 + g * (1 - sig))
    if name == "gelu":
        cdf = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))
    return g * (g > 0), (g > 0).to(g.dtype)


def _ffn(s, case):
    if own:
        import graphcuda_b200 as gc
        if case["mode"] == "fp8":
            return gc.gated_ffn_fp8(s["x8"], s["x_scale"], s["w8"], s["w_scale"], s["w_out"], activation=case["act"])
        if case["mode"] == "forward":
            with torch.no_grad():
                return gc.gated_ffn(s["x"], s["w_in"], s["w_out"], activation=case["act"])
        x, w_in, w_out = (s[k].detach().requires_grad_() for k in ("x", "w_in", "w_out"))
        y = gc.gated_ffn(x, w_in, w_out, activation=case["act"])
        dx, dw_in, dw_out = torch.autograd.grad(y, (x, w_in, w_out), s["dy"])
        return {"y": y, "dx": dx, "dw_in": dw_in, "dw_out": dw_out}
    h = case["hidden"]
    w_out = s["w_out"].float()
    if case["mode"] == "fp8":
        gu = (s["x8"].float() @ s["w8"].float().t()) * s["x_scale"][:, None] * s["w_scale"]
    else:
        x, w_in = s["x"].float(), s["w_in"].float()
        gu = x @ w_in
    act, slope = _act(case["act"], gu[:, :h])
    a = act * gu[:, h:]
    y = (a @ w_out).to(BF16)
    if case["mode"] != "train":
        return y
    dy = s["dy"].float()
    da = dy @ w_out.t()
    dgu = torch.cat((da * gu[:, h:] * slope, da * act), 1)
    return {"y": y, "dx": (dgu @ w_in.t()).to(BF16), "dw_in": (x.t() @ dgu).to(BF16), "dw_out": (a.t() @ dy).to(BF16)}


# ---- AdamW: moments of 8 bits
# A block of 256 elements has an fp32 scale per moment.  exp_avg: e4m3 (sign, 4 bits of exponent, 3 of mantissa, largest
# value 448).  exp_avg_sq: the upper byte of a positive fp16 number without its sign bit (5 and 3 bits, largest value
# 61440), never below the smallest code where the block is not zero.  Values are rounded up or down at random, in
# proportion: an average that moves by 0.1 % a step would stand still under rounding to nearest.
def _round(t, u, mantissa, lowest, top):
    """t >= 0 rounded to `mantissa` bits (to a fixed grid below 2^lowest), up with the probability that u < fraction."""
    e = (t.view(torch.int32) >> 23) - 127
    ulp = ((e.clamp(min=lowest) - mantissa + 127) << 23).view(torch.float32)
    return (torch.floor(t / ulp + u) * ulp).clamp(max=top)


def _scaled(x, top):
    scale = x.abs().amax(1, keepdim=True) * (1.0 / top)
    scale = torch.where(scale < 2.0 ** -126, torch.zeros_like(scale), scale)
    return x * torch.where(scale > 0, scale.reciprocal(), torch.zeros_like(scale)), scale


def _pack(m, v, um, uv, live):
    t, ms = _scaled(m, 448.0)
    mq = torch.copysign(_round(t.abs(), um, 3, -6, 448.0), t).to(F8)
    t, vs = _scaled(v, 61440.0)
    vq = _round(t, uv, 3, -14, 61440.0).clamp(min=2.0 ** -17) * ((vs > 0) & live)
    vq = (vq.to(torch.float16).view(torch.int16) >> 7).to(torch.uint8)
    return mq.view(torch.uint8), ms.squeeze(1), vq, vs.squeeze(1)


def _unpack(m, ms, v, vs):
    return m.view(F8).float() * ms[:, None], (v.to(torch.int16) << 7).view(torch.float16).float() * vs[:, None]


def _mix(x):
    """The finalizer of MurmurHash3 on 32-bit words held in int64."""
    x = x & 0xFFFFFFFF
    x = ((x ^ (x >> 16)) * 0x85EBCA6B) & 0xFFFFFFFF
    x = ((x ^ (x >> 13)) * 0xC2B2AE35) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _uniform(s, step):
    """Two numbers in [0, 1) of 16 bits for every element, by (seed, step, tensor, element)."""
    key = _mix(_mix(torch.tensor(SEED, device=DEV) + step * 0x9E3779B9) + s["tensor"])
    r = _mix(key[:, None] + s["within"][:, None] * BLOCK + torch.arange(BLOCK, device=DEV))
    return (r & 0xFFFF).float() * 2.0 ** -16, (r >> 16).float() * 2.0 ** -16


def _adamw(s, case):
    lists = s["views"]
    mixed = case["params"] == "bf16"
    hyper = dict(lr=LR, betas=BETAS, eps=ADAM_EPS, weight_decay=DECAY)
    if own:
        import graphcuda_b200 as gc
        scales = (lists["m_scale"], lists["v_scale"]) if case["bits"] == 8 else None
        gc.adamw_step(lists["p" if mixed else "master"], lists["g"], lists["m"], lists["v"], s["device_step"],
                      masters=lists["master"] if mixed else None, scales=scales, seed=SEED, **hyper)
        if case["bits"] == 8:
            gc.adamw_moments(lists["m"], lists["v"], scales, out=(lists["m_values"], lists["v_values"]))
    else:
        s["step"] += 1
        b1, b2 = BETAS
        g = s["g"].float()
        m, v = (s["m"], s["v"]) if case["bits"] == 32 else _unpack(s["m"], s["m_scale"], s["v"], s["v_scale"])
        m = m * b1 + g * (1 - b1)
        v = v * b2 + g * g * (1 - b2)
        rest = 1 - b2 ** s["step"]
        update = m / (v.sqrt() / math.sqrt(rest) + ADAM_EPS) * (LR / (1 - b1 ** s["step"]))
        s["master"].mul_(1 - LR * DECAY).sub_(update)
        if mixed:
            s["p"].copy_(s["master"])
        if case["bits"] == 32:
            s["m"].copy_(m)
            s["v"].copy_(v)
        else:
            s["m"][:], s["m_scale"][:], s["v"][:], s["v_scale"][:] = _pack(m, v, *_uniform(s, s["step"]), s["live"])
            s["m_values"][:], s["v_values"][:] = _unpack(s["m"], s["m_scale"], s["v"], s["v_scale"])
    got = {"params": s["master"]}
    if mixed:
        got["params16"] = s["p"]
    kind = "_values" if case["bits"] == 8 else ""
    got["exp_avg"], got["exp_avg_sq"] = s["m" + kind], s["v" + kind]
    return got


# ------------------------------------------------------------------ the same in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    wide = lambda k: s[k].to(torch.float64)  # noqa: E731
    if case["op"] == "norm":
        h, w = wide("x") + wide("residual"), wide("weight")
        size = (h * h).sum(1, keepdim=True) / case["width"] + EPS
        y = h * w / size.sqrt()
        if case["out"] == "fp8":
            top = y.abs().max(1, keepdim=True).values / 448.0
            return {"y": (y / top).float().to(F8).double(), "scale": top[:, 0], "stream": h}
        if case["mode"] == "forward":
            return {"y": y, "stream": h}
        dy = wide("dy")
        # d/dh of sum(dy w h / sqrt(size)): the direct term, and the one through size = sum(h^2) / width + eps
        direct = dy * w / size.sqrt()
        through = h * (dy * w * h).sum(1, keepdim=True) / (case["width"] * size * size.sqrt())
        dh = direct - through + wide("dstream")
        return {"y": y, "stream": h, "dx": dh, "dresidual": dh, "dweight": (dy * h / size.sqrt()).sum(0)}
    if case["op"] == "ffn":
        n, w_out = case["hidden"], wide("w_out")
        if case["mode"] == "fp8":
            x, w_in = wide("x8") * wide("x_scale")[:, None], (wide("w8") * wide("w_scale")[:, None]).t()
        else:
            x, w_in = wide("x"), wide("w_in")
        gate, up = x @ w_in[:, :n], x @ w_in[:, n:]
        if case["act"] == "silu":
            e = torch.exp(-gate.abs())
            sig = torch.where(gate >= 0, 1 / (1 + e), e / (1 + e))
            act, slope = gate * sig, sig + gate * sig * (1 - sig)
        elif case["act"] == "gelu":
            half = torch.special.erfc(-gate / math.sqrt(2)) / 2
            act, slope = gate * half, half + gate * torch.exp(-gate * gate / 2) / math.sqrt(2 * math.pi)
        else:
            act, slope = gate.clamp(min=0), torch.heaviside(gate, torch.zeros_like(gate))
        hidden = act * up
        y = hidden @ w_out
        if case["mode"] != "train":
            return y
        dy = wide("dy")
        back = dy @ w_out.t()
        d_gate, d_up = back * up * slope, back * act
        dw_in = torch.cat((x.t() @ d_gate, x.t() @ d_up), 1)
        return {"y": y, "dx": d_gate @ w_in[:, :n].t() + d_up @ w_in[:, n:].t(), "dw_in": dw_in, "dw_out": hidden.t() @ dy}
    # AdamW.  The moments of 8 bits are compared as the values they stand for, rounded by the same random numbers.
    b1, b2 = BETAS
    t = FIRST_STEP + 1
    g, p = wide("g"), wide("master")
    if case["bits"] == 8:
        m0, v0 = s["m"].view(F8).double() * wide("m_scale")[:, None], _half(s["v"]) * wide("v_scale")[:, None]
    else:
        m0, v0 = wide("m"), wide("v")
    m, v = b1 * m0 + (1 - b1) * g, b2 * v0 + (1 - b2) * g ** 2
    p = p - LR * DECAY * p - LR * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + ADAM_EPS)
    got = {"params": p}
    if case["params"] == "bf16":
        got["params16"] = p
    if case["bits"] == 8:
        um, uv = (u.double() for u in _uniform(s, t))
        top = m.abs().amax(1, keepdim=True) / 448
        m = m.sign() * _grid(m.abs() / top.clamp(min=1e-300), um, -6).clamp(max=448.0) * top
        top = v.amax(1, keepdim=True) / 61440
        v = _grid(v / top.clamp(min=1e-300), uv, -14).clamp(min=2.0 ** -17, max=61440.0) * top * s["live"]
    got["exp_avg"], got["exp_avg_sq"] = m, v
    return got


def _half(code):
    """The value of an 8-bit second moment: 5 bits of exponent, 3 of mantissa."""
    e, f = (code >> 3).double(), (code & 7).double()
    return torch.where(e > 0, (1 + f / 8) * torch.exp2(e - 15), f / 8 * 2.0 ** -14)


def _grid(t, u, lowest):
    """t >= 0 to 3 bits of mantissa, up where u is large enough."""
    step = torch.exp2((torch.frexp(t).exponent - 1).clamp(min=lowest).double() - 3)
    return torch.floor(t / step + u) * step
