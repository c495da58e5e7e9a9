"""Operators that train a model with weights per kind of row, train a small model from a large one's answers, and serve it
from weights of 4 bits, as cases that can be timed.

  distill   loss of a student's logits against a teacher's top logits: its value, or its value and the logits' gradient
  grouped   rows sorted by group, each group times its own weights: forward, or forward and backward
  linear4   rows times weights of 4 bits with a scale (and a zero point) per group of inputs
  block4    gated feed-forward block whose two weights have 4 bits: y = (act(x Wg) * (x Wu)) Wo

run() computes them in plain torch operations in 32 bits, or (``own``) through graphcuda_b200.  Widths and row counts are
those of the graph configurations (synth.py: 2708, 169,343 vertices; widths 64 to 256, 7 to 47 classes) and, beyond them,
powers of two and sizes as they fall.
"""
import math

import torch

own = False
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32
TYPES = {"bf16": BF16, "fp32": F32}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # A two-layer student on the small citation graph learns from a deep model on the labelled rows alone.  All latency.
        dict(name="distill_small", op="distill", rows=2708, classes=7, k=3, type="fp32", temperature=2.0, selected=0.05,
             holes=False, mode="train"),
        # The same over all vertices of the larger one, in a class count of its own.
        dict(name="distill_graph", op="distill", rows=169_343, classes=47, k=8, type="fp32", temperature=4.0, selected=1.0,
             holes=False, mode="train"),
        # Many classes, an odd count of them, lists of different lengths: how far the student is, without a gradient.
        dict(name="distill_odd_value", op="distill", rows=1000, classes=30_011, k=20, type="bf16", temperature=1.0,
             selected=0.7, holes=True, mode="forward"),
        # A training step over a large vocabulary.
        dict(name="distill_wide", op="distill", rows=4096, classes=65_536, k=64, type="bf16", temperature=2.0, selected=1.0,
             holes=False, mode="train"),
        # Every vertex through the weights of its kind, forward and backward: memory.
        dict(name="grouped_train_graph", op="grouped", rows=169_343, groups=8, inputs=256, outputs=256, skew=1.0, spare=0,
             mode="train"),
        # Wide weights, as many rows for a group as fill tiles: long products.
        dict(name="grouped_train_wide", op="grouped", rows=16_384, groups=16, inputs=2048, outputs=4096, skew=0.5, spare=0,
             mode="train"),
        # A server's batch: one or two rows for most groups, none for many.
        dict(name="grouped_rows", op="grouped", rows=64, groups=64, inputs=2048, outputs=2048, skew=0.7, spare=0, mode="forward"),
        # Odd widths, empty groups, rows behind the last group.
        dict(name="grouped_train_odd", op="grouped", rows=2708, groups=5, inputs=100, outputs=47, skew=2.0, spare=9, mode="train"),
        # One row through a wide layer's weights: latency.
        dict(name="linear4_row", op="linear4", rows=1, inputs=2048, outputs=8192, group=64, zeros=False),
        # A batch of rows, fine groups, zero points.
        dict(name="linear4_rows", op="linear4", rows=16, inputs=16_384, outputs=8192, group=32, zeros=True),
        # One row through a whole gated block.
        dict(name="block4_row", op="block4", rows=1, width=2048, hidden=8192, out=2048, act="silu", group=64, zeros=False),
        # Evaluation of every vertex of the larger citation graph.
        dict(name="block4_graph", op="block4", rows=169_343, width=256, hidden=1024, out=256, act="silu", group=128, zeros=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """Half of them as users choose widths (multiples of 8), half as they fall."""
    n = _log(rng, lo, hi)
    return max(8, n // 8 * 8) if rng.random() < 0.5 else n


def draw(rng):
    while True:
        op = rng.choice(("distill", "grouped", "linear4", "block4"))
        if op == "distill":
            classes = _log(rng, 2, 200_000)
            case = dict(op=op, rows=_log(rng, 1, 200_000), classes=classes, k=_log(rng, 1, min(classes, 256)),
                        type=rng.choice(("fp32", "bf16")), temperature=rng.choice((1.0, 2.0, 4.0)),
                        selected=rng.choice((1.0, 1.0, 0.5)), holes=rng.random() < 0.3,
                        mode=rng.choice(("forward", "train", "train")))
        elif op == "grouped":
            case = dict(op=op, rows=_log(rng, 1, 200_000), groups=_log(rng, 1, 128), inputs=_size(rng, 8, 4096),
                        outputs=_size(rng, 8, 4096), skew=rng.choice((0.0, 0.5, 1.0, 2.0)), spare=rng.choice((0, 0, 7)),
                        mode=rng.choice(("forward", "train", "train")))
        elif op == "linear4":
            case = dict(op=op, rows=_log(rng, 1, 20_000) if rng.random() < 0.4 else _log(rng, 1, 64),
                        inputs=_size(rng, 16, 16_384), outputs=_size(rng, 8, 16_384), group=rng.choice((32, 64, 128)),
                        zeros=rng.random() < 0.5)
        else:
            case = dict(op=op, rows=_log(rng, 1, 200_000) if rng.random() < 0.4 else _log(rng, 1, 64),
                        width=_size(rng, 16, 4096), hidden=_size(rng, 16, 8192), out=_size(rng, 16, 4096),
                        act=rng.choice(("silu", "gelu", "relu")), group=rng.choice((32, 64, 128)), zeros=rng.random() < 0.5)
        w = work(case)
        inner = case["rows"] * case.get("hidden", 0)
        if w["flops"] <= 7e11 and w["bytes"] <= 1e9 and inner <= 2e8:
            return case


def _weights4(inputs, outputs, case):
    """Bytes of codes, scales and zero points."""
    groups = -(-inputs // case["group"])
    return (inputs * outputs + 1) // 2 + groups * outputs * 2 + ((groups * outputs + 1) // 2 if case["zeros"] else 0)


def _shares(case):
    """Groups' shares of the rows, which fall off as a power of the rank."""
    share = [(i + 1) ** -case["skew"] for i in range(case["groups"])]
    return [p / sum(share) for p in share]


def _groups_with_rows(case):
    """How many groups are expected to have a row."""
    return round(sum(1 - (1 - p) ** case["rows"] for p in _shares(case)))


def work(case):
    m = case["rows"]
    if case["op"] == "distill":
        size = 4 if case["type"] == "fp32" else 2
        n, k = m * case["classes"] * case["selected"], m * case["k"] * case["selected"]
        train = case["mode"] == "train"
        return {"bytes": int(n * size + k * (size + 8) + m + (m * case["classes"] * size if train else 0)),
                "flops": int(n * (8 if train else 4) + k * 8)}
    if case["op"] == "grouped":
        d, o = case["inputs"], case["outputs"]
        weights = d * o * _groups_with_rows(case)
        if case["mode"] == "forward":
            return {"bytes": 2 * (m * d + m * o + weights), "flops": 2 * m * d * o}
        # x, weights and the output's gradient in; output and both gradients out
        return {"bytes": 2 * (2 * m * d + 2 * m * o + weights + case["groups"] * d * o), "flops": 6 * m * d * o}
    if case["op"] == "linear4":
        d, o = case["inputs"], case["outputs"]
        return {"bytes": 2 * m * (d + o) + _weights4(d, o, case), "flops": 2 * m * d * o}
    d, h, o = case["width"], case["hidden"], case["out"]
    return {"bytes": 2 * m * (d + o) + _weights4(d, 2 * h, case) + _weights4(h, o, case), "flops": 2 * m * h * (2 * d + o)}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, generator=g, device=DEV)  # noqa: E731
    rand = lambda *shape: torch.rand(*shape, generator=g, device=DEV)  # noqa: E731
    m = case["rows"]
    if case["op"] == "distill":
        # the teacher agrees with the student by half, and is surer
        t = TYPES[case["type"]]
        logits = (2 * randn(m, case["classes"])).to(t)
        top, index = (0.7 * logits + 2.5 * randn(m, case["classes"])).topk(case["k"], dim=1)
        if case["holes"]:  # some rows have fewer entries, down to none
            count = (rand(m, 1) * 1.3 * (case["k"] + 1)).floor()
            index = torch.where(torch.arange(case["k"], device=DEV) < count, index, -1)
        s = dict(case=case, logits=logits, top=top.to(t), index=index, mask=None, scale=1.0 / m)
        if case["selected"] < 1:
            s["mask"] = rand(m) < case["selected"]
            s["scale"] = 1.0 / max(1, round(m * case["selected"]))
        return s
    if case["op"] == "grouped":
        n, d, o = case["groups"], case["inputs"], case["outputs"]
        share = torch.tensor(_shares(case), device=DEV)[torch.randperm(n, generator=g, device=DEV)]  # in a random order
        kind = torch.searchsorted(torch.cumsum(share, 0)[:-1].contiguous(), rand(m))
        counts = torch.bincount(kind, minlength=n)
        offsets = torch.zeros(n + 1, dtype=torch.int32, device=DEV)
        offsets[1:] = torch.cumsum(counts, 0)
        rows = m + case["spare"]
        s = dict(case=case, x=randn(rows, d).to(BF16), w=(randn(n, d, o) / math.sqrt(d)).to(BF16), offsets=offsets,
                 bounds=offsets.tolist())
        if case["mode"] == "train":
            s["dy"] = randn(rows, o).to(BF16)
        return s
    if case["op"] == "linear4":
        s = dict(case=case, x=randn(m, case["inputs"]).to(BF16))
        s["w"] = _pack(randn(case["inputs"], case["outputs"]) / math.sqrt(case["inputs"]), case)
    else:
        d, h, o = case["width"], case["hidden"], case["out"]
        s = dict(case=case, x=randn(m, d).to(BF16))
        s["w_in"] = _pack(randn(d, 2 * h) / math.sqrt(d), case)
        s["w_out"] = _pack(randn(h, o) / math.sqrt(h), case)
    if own:  # a server lays its weights out once
        import graphcuda_b200 as gc
        for key in [k for k in ("w", "w_in", "w_out") if k in s]:
            s["laid_" + key] = gc.Int4Weight.from_codes(*s[key], group=case["group"])
    return s


def _groups(t, group):
    """Rows of t by their group: [groups, group, columns], the last one filled up with the last row."""
    n = -(-t.size(0) // group)
    index = torch.arange(n * group, device=t.device).clamp(max=t.size(0) - 1)
    return t[index].view(n, group, t.size(1))


def _pack(w, case):
    """Codes 0 to 15 [inputs, outputs], scales [groups, outputs], zero points [groups, outputs] or None: a weight is
    (code - zero point) * scale, the zero point 8 where there are none."""
    inputs, group = w.size(0), case["group"]
    t = _groups(w, group)
    if case["zeros"]:
        low, high = t.amin(1).clamp(max=0), t.amax(1).clamp(min=0)
        scale = ((high - low) / 15).to(BF16)
        zero = (-low / scale.float()).round().clamp(0, 15)
    else:
        scale = (t.abs().amax(1) / 7.5).to(BF16)
        zero = torch.full_like(scale, 8, dtype=F32)
    each = lambda v: v.float().repeat_interleave(group, 0)[:inputs]  # noqa: E731
    codes = (w / each(scale) + each(zero)).round().clamp(0, 15).to(torch.uint8)
    return codes, scale, zero.to(torch.uint8) if case["zeros"] else None


# ------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    return {"distill": _distill, "grouped": _grouped, "linear4": _linear4, "block4": _block4}[case["op"]](state, case)


def _distill(s, case):
    train, temperature = case["mode"] == "train", case["temperature"]
    if own:
        import graphcuda_b200 as gc
        if not train:
            with torch.no_grad():
                return {"loss": gc.distill_loss(s["logits"], s["top"], s["index"], s["mask"], temperature, scale=s["scale"])}
        logits = s["logits"].detach().requires_grad_()
        loss = gc.distill_loss(logits, s["top"], s["index"], s["mask"], temperature, scale=s["scale"])
        return {"loss": loss.detach(), "dlogits": torch.autograd.grad(loss, logits)[0]}
    z = s["logits"].float() / temperature
    z = z - z.amax(1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    index, there = s["index"].clamp(min=0), s["index"] >= 0
    t = torch.where(there, s["top"].float() / temperature, -math.inf)
    t = t - t.amax(1, keepdim=True)
    u = torch.where(there, torch.exp(t), 0.0)
    usum = u.sum(1, keepdim=True)
    counts = (usum > 0) if s["mask"] is None else (usum > 0) & s["mask"][:, None]
    p = u / torch.where(usum > 0, usum, 1.0)
    log_p = torch.where(p > 0, t - torch.log(torch.where(usum > 0, usum, 1.0)), 0.0)
    log_q = z.gather(1, index) - torch.log(total)
    row = (p * (log_p - log_q)).sum(1, keepdim=True)
    loss = torch.where(counts, row, 0.0).sum() * (temperature * temperature * s["scale"])
    if not train:
        return {"loss": loss}
    d = (e / total).scatter_add_(1, index, -p)
    d = torch.where(counts, d * (temperature * s["scale"]), 0.0)
    return {"loss": loss, "dlogits": d.to(s["logits"].dtype)}


def _grouped(s, case):
    train = case["mode"] == "train"
    if own:
        import graphcuda_b200 as gc
        if not train:
            with torch.no_grad():
                return gc.grouped_linear(s["x"], s["w"], s["offsets"])
        x, w = s["x"].detach().requires_grad_(), s["w"].detach().requires_grad_()
        y = gc.grouped_linear(x, w, s["offsets"])
        dx, dw = torch.autograd.grad(y, (x, w), s["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw}
    x, w, b = s["x"], s["w"], s["bounds"]
    y = x.new_zeros(x.size(0), w.size(2))
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    for i in range(w.size(0)):
        if b[i] == b[i + 1]:
            continue
        rows = slice(b[i], b[i + 1])
        xi, wi = x[rows].float(), w[i].float()
        y[rows] = (xi @ wi).to(BF16)
        if train:
            di = s["dy"][rows].float()
            dx[rows] = (di @ wi.t()).to(BF16)
            dw[i] = (xi.t() @ di).to(BF16)
    return {"y": y, "dx": dx, "dw": dw} if train else y


def _unpack(packed, case):
    codes, scale, zero = packed
    t = _groups(codes, case["group"]).float()
    w = (t - (8.0 if zero is None else zero.float()[:, None])) * scale.float()[:, None]
    return w.view(-1, codes.size(1))[:codes.size(0)]


def _linear4(s, case):
    if own:
        import graphcuda_b200 as gc
        return gc.linear_int4(s["x"], s["laid_w"])
    return (s["x"].float() @ _unpack(s["w"], case)).to(BF16)


def _block4(s, case):
    if own:
        import graphcuda_b200 as gc
        return gc.gated_ffn_int4(s["x"], s["laid_w_in"], s["laid_w_out"], activation=case["act"])
    h = case["hidden"]
    gu = s["x"].float() @ _unpack(s["w_in"], case)
    g = gu[:, :h]
    if case["act"] == "silu":
        a = g * torch.sigmoid(g)
    elif case["act"] == "gelu":
        a = g * (0.5 * (1 + torch.erf(g * math.sqrt(0.5))))
    else:
        a = g * (g > 0)
    return ((a * gu[:, h:]) @ _unpack(s["w_out"], case)).to(BF16)


# ------------------------------------------------------------------ the same in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "distill":
        t, m = case["temperature"], case["rows"]
        log_q = torch.log_softmax(s["logits"].double() / t, 1)
        # the teacher over all classes: what its list does not name has no probability
        here = s["index"] >= 0
        z = s["top"].double() / t
        z[~here] = -math.inf
        some = here.any(1)
        if s["mask"] is not None:
            some &= s["mask"]
        log_p = (z - torch.logsumexp(z, 1, keepdim=True)).masked_fill(~here, 0)
        p = (log_p.exp() * here).masked_fill(~some[:, None], 0)
        kl = (p * (log_p.masked_fill(~some[:, None], 0) - log_q.gather(1, s["index"].clamp(min=0)))).sum(1)
        got = {"loss": t * t * s["scale"] * kl.sum()}
        if case["mode"] == "train":
            d = log_q.exp_() * some[:, None]
            for j in range(case["k"]):  # an index stands once in a row's list
                d[torch.arange(m, device=DEV), s["index"][:, j].clamp(min=0)] -= p[:, j]
            got["dlogits"] = d * (t * s["scale"])
        return got
    if case["op"] == "grouped":
        # every row's group by comparison with the bounds, then one group after the other by selection
        rows = torch.arange(s["x"].size(0), device=DEV)
        kind = (rows[:, None] >= s["offsets"][1:].long()).sum(1)
        y = torch.zeros(rows.numel(), case["outputs"], dtype=torch.float64, device=DEV)
        dx, dw = torch.zeros(s["x"].shape, dtype=torch.float64, device=DEV), torch.zeros(s["w"].shape, dtype=torch.float64, device=DEV)
        for i in kind.unique().tolist():
            if i == case["groups"]:
                continue
            pick = (kind == i).nonzero()[:, 0]
            xi, wi = s["x"][pick].double(), s["w"][i].double()
            y.index_copy_(0, pick, torch.mm(xi, wi))
            if case["mode"] == "train":
                di = s["dy"][pick].double()
                dx.index_copy_(0, pick, torch.mm(di, wi.mT))
                dw[i] = torch.mm(xi.mT, di)
        return {"y": y, "dx": dx, "dw": dw} if case["mode"] == "train" else y

    def weights(packed):
        codes, scale, zero = packed
        group = torch.arange(codes.size(0), device=DEV) // case["group"]
        offset = 8 if zero is None else zero.double()[group]
        return (codes.double() - offset) * scale.double()[group]

    x = s["x"].double()
    if case["op"] == "linear4":
        return torch.mm(x, weights(s["w"]))
    gate, up = torch.mm(x, weights(s["w_in"])).split(case["hidden"], 1)
    if case["act"] == "silu":
        e = torch.exp(-gate.abs())
        act = gate * torch.where(gate >= 0, 1 / (1 + e), e / (1 + e))
    elif case["act"] == "gelu":
        act = gate * torch.special.erfc(-gate / math.sqrt(2)) / 2
    else:
        act = gate.clamp(min=0)
    return torch.mm(act * up, weights(s["w_out"]))
