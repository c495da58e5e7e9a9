"""AdamW over many tensors: 32 bits against the formula in 64 bits, 8 bits against the same codes formed on the host.

Tolerances: one step is a handful of float32 operations per element: 16 roundings of 2^-24 (1e-6) of the magnitudes that
meet in it are allowed, times the number of steps."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

HYPER = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
SIZES = [1, 3, 255, 256, 257, 1024, 2047, 2048, 2049, 5000, 70_001]


def _reference(p, g, m, v, t, lr, betas, eps, weight_decay):
    b1, b2 = betas
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    p = p - lr * weight_decay * p - lr * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + eps)
    return p, m, v


def _randn(n, seed, scale=1.0):
    return scale * torch.randn(n, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_32_bits_against_64(cuda, dtype):
    import graphcuda_b200 as gc
    start = [_randn(n, i).to(dtype) for i, n in enumerate(SIZES)]
    ps = [torch.nn.Parameter(t.to(cuda)) for t in start]
    opt = gc.FusedAdamW(ps, **HYPER)
    ref = [(t.double(), torch.zeros(t.shape, dtype=torch.float64), torch.zeros(t.shape, dtype=torch.float64)) for t in start]
    for t in range(1, 6):
        gs = [_randn(n, 100 * t + i, 10.0 ** (i % 5 - 3)).to(dtype) for i, n in enumerate(SIZES)]
        for p, g in zip(ps, gs):
            p.grad = g.to(cuda)
        opt.step()
        ref = [_reference(p, g.double(), m, v, t, **HYPER) for (p, m, v), g in zip(ref, gs)]
        for p, (rp, rm, rv) in zip(ps, ref):
            st = opt.state[p]
            full = st["master"] if dtype == torch.bfloat16 else p.detach()
            assert float((full.cpu().double() - rp).abs().max()) <= t * 1e-6 * (float(rp.abs().max()) + 1)
            assert float((st["exp_avg"].cpu().double() - rm).abs().max()) <= t * 1e-6 * float(rm.abs().max() + 1e-30)
            assert float(((st["exp_avg_sq"].cpu().double() - rv).abs() / (rv + 1e-30)).max()) <= t * 1e-6
            if dtype == torch.bfloat16:
                assert torch.equal(p.detach(), st["master"].to(dtype))
    assert opt.steps_taken() == 5


def test_follows_torch(cuda):
    import graphcuda_b200 as gc
    ours = [torch.nn.Parameter(_randn(n, i).to(cuda)) for i, n in enumerate(SIZES)]
    theirs = [torch.nn.Parameter(p.detach().cpu().clone()) for p in ours]
    a, b = gc.FusedAdamW(ours, **HYPER), torch.optim.AdamW(theirs, **HYPER)
    for t in range(4):
        for i, (p, q) in enumerate(zip(ours, theirs)):
            q.grad = _randn(p.numel(), 10 * t + i)
            p.grad = q.grad.to(cuda)
        a.step()
        b.step()
    for p, q in zip(ours, theirs):
        assert float((p.detach().cpu() - q.detach()).abs().max()) < 1e-5


# ---- 8 bits, formed on the host
def _mix(x):
    x = np.uint32(x) if np.isscalar(x) else x.astype(np.uint32)
    with np.errstate(over="ignore"):
        x = (x ^ (x >> np.uint32(16))) * np.uint32(0x85EBCA6B)
        x = (x ^ (x >> np.uint32(13))) * np.uint32(0xC2B2AE35)
    return x ^ (x >> np.uint32(16))


def _random(seed, step, tensor, n):
    with np.errstate(over="ignore"):
        key = _mix(np.uint32((seed + step * 0x9E3779B9) & 0xFFFFFFFF))
        key = _mix(np.uint32((int(key) + tensor) & 0xFFFFFFFF))
        return _mix(np.arange(n, dtype=np.uint32) + key)


def _blocks(x):
    out = np.zeros(-(-x.size // 256) * 256, dtype=np.float32)
    out[:x.size] = x
    return out.reshape(-1, 256)


def _scale(x, top):
    s = np.abs(x).max(1, keepdims=True) * np.float32(1.0 / top)
    s = np.where(s < np.float32(2.0 ** -126), np.float32(0), s)
    with np.errstate(divide="ignore"):
        inv = np.where(s > 0, np.float32(1) / s, np.float32(0)).astype(np.float32)
    return s.astype(np.float32), (x * inv).astype(np.float32)


def _values(mantissa, lowest, top):
    """The positive numbers of the format, ascending from zero."""
    v, e = [k * 2.0 ** (lowest - mantissa) for k in range(2 ** mantissa)], lowest
    while 2.0 ** e <= top:
        v += [2.0 ** e * (1 + k / 2 ** mantissa) for k in range(2 ** mantissa)]
        e += 1
    return np.array([x for x in v if x <= top])


M_VALUES, V_VALUES = _values(3, -6, 448.0), _values(3, -14, 61440.0)


def _codes(t, u16, values):
    """t (float32, >= 0) to the index of one of its two neighbours: the upper one where the place between them, in 2^-16
    and rounded as float32 sums are below the smallest normal number, and u16 reach 1."""
    t64 = t.astype(np.float64)
    low = np.clip(np.searchsorted(values, t64, side="right") - 1, 0, len(values) - 1)
    high = np.minimum(low + 1, len(values) - 1)
    step = np.where(high > low, values[high] - values[low], 1.0)
    even = t64 < values[8]  # the evenly spaced part: the sum in units of the step is a float32
    units = (t64 / values[1]).astype(np.float32) + (u16 * 2.0 ** -16).astype(np.float32)
    up = (t64 - values[low]) / step + u16 * 2.0 ** -16 >= 1
    return np.where(even, units.astype(np.int64), np.where(up, high, low))


def _host_step(g, m, v, seed, step, tensor):
    """One update of 8-bit moments: (codes, scales, values) of both."""
    b1, b2 = HYPER["betas"]
    g = _blocks(g)
    m = m * np.float32(b1) + g * np.float32(1 - b1)
    v = v * np.float32(b2) + (g * g) * np.float32(1 - b2)
    r = _random(seed, step, tensor, g.size).reshape(-1, 256)
    ms, tm = _scale(m, 448.0)
    vs, tv = _scale(v, 61440.0)
    qm = _codes(np.abs(tm), r & np.uint32(0xFFFF), M_VALUES)
    qv = np.where(vs > 0, np.maximum(_codes(tv, r >> np.uint32(16), V_VALUES), 1), 0)
    m_code = qm | (np.signbit(tm).astype(np.int64) << 7)
    return m_code, qv, ms, vs, (np.copysign(M_VALUES[qm], tm).astype(np.float32) * ms), V_VALUES[qv].astype(np.float32) * vs


def test_8_bit_codes_are_those_of_the_formula(cuda):
    import graphcuda_b200 as gc
    grads = {
        "normal": _randn(3000, 1).numpy(),
        "spread": (_randn(2049, 2) * torch.exp(6 * _randn(2049, 3))).numpy(),
        "zeros": np.zeros(600, dtype=np.float32),
        "one": np.eye(1, 700, 300, dtype=np.float32)[0] * 3,
        "tiny": (_randn(512, 4) * 1e-22).numpy(),
        "subnormal": (_randn(512, 5) * 1e-38).numpy(),
        "large": (_randn(512, 6) * 1e18).numpy(),
        "short": _randn(5, 7).numpy(),
    }
    names, seed = list(grads), 0xFFFFFFF0
    ps = [torch.zeros(grads[k].size, device=cuda) for k in names]
    codes = [[torch.zeros(p.numel(), dtype=torch.uint8, device=cuda) for p in ps] for _ in range(2)]
    scales = [[torch.zeros(-(-p.numel() // 256), device=cuda) for p in ps] for _ in range(2)]
    step = torch.zeros(2, dtype=torch.int64, device=cuda)
    host = {k: (np.zeros_like(_blocks(grads[k])), np.zeros_like(_blocks(grads[k]))) for k in names}
    for t in range(1, 5):
        sign = 1 if t % 2 else -0.5
        gs = {k: (grads[k] * np.float32(sign)).astype(np.float32) for k in names}
        gc.adamw_step(ps, [torch.from_numpy(gs[k]).to(cuda) for k in names], *codes, step, scales=scales, seed=seed, **HYPER)
        got_m, got_v = gc.adamw_moments(*codes, scales)
        for i, k in enumerate(names):
            n = grads[k].size
            qm, qv, ms, vs, m, v = _host_step(gs[k], *host[k], seed, t, i)
            host[k] = m, v
            assert np.array_equal(scales[0][i].cpu().numpy(), ms[:, 0]), (k, t)
            assert np.array_equal(scales[1][i].cpu().numpy(), vs[:, 0]), (k, t)
            assert np.array_equal(codes[0][i].cpu().numpy(), qm.reshape(-1)[:n]), (k, t)
            assert np.array_equal(codes[1][i].cpu().numpy(), qv.reshape(-1)[:n]), (k, t)
            assert np.array_equal(got_m[i].cpu().numpy(), m.reshape(-1)[:n]), (k, t)
            assert np.array_equal(got_v[i].cpu().numpy(), v.reshape(-1)[:n]), (k, t)
            # beyond the tensor's end the host's blocks are zeros, as the kernel takes them to be
            host[k][0].reshape(-1)[n:] = 0
            host[k][1].reshape(-1)[n:] = 0
    assert int(step[0]) == 4 and int(step[1]) == 0


def test_8_bit_rounding_has_no_bias(cuda):
    """A constant gradient: the moments, rounded at random every step, keep the mean of the exact ones.  The spread of one
    element's relative error is under 0.25 (2^-4 per step over a memory of 1 / (1 - beta)); over 2^18 elements the mean's is
    under 5e-4, and five of those are allowed."""
    import graphcuda_b200 as gc
    n = 1 << 18
    g = torch.ones(n, device=cuda)
    g[::256] = 4.0  # the block's largest element: the others lie between codes
    p = torch.zeros(n, device=cuda)
    codes = [[torch.zeros(n, dtype=torch.uint8, device=cuda)] for _ in range(2)]
    scales = [[torch.zeros(n // 256, device=cuda)] for _ in range(2)]
    step = torch.zeros(2, dtype=torch.int64, device=cuda)
    rest = torch.ones(n, dtype=torch.bool, device=cuda)
    rest[::256] = False
    for _ in range(60):
        gc.adamw_step([p], [g], *codes, step, scales=scales, **HYPER)
    m, v = (t[0][rest].double().mean().item() for t in gc.adamw_moments(*codes, scales))
    assert abs(m / (1 - 0.9 ** 60) - 1) < 2.5e-3 and abs(v / (1 - 0.99 ** 60) - 1) < 2.5e-3


def test_8_bit_block_with_nan_or_infinity(cuda):
    """Only the block that met it is lost, and it says so."""
    import graphcuda_b200 as gc
    for bad in (float("nan"), float("inf")):
        p, g = torch.zeros(1024, device=cuda), torch.ones(1024, device=cuda)
        g[300] = bad
        codes = [[torch.zeros(1024, dtype=torch.uint8, device=cuda)] for _ in range(2)]
        scales = [[torch.zeros(4, device=cuda)] for _ in range(2)]
        step = torch.zeros(2, dtype=torch.int64, device=cuda)
        gc.adamw_step([p], [g], *codes, step, scales=scales, **HYPER)
        keep = torch.ones(4, dtype=torch.bool)
        keep[1] = False
        for s in scales:
            assert torch.equal(torch.isfinite(s[0]).cpu(), keep)
        m, _ = gc.adamw_moments(*codes, scales)
        assert torch.isfinite(m[0][:256]).all() and torch.isfinite(m[0][512:]).all() and not torch.isfinite(m[0][300])
        assert torch.isfinite(p[:256]).all() and not torch.isfinite(p[300])


def test_small_elements_of_a_block_do_not_run_away(cuda):
    """Beside an element a million times their size, the others' second moments are at the bottom of their range: no step may
    be larger than a few learning rates."""
    import graphcuda_b200 as gc
    g = _randn(2048, 8, 1e-6).to(cuda)
    g[::256] = 1.0
    p = torch.nn.Parameter(torch.zeros(2048, device=cuda))
    opt = gc.FusedAdamW([p], lr=1.0, weight_decay=0.0, state_bits=8)
    for t in range(50):
        before = p.detach().clone()
        p.grad = g * (1 if t % 3 else -1) * (0.0 if t % 5 == 4 else 1.0)
        opt.step()
        assert float((p.detach() - before).abs().max()) < 10


def test_unaligned_tensors_and_many_of_them(cuda):
    """Views at odd offsets, an empty tensor, more tensors than a launch takes: equal to the aligned ones bit for bit."""
    import graphcuda_b200 as gc
    sizes = [(i * 37) % 700 for i in range(1000)]
    for bits, dtype in ((32, torch.float32), (8, torch.float32), (8, torch.bfloat16), (32, torch.bfloat16)):
        runs = []
        for off in (0, 1):
            def place(n, kind, fill=None):
                base = torch.zeros(n + 8, dtype=kind, device=cuda)
                v = base[off:off + n]
                if fill is not None:
                    v.copy_(fill)
                return v
            ps = [place(n, dtype, _randn(n, i)) for i, n in enumerate(sizes)]
            gs = [place(n, dtype, _randn(n, 1000 + i)) for i, n in enumerate(sizes)]
            kind = torch.uint8 if bits == 8 else torch.float32
            m, v = ([place(n, kind) for n in sizes] for _ in range(2))
            scales = tuple([torch.zeros(-(-n // 256), device=cuda) for n in sizes] for _ in range(2)) if bits == 8 else None
            masters = [place(n, torch.float32, p) for n, p in zip(sizes, ps)] if dtype == torch.bfloat16 else None
            step = torch.zeros(2, dtype=torch.int64, device=cuda)
            for _ in range(3):
                gc.adamw_step(ps, gs, m, v, step, masters=masters, scales=scales, **HYPER)
            assert int(step[0]) == 3
            runs.append(ps + m + v + (masters or []) + (list(scales[0]) + list(scales[1]) if scales else []))
        assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_8_bits_train_like_32(cuda):
    """A small regression: the loss falls as far with 8-bit moments, and in bf16 with masters."""
    import graphcuda_b200 as gc
    g = torch.Generator().manual_seed(0)
    X, W = torch.randn(512, 64, generator=g).to(cuda), torch.randn(64, 32, generator=g).to(cuda)
    losses = {}
    for bits, dtype in ((32, torch.float32), (8, torch.float32), (8, torch.bfloat16)):
        p = torch.nn.Parameter(torch.zeros(64, 32, device=cuda, dtype=dtype))
        opt = gc.FusedAdamW([p], lr=0.02, weight_decay=0.0, state_bits=bits)
        for _ in range(300):
            opt.zero_grad(set_to_none=True)
            loss = (X @ p.float() - X @ W).square().mean()
            loss.backward()
            opt.step()
        losses[bits, dtype] = loss.item()
    first = (X @ W).square().mean().item()
    assert all(v < 1e-3 * first for v in losses.values()), losses


def test_parameters_that_join_late_or_pause_count_their_own_steps(cuda):
    import graphcuda_b200 as gc
    ours = [torch.nn.Parameter(_randn(n, i).to(cuda)) for i, n in enumerate((300, 40, 513))]
    theirs = [torch.nn.Parameter(p.detach().cpu().clone()) for p in ours]
    a, b = gc.FusedAdamW(ours, **HYPER), torch.optim.AdamW(theirs, **HYPER)
    for t, has in enumerate(((1, 0, 1), (1, 1, 1), (0, 1, 1), (1, 1, 1), (1, 1, 0))):
        for i, (p, q) in enumerate(zip(ours, theirs)):
            q.grad = _randn(p.numel(), 10 * t + i) if has[i] else None
            p.grad = q.grad.to(cuda) if has[i] else None
        a.step()
        b.step()
    for p, q in zip(ours, theirs):
        assert int(a.state[p]["step"][0]) == int(b.state[q]["step"])
        assert float((p.detach().cpu() - q.detach()).abs().max()) < 1e-5


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_checkpoint(cuda, bits, dtype, tmp_path):
    """Saved and loaded, a run continues bit for bit."""
    import graphcuda_b200 as gc
    sizes = (700, 33, 4096)

    def run(resume):
        ps = [torch.nn.Parameter(_randn(n, i).to(cuda, dtype)) for i, n in enumerate(sizes)]
        opt = gc.FusedAdamW(ps, **HYPER, state_bits=bits, seed=3)
        for t in range(6):
            if resume and t == 3:
                torch.save({"opt": opt.state_dict(), "ps": [p.detach() for p in ps]}, tmp_path / "c.pt")
                saved = torch.load(tmp_path / "c.pt", weights_only=True)
                ps = [torch.nn.Parameter(x.clone()) for x in saved["ps"]]
                opt = gc.FusedAdamW(ps, lr=1.0, state_bits=bits)
                opt.load_state_dict(saved["opt"])
            for i, p in enumerate(ps):
                p.grad = _randn(p.numel(), 10 * t + i).to(cuda, dtype)
            opt.step()
        return ps, [opt.moments(p) for p in ps], opt.steps_taken()

    a, b = run(False), run(True)
    assert a[2] == b[2] == 6
    assert all(torch.equal(x, y) for x, y in zip(a[0], b[0]))
    assert all(torch.equal(x, y) for s, t in zip(a[1], b[1]) for x, y in zip(s, t))


@pytest.mark.parametrize("bits", [8, 32])
def test_recorded_step(cuda, bits):
    import graphcuda_b200 as gc
    runs = []
    for recorded in (False, True):
        p = torch.nn.Parameter(_randn(5000, 0).to(cuda))
        p.grad = _randn(5000, 1).to(cuda)
        opt = gc.FusedAdamW([p], **HYPER, state_bits=bits)
        opt.step()
        if recorded:
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                opt.step()
        for _ in range(4):
            graph.replay() if recorded else opt.step()
        runs.append((p.detach().clone(), *opt.moments(p), opt.steps_taken()))
    assert runs[0][3] == runs[1][3] == 5
    assert all(torch.equal(a, b) for a, b in zip(runs[0][:3], runs[1][:3]))


def test_refusals(cuda):
    import graphcuda_b200 as gc
    p, step = torch.zeros(300, device=cuda), torch.zeros(2, dtype=torch.int64, device=cuda)
    b, s = torch.zeros(300, dtype=torch.uint8, device=cuda), torch.zeros(2, device=cuda)
    ok = dict(lr=0.1)
    for bad in (lambda: gc.adamw_step([p], [p.cpu()], [p], [p], step, **ok),
                lambda: gc.adamw_step([p.cpu()], [p], [p], [p], step, **ok),
                lambda: gc.adamw_step([p], [p[:299]], [p], [p], step, **ok),
                lambda: gc.adamw_step([p], [p.double()], [p], [p], step, **ok),
                lambda: gc.adamw_step([p], [p], [p], [], step, **ok),
                lambda: gc.adamw_step([p], [p], [b], [b], step, **ok),
                lambda: gc.adamw_step([p], [p], [b], [p], step, scales=([s], [s]), **ok),
                lambda: gc.adamw_step([p], [p], [b], [b], step, scales=([s[:1]], [s]), **ok),
                lambda: gc.adamw_step([p], [p], [p], [p], step, scales=([s], [s]), **ok),
                lambda: gc.adamw_step([p.bfloat16()], [p.bfloat16()], [p], [p], step, **ok),
                lambda: gc.adamw_step([p], [p], [p], [p], step, masters=[p], **ok),
                lambda: gc.adamw_step([p.view(20, 15).t()], [p], [p], [p], step, **ok),
                lambda: gc.adamw_step([p], [p], [p], [p], step.cpu(), **ok),
                lambda: gc.adamw_step([p], [p], [p], [p], step[:1], **ok),
                lambda: gc.adamw_step([p], [p], [p], [p], step, lr=-1.0),
                lambda: gc.adamw_step([p], [p], [p], [p], step, lr=0.1, betas=(1.0, 0.9)),
                lambda: gc.adamw_moments([p], [p], ([s], [s])),
                lambda: gc.adamw_moments([b], [b], ([s], [s[:1]]))):
        with pytest.raises(RuntimeError):
            bad()
    assert not p.any() and not step.any()
    for bad in (dict(lr=-1), dict(betas=(0.9, 1.0)), dict(state_bits=16), dict(weight_decay=-0.1)):
        with pytest.raises(ValueError):
            gc.FusedAdamW([torch.nn.Parameter(p)], **bad)
