"""The gated feed-forward block against its formula in 64 bits, at sizes around its tiles, and in its layouts and types.

Tolerances.  u = 2^-8 is what rounding to bf16 may change a value by, relative.  Rounded are: the hidden row before the second
product; G, U and the gradients dG, dU for the backward pass; the outputs.  An operand's roundings are independent, so a sum
of products picks up a random error of u / sqrt(3) times the root of its summed squares at most; six of those (3.5 u) are
allowed, and u of the output itself.  float32 sums add K 2^-23 of the summed magnitudes at most, under 2e-5 here and
covered by the 1 % on u.  The second derivatives of the activations are under 0.8, the first under 1.13."""
import pytest
import torch
import torch.autograd.forward_ad as fw

pytestmark = pytest.mark.gpu

U = 2.0 ** -8 * 1.01
SHAPES = [(1, 1, 1, 1), (1, 8, 8, 8), (3, 5, 7, 9), (1, 256, 1024, 256), (2, 64, 64, 64), (130, 72, 200, 40), (129, 100, 267, 47),
          (300, 47, 65, 100), (257, 256, 512, 256), (1000, 8, 1000, 8), (33, 1433, 16, 7), (513, 129, 1032, 260),
          (128, 128, 128, 128), (2708, 64, 171, 64), (5, 2048, 4096, 1024)]
LARGE = [(20_001, 256, 1024, 256), (4096, 512, 2048, 520), (9473, 136, 256, 1024), (70_000, 16, 24, 32)]


def _inputs(shape, seed=0):
    m, d, h, o = shape
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    return [t.bfloat16() for t in (randn(m, d), randn(d, 2 * h) / d ** 0.5, randn(h, o) / h ** 0.5, randn(m, o))]


def _act(name, g):
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    if name == "gelu":
        c = 0.5 * torch.special.erfc(-g * 0.5 ** 0.5)
        return g * c, c + g * torch.exp(-0.5 * g * g) * 0.3989422804014327
    return g.clamp(min=0), (g > 0).double()


def _exact(x, w_in, w_out, dy, act):
    """Outputs and gradients, and what the roundings may change them by."""
    x, w_in, w_out, dy = (t.double() for t in (x, w_in, w_out, dy))
    h = w_out.size(0)
    g, u = x @ w_in[:, :h], x @ w_in[:, h:]
    a, slope = _act(act, g)
    hid = a * u
    y = hid @ w_out
    da = dy @ w_out.t()
    dg, du = da * u * slope, da * a
    curve = 0.0 if act == "relu" else 0.8
    eg = 2 * dg.abs() + curve * (da * u * g).abs()
    eu = du.abs() + 1.13 * (da * g).abs()
    dgu, e = torch.cat((dg, du), 1), torch.cat((eg, eu), 1)
    got = {"y": y, "dx": dgu @ w_in.t(), "dw_in": x.t() @ dgu, "dw_out": hid.t() @ dy}
    sq = torch.square
    noise = {"y": sq(hid) @ sq(w_out), "dx": sq(e) @ sq(w_in).t(), "dw_in": sq(x).t() @ sq(e), "dw_out": sq(hid).t() @ sq(dy)}
    return got, {k: U * (got[k].abs() + 3.5 * noise[k].sqrt()) + 1e-30 for k in got}


def _run(x, w_in, w_out, dy, act):
    import graphcuda_b200 as gc
    leaves = [t.detach().requires_grad_() for t in (x, w_in, w_out)]
    y = gc.gated_ffn(*leaves, activation=act)
    return dict(zip(("y", "dx", "dw_in", "dw_out"), (y.detach(), *torch.autograd.grad(y, leaves, dy))))


def _check(got, ref, tol):
    for k in got:
        assert got[k].dtype == torch.bfloat16 and got[k].shape == ref[k].shape, k
        over = (got[k].double() - ref[k]).abs() - tol[k]
        assert not over.numel() or float(over.max()) <= 0, (k, float(over.max()), int((over > 0).sum()), int(over.argmax()))


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward_and_backward(cuda, shape, act):
    from graphcuda_b200 import ops
    t = _inputs(shape)
    got = _run(*t, act)
    _check(got, *_exact(*t, act))
    import graphcuda_b200 as gc
    with torch.no_grad():
        assert torch.equal(gc.gated_ffn(*t[:3], activation=act), got["y"])
    ops.check_gemm_flag(cuda)


@pytest.mark.parametrize("shape", LARGE, ids=str)
def test_large(cuda, shape):
    from graphcuda_b200 import ops
    t = _inputs(shape, seed=1)
    got = _run(*t, "silu")
    _check(got, *_exact(*t, "silu"))
    again = _run(*t, "silu")
    assert all(torch.equal(got[k], again[k]) for k in got)
    ops.check_gemm_flag(cuda)


@pytest.mark.parametrize("shape", [(1, 1, 1, 1), (1, 256, 1024, 256), (3, 5, 7, 9), (129, 100, 267, 47), (300, 144, 65, 100),
                                   (257, 256, 512, 256), (33, 1433, 16, 7), (20_001, 256, 1024, 256), (4096, 1040, 520, 64)], ids=str)
def test_eight_bits(cuda, shape):
    """The operands' 8-bit values are the inputs here: the products of them are exact, the rest is as in 16 bits."""
    import graphcuda_b200 as gc
    x, w_in, w_out, _ = _inputs(shape, seed=2)
    x8, xs = gc.quantize_weight_fp8(x.t())  # a scale per row of x
    w8, ws = gc.quantize_weight_fp8(w_in)
    assert w8.shape == (w_in.size(1), w_in.size(0))
    value = w8.double() * ws.double()[:, None]
    wt = w_in.double().t()
    assert float(((value - wt).abs() - wt.abs() * 0.0626 - ws.double()[:, None] * 2.0 ** -9).max()) <= 0
    for act in ("silu", "gelu", "relu"):
        got = gc.gated_ffn_fp8(x8, xs, w8, ws, w_out, activation=act)
        gu = (x8.double() * xs.double()[:, None]) @ value.t()
        h = w_out.size(0)
        hid = _act(act, gu[:, :h])[0] * gu[:, h:]
        y = hid @ w_out.double()
        # float32 scales and products change gu by 2^-22 of the sum's magnitude
        tol = U * (y.abs() + 3.5 * (hid.square() @ w_out.double().square()).sqrt()) + 1e-30
        assert float(((got.double() - y).abs() - tol).max()) <= 0


def test_norm_feeds_the_block_in_eight_bits(cuda):
    import graphcuda_b200 as gc
    torch.manual_seed(0)
    norm, ffn = gc.RMSNorm(96, out_dtype=torch.bfloat16).to(cuda), gc.GatedFFN(96, 160, 96).to(cuda)
    x, r = torch.randn(200, 96, device=cuda).bfloat16(), torch.randn(200, 96, device=cuda)
    with torch.no_grad():
        a, h = norm(x, r)
        y = ffn(a)
        y8 = ffn.for_serving()(*norm.fp8(x, r)[:2])
    assert y8.dtype == torch.bfloat16
    assert float((y8.float() - y.float()).norm() / y.float().norm()) < 0.08  # two operands, each off by up to 2^-4


def test_layouts(cuda):
    """Slices with another pitch, bases that are not aligned, transposes, broadcast rows: equal to contiguous copies."""
    x, w_in, w_out, dy = _inputs((200, 320, 640, 320), seed=3)
    for views in ((x[:, 8:264], w_in[:256, 128:384], w_out[:128, 8:72], dy[:, 16:80]),
                  (x[:, 3:259], w_in[1:257, 5:261], w_out[:128, 1:65], dy[:, 3:67]),
                  (w_in[:200, :256], x[:64].t()[:256, :64], w_out[:64, :64].t()[:32], dy.t()[:64, :200].t()),
                  (x[:1, :256].expand(200, 256), w_in[:256, :64], w_out[:32, :64], dy[:1, :64].expand(200, 64))):
        m = views[0].size(0)
        views = (*views[:3], views[3][:m])
        a, b = _run(*views, "silu"), _run(*[v.clone(memory_format=torch.contiguous_format) for v in views], "silu")
        assert all(torch.equal(a[k], b[k]) for k in a)


@pytest.mark.parametrize("shape", [(0, 8, 8, 8), (4, 0, 8, 8), (4, 8, 0, 8), (4, 8, 8, 0), (0, 0, 0, 0)], ids=str)
def test_empty(cuda, shape):
    import graphcuda_b200 as gc
    m, d, h, o = shape
    t = [torch.randn(s, device=cuda).bfloat16() for s in ((m, d), (d, 2 * h), (h, o), (m, o))]
    got = _run(*t, "silu")
    assert got["y"].shape == (m, o) and not any(v.any() for v in got.values())
    x8 = torch.zeros(m, d, device=cuda).to(torch.float8_e4m3fn)
    y = gc.gated_ffn_fp8(x8, torch.ones(m, device=cuda), *gc.quantize_weight_fp8(t[1]), t[2])
    assert y.shape == (m, o) and not y.any()


def test_infinities_and_nan_stay_in_their_rows(cuda):
    x, w_in, w_out, dy = _inputs((150, 64, 96, 32), seed=4)
    ref = _run(x, w_in, w_out, dy, "silu")
    x = x.clone()
    x[7, 3], x[140, 0] = float("nan"), float("inf")
    got = _run(x, w_in, w_out, dy, "silu")
    keep = torch.ones(150, dtype=torch.bool, device=cuda)
    keep[[7, 140]] = False
    assert torch.equal(got["y"][keep], ref["y"][keep]) and torch.equal(got["dx"][keep], ref["dx"][keep])
    assert torch.isnan(got["y"][7]).all() and not torch.isfinite(got["y"][140]).any()
    relu = _run(x, w_in, w_out, dy, "relu")
    assert torch.isnan(relu["y"][7]).all()


def test_large_arguments_of_the_activations(cuda):
    x, w_in, w_out, dy = _inputs((64, 64, 64, 64), seed=5)
    for act in ("silu", "gelu", "relu"):
        t = (x * 100, w_in, w_out, dy)
        ref, tol = _exact(*t, act)
        _check(_run(*t, act), ref, tol)


def test_gradient_against_differences(cuda):
    """A central difference of the formula in 64 bits along a direction: what the gradients say of it, to 2 %, the spread that
    bf16 leaves in a sum over all elements being far below."""
    t = _inputs((40, 24, 48, 16), seed=6)
    for act in ("silu", "gelu"):
        got = _run(*t, act)
        for i, k in enumerate(("dx", "dw_in", "dw_out")):
            d = torch.randn(t[i].shape, device=cuda, dtype=torch.float64)
            def value(s):
                v = [u.double() + (s * d if j == i else 0) for j, u in enumerate(t[:3])]
                h = v[2].size(0)
                gu = v[0] @ v[1]
                return float(((_act(act, gu[:, :h])[0] * gu[:, h:]) @ v[2] * t[3].double()).sum())
            slope = (value(1e-5) - value(-1e-5)) / 2e-5
            scale = float(got[k].double().norm() * d.norm()) / d.numel() ** 0.5
            assert abs(slope - float((got[k].double() * d).sum())) < 0.02 * (abs(slope) + scale)


def test_only_what_is_needed(cuda):
    import graphcuda_b200 as gc
    for shape in ((129, 96, 136, 40), (50, 33, 67, 21)):
        x, w_in, w_out, dy = _inputs(shape, seed=7)
        full = _run(x, w_in, w_out, dy, "silu")
        for need in range(1, 8):
            t = [v.clone().requires_grad_(bool(need >> i & 1)) for i, v in enumerate((x, w_in, w_out))]
            gc.gated_ffn(*t).backward(dy)
            for i, k in enumerate(("dx", "dw_in", "dw_out")):
                assert torch.equal(t[i].grad, full[k]) if need >> i & 1 else t[i].grad is None


def test_streams_graph_and_trace(cuda):
    import graphcuda_b200 as gc
    x, w_in, w_out, dy = _inputs((300, 128, 256, 128), seed=8)
    expect = _run(x, w_in, w_out, dy, "silu")
    sides = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in sides:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(_run(x, w_in, w_out, dy, "silu"))
    torch.cuda.synchronize()
    assert all(torch.equal(g[k], expect[k]) for g in got for k in expect)
    leaves = [t.clone().requires_grad_() for t in (x, w_in, w_out)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = gc.gated_ffn(*leaves)
        grads = torch.autograd.grad(y, leaves, dy)
    new = _inputs((300, 128, 256, 128), seed=9)
    with torch.no_grad():
        for a, b in zip(leaves, new):
            a.copy_(b)
        dy.copy_(new[3])
    graph.replay()
    expect = _run(*new, "silu")
    assert all(torch.equal(a.detach(), b) for a, b in zip((y, *grads), expect.values()))
    for grad in (False, True):
        block = gc.GatedFFN(128, 64, 32).to(cuda).requires_grad_(grad)
        with torch.set_grad_enabled(grad):
            traced = torch.jit.trace(block, (x,), check_trace=False)
            assert torch.equal(traced(new[0]), block(new[0]))
            if grad:
                a, b = (torch.autograd.grad(f(new[0]).float().sum(), tuple(block.parameters())) for f in (traced, block))
                assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_refusals(cuda):
    import graphcuda_b200 as gc
    x, w_in, w_out, _ = _inputs((8, 16, 24, 32))
    x8, xs = gc.quantize_weight_fp8(x.t())
    w8, ws = gc.quantize_weight_fp8(w_in)
    for bad in (lambda: gc.gated_ffn(x.cpu(), w_in, w_out), lambda: gc.gated_ffn(x.float(), w_in, w_out),
                lambda: gc.gated_ffn(x, w_in.float(), w_out), lambda: gc.gated_ffn(x, w_in, w_out.cpu()),
                lambda: gc.gated_ffn(x, w_in[:, :47], w_out), lambda: gc.gated_ffn(x, w_in[:15], w_out),
                lambda: gc.gated_ffn(x, w_in, w_out[:23]), lambda: gc.gated_ffn(x[0], w_in, w_out),
                lambda: gc.gated_ffn_fp8(x, xs, w8, ws, w_out), lambda: gc.gated_ffn_fp8(x8, xs[:7], w8, ws, w_out),
                lambda: gc.gated_ffn_fp8(x8, xs, w8, ws.double(), w_out), lambda: gc.gated_ffn_fp8(x8, xs, w8[:47], ws, w_out),
                lambda: gc.gated_ffn_fp8(x8, xs, w8, ws, w_out.requires_grad_()), lambda: gc.quantize_weight_fp8(x8[0])):
        with pytest.raises(RuntimeError):
            bad()
    with pytest.raises(ValueError):
        gc.gated_ffn(x, w_in, w_out, activation="tanh")
    y = gc.gated_ffn(x.requires_grad_(), w_in, w_out.detach())
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(y.sum(), x, create_graph=True)
    with fw.dual_level(), pytest.raises(RuntimeError, match="jvp"):
        gc.gated_ffn(fw.make_dual(x.detach(), torch.ones_like(x)), w_in, w_out.detach())
