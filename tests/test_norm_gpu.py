"""The residual norm against its formula in 64 bits, at the widths, types, layouts and values where it can go wrong.

Tolerances: a sum over a row passes through at most 32 additions in a thread and 8 joins, the rest is a handful of
operations: under 64 roundings of 2^-24, 3.8e-6 of the summed magnitudes; 8e-6 is allowed.  A 16-bit result is rounded
once more (2^-8), an 8-bit one by half a step (2^-4, or 2^-10 scales below the smallest normal number)."""
import pytest
import torch
import torch.autograd.forward_ad as fw

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
SUM = 8e-6
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8 * 1.01}
SHAPES = [(1, 1), (1, 256), (3, 7), (40, 16), (33, 64), (17, 100), (5, 256), (300, 257), (9, 512), (6, 1000), (4, 1024),
          (11, 1433), (3, 2048), (3, 4096), (2, 5001), (2, 8192), (3, 8200), (2, 9001)]
TYPES = [(F32, F32, F32), (BF16, BF16, BF16), (BF16, F32, BF16), (F32, F32, BF16), (BF16, BF16, F32)]


def _inputs(shape, tx, ts, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g).to(tx)
    r = (2 * torch.randn(shape, generator=g)).to(ts)
    w = 1 + 0.2 * torch.randn(shape[1], generator=g)
    return x, r, w


def _exact(x, r, w, eps):
    h = x.double() if r is None else x.double() + r.double()
    c = 1 / (h.square().mean(1, keepdim=True) + eps).sqrt()
    return h, c, h * c * w.double()


def _close(got, ref, tol):
    assert got.shape == ref.shape
    over = (got.detach().cpu().double() - ref).abs() - tol
    assert not over.numel() or float(over.max()) <= 0, float(over.max())


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward_and_backward(cuda, shape, types):
    import graphcuda_b200 as gc
    tx, ts, ty = types
    for add in (True, False):
        if not add and ts != tx:
            continue
        x, r, w = _inputs(shape, tx, ts)
        g = torch.Generator().manual_seed(1)
        dy, ds = torch.randn(shape, generator=g).to(ty), torch.randn(shape, generator=g).to(ts)
        leaves = [t.to(cuda).requires_grad_() for t in ((x, w, r) if add else (x, w))]
        got = gc.rms_norm(leaves[0], leaves[1], leaves[2] if add else None, eps=1e-5, out_dtype=ty)
        h, c, y = _exact(x, r if add else None, w, 1e-5)
        _close(got[0] if add else got, y, (SUM + HALF[ty]) * y.abs() + 1e-30)
        if add:
            assert got[1].dtype == ts
            _close(got[1], h, HALF[ts] * h.abs())
            grads = torch.autograd.grad(got, leaves, (dy.to(cuda), ds.to(cuda)))
        else:
            grads = torch.autograd.grad(got, leaves, dy.to(cuda))
        gw, hat = dy.double() * w.double(), h * c
        direct, through = c * gw, c * hat * (gw * hat).mean(1, keepdim=True)
        d = direct - through + (ds.double() if add else 0)
        tol = SUM * (direct.abs() + (c * hat).abs() * (gw * hat).abs().mean(1, keepdim=True) + (ds.double().abs() if add else 0))
        assert grads[0].dtype == tx and grads[1].dtype == F32
        _close(grads[0], d, tol + HALF[tx] * d.abs())
        _close(grads[1], (dy.double() * hat).sum(0), SUM * (dy.double() * hat).abs().sum(0))
        if add:
            assert grads[2].dtype == ts
            _close(grads[2], d, tol + HALF[ts] * d.abs())


@pytest.mark.parametrize("types", [(F32, F32), (BF16, BF16), (BF16, F32)], ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_eight_bits(cuda, shape, types):
    import graphcuda_b200 as gc
    x, r, w = _inputs(shape, *types, seed=2)
    y8, scale, stream = gc.rms_norm_fp8(x.to(cuda), w.to(cuda), r.to(cuda))
    h, _, y = _exact(x, r, w, 1e-6)
    top = y.abs().max(1).values / 448
    _close(scale, top, SUM * top)
    _close(stream, h, HALF[types[1]] * h.abs())
    assert y8.dtype == torch.float8_e4m3fn and float(y8.float().abs().max()) == 448
    value = y8.float().cpu().double() * scale.cpu().double()[:, None]
    _close(value, y, y.abs() * 2.0 ** -4 + top[:, None] * 2.0 ** -10 + 1e-5 * y.abs())


def test_many_rows_and_their_weight_gradient(cuda):
    """More rows than groups of the backward grid: every group has several."""
    import graphcuda_b200 as gc
    for shape in ((50_001, 24), (20_011, 96), (3001, 2056)):
        x, r, w = _inputs(shape, BF16, F32)
        dy = torch.randn(shape, generator=torch.Generator().manual_seed(3)).to(BF16)
        leaves = [t.to(cuda).requires_grad_() for t in (x, w, r)]
        y, _ = gc.rms_norm(leaves[0], leaves[1], leaves[2])
        dx, dw, dr = torch.autograd.grad(y, leaves, dy.to(cuda))
        h, c, _ = _exact(x, r, w, 1e-6)
        hat = h * c
        _close(dw, (dy.double() * hat).sum(0), 2e-5 * (dy.double() * hat).abs().sum(0))
        gw = dy.double() * w.double()
        d = c * (gw - hat * (gw * hat).mean(1, keepdim=True))
        _close(dr, d, SUM * c * (gw.abs() + hat.abs() * (gw * hat).abs().mean(1, keepdim=True)) + HALF[F32] * d.abs())
        again = torch.autograd.grad(gc.rms_norm(leaves[0], leaves[1], leaves[2])[0], leaves, dy.to(cuda))
        assert all(torch.equal(a, b) for a, b in zip((dx, dw, dr), again))


def test_layouts(cuda):
    """Slices with another pitch, bases that are not aligned, columns that are not contiguous, broadcast rows."""
    import graphcuda_b200 as gc
    big, wbig = torch.randn(37, 300, device=cuda), torch.randn(300, device=cuda)
    wide = torch.randn(256, 37, device=cuda)
    for x, r, w in ((big[:, 8:264], big[:, 16:272], wbig[:256]), (big[:, 3:259], big[:, 44:300], wbig[1:257]),
                    (wide.t(), big[:, :256], wbig[:256]), (big[:1, :256].expand(37, 256), big[:, :256], wbig[:256]),
                    (big[:, :256], wide.t(), wbig[::1][:256])):
        x, r, w = (t.detach().requires_grad_() for t in (x, r, w))
        y, h = gc.rms_norm(x, w, r)
        ref = [t.detach().clone().contiguous().requires_grad_() for t in (x, r, w)]
        y2, h2 = gc.rms_norm(ref[0], ref[2], ref[1])
        _close(y, y2.detach().cpu().double(), SUM * y2.detach().cpu().double().abs())
        assert torch.equal(h, h2)
        dy = torch.randn(256, 37, device=cuda).t()
        for a, b in zip(torch.autograd.grad(y, (x, r, w), dy), torch.autograd.grad(y2, (ref[0], ref[1], ref[2]), dy.contiguous())):
            _close(a, b.cpu().double(), 1e-5 * b.cpu().double().abs().max())


def test_rows_of_zeros_infinities_and_nan(cuda):
    import graphcuda_b200 as gc
    x = torch.randn(8, 256)
    x[1] = 0
    x[2, 5] = float("inf")
    x[3, 7] = float("nan")
    x[4] = 1e-30  # the square underflows: eps decides
    x[5] *= 1e15
    x[6] = 0
    x[6, 3] = -0.5
    w = torch.ones(256)
    y = gc.rms_norm(x.to(cuda), w.to(cuda)).cpu()
    ref = _exact(x, None, w, 1e-6)[2]
    assert torch.equal(y[1], torch.zeros(256))
    assert torch.isnan(y[3]).all() and torch.isnan(y[2, 5])
    for i in (0, 4, 5, 6):
        _close(y[i], ref[i], SUM * ref[i].abs() + 1e-38)
    y8, scale = gc.rms_norm_fp8(x.to(cuda), w.to(cuda))
    value = (y8.float() * scale[:, None]).cpu()
    assert torch.equal(value[1], torch.zeros(256)) and float(scale[1]) == 0
    assert not torch.isfinite(value[2]).all() and torch.isnan(value[3]).any()
    for i in (0, 5, 6):
        _close(value[i], ref[i], ref[i].abs() * 0.0626 + float(scale[i]) * 2.0 ** -10)


def test_empty(cuda):
    import graphcuda_b200 as gc
    for shape in ((0, 16), (5, 0), (0, 0)):
        x, r = torch.zeros(shape, device=cuda, requires_grad=True), torch.zeros(shape, device=cuda, requires_grad=True)
        w = torch.ones(shape[1], device=cuda, requires_grad=True)
        y, h = gc.rms_norm(x, w, r)
        assert y.shape == h.shape == x.shape
        dx, dr, dw = torch.autograd.grad(y.sum() + h.sum(), (x, r, w))
        assert dx.shape == x.shape and torch.equal(dw, torch.zeros_like(w))
        with torch.no_grad():
            y8, s = gc.rms_norm_fp8(x, w)
        assert y8.shape == x.shape and s.shape == (shape[0],)


def test_gradient_against_differences(cuda):
    """Central differences of sum(y dy) + sum(h ds) along random directions: step 1e-2, error of the third order under 1e-3
    of the slope's scale, rounding 1e-6 / 1e-2."""
    import graphcuda_b200 as gc
    g = torch.Generator().manual_seed(5)
    x, r, dy, ds = (torch.randn(6, 48, generator=g).to(cuda) for _ in range(4))
    w = (1 + 0.2 * torch.randn(48, generator=g)).to(cuda)

    def value(*t):
        with torch.no_grad():
            y, h = gc.rms_norm(t[0], t[2], t[1], eps=0.1)
        return ((y * dy).double().sum() + (h * ds).double().sum()).item()

    leaves = [t.clone().requires_grad_() for t in (x, r, w)]
    grads = torch.autograd.grad(gc.rms_norm(leaves[0], leaves[2], leaves[1], eps=0.1), leaves, (dy, ds))
    for which in range(3):
        d = torch.randn(leaves[which].shape, generator=g).to(cuda)
        args = [[t + s * 1e-2 * d if i == which else t for i, t in enumerate((x, r, w))] for s in (1, -1)]
        slope = (value(*args[0]) - value(*args[1])) / 2e-2
        expect = (grads[which] * d).double().sum().item()
        assert abs(slope - expect) < 2e-3 * (float(grads[which].norm() * d.norm()) + 1)


def test_only_what_is_needed(cuda):
    """One output unused, one input without a gradient."""
    import graphcuda_b200 as gc
    x, r, w = (t.to(cuda) for t in _inputs((20, 96), BF16, F32))
    full = [t.clone().requires_grad_() for t in (x, r, w)]
    y, h = gc.rms_norm(full[0], full[2], full[1])
    dy = torch.randn(20, 96, device=cuda).to(BF16)
    both = torch.autograd.grad(y, full, dy)
    for need in range(1, 8):
        part = [t.clone().requires_grad_(bool(need >> i & 1)) for i, t in enumerate((x, r, w))]
        y, h = gc.rms_norm(part[0], part[2], part[1])
        y.backward(dy)
        for i in range(3):
            assert torch.equal(part[i].grad, both[i]) if need >> i & 1 else part[i].grad is None
    y, h = gc.rms_norm(full[0], full[2], full[1])
    dx, dr, dw = torch.autograd.grad(h, full, torch.ones_like(h))
    assert torch.equal(dr, torch.ones_like(r)) and torch.equal(dx, torch.ones_like(x)) and not dw.any()


def test_stream_graph_and_trace(cuda):
    import graphcuda_b200 as gc
    x, r, w = (t.to(cuda) for t in _inputs((700, 256), BF16, BF16))
    expect = gc.rms_norm(x, w, r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = gc.rms_norm(x, w, r)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, expect))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, h = gc.rms_norm(x, w, r)
    x2 = torch.randn_like(x)
    expect2 = gc.rms_norm(x2, w, r)
    x.copy_(x2)
    graph.replay()
    assert torch.equal(y, expect2[0]) and torch.equal(h, expect2[1])
    for grad in (False, True):
        model = _Model(r, grad).to(cuda)
        with torch.set_grad_enabled(grad):
            traced = torch.jit.trace(model, (x,), check_trace=False)
            a = torch.randn_like(x)
            y, h = traced(a)
            expect = model(a)
        assert torch.equal(y, expect[0]) and torch.equal(h, expect[1])
        if grad:
            of = lambda t: torch.autograd.grad(t, model.norm.weight, torch.ones_like(t))[0]  # noqa: E731
            assert torch.equal(of(y), of(expect[0]))


class _Model(torch.nn.Module):
    def __init__(self, residual, grad):
        import graphcuda_b200 as gc
        super().__init__()
        self.norm = gc.RMSNorm(residual.size(1)).requires_grad_(grad)
        self.register_buffer("residual", residual)

    def forward(self, x):
        return self.norm(x, self.residual)


def test_module(cuda):
    import graphcuda_b200 as gc
    m = gc.RMSNorm(64, out_dtype=BF16).to(cuda)
    assert list(m.state_dict()) == ["weight"]
    x = torch.randn(5, 64, device=cuda)
    assert m(x).dtype == BF16 and m(x, x)[1].dtype == F32
    with torch.no_grad():
        assert m.fp8(x, x)[0].dtype == torch.float8_e4m3fn


def test_refusals(cuda):
    import graphcuda_b200 as gc
    x, w = torch.randn(4, 32, device=cuda), torch.ones(32, device=cuda)
    for bad in (lambda: gc.rms_norm(x.cpu(), w), lambda: gc.rms_norm(x, w.cpu()), lambda: gc.rms_norm(x.half(), w),
                lambda: gc.rms_norm(x, w.bfloat16()), lambda: gc.rms_norm(x, w[:31]), lambda: gc.rms_norm(x[0], w),
                lambda: gc.rms_norm(x, w, x[:3]), lambda: gc.rms_norm(x, w, x.cpu()),
                lambda: gc.rms_norm(x, w, x.bfloat16()), lambda: gc.rms_norm(x, w, eps=-1.0),
                lambda: gc.rms_norm(x, w, out_dtype=torch.float16),
                lambda: gc.rms_norm_fp8(x.requires_grad_(), w)):
        with pytest.raises(RuntimeError):
            bad()
    y = gc.rms_norm(x, w)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(y.sum(), x, create_graph=True)
    with fw.dual_level(), pytest.raises(RuntimeError, match="jvp"):
        gc.rms_norm(fw.make_dual(x.detach(), torch.ones_like(x)), w)
