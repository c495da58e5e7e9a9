"""The gated block where its kept G and U leave the range of fp16, around the boundary of its form for few rows, and where
offsets pass 32 bits.

Tolerances are those of a bf16 product: u = 2^-8 for the rounding of an operand, of which sums pick up u / sqrt(3) times the
root of their summed squares per operand at most; six of those (3.5 u) are allowed, and u of the output itself.  G and U are
kept to 2^-11 or better of the largest of 32 columns, an eighth of u."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -8 * 1.01


def _randn(*s, seed=0):
    return torch.randn(*s, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def _gradients(x, w_in, w_out, dy, act="relu"):
    import graphcuda_b200 as gc
    leaves = [t.detach().requires_grad_() for t in (x, w_in, w_out)]
    y = gc.gated_ffn(*leaves, activation=act)
    return (y.detach(), *torch.autograd.grad(y, leaves, dy))


def _relu_exact(x, w_in, w_out, dy):
    """Outputs, gradients and their tolerances with relu, whose products scale with their operands at any magnitude."""
    x, w_in, w_out, dy = (t.double() for t in (x, w_in, w_out, dy))
    h = w_out.size(0)
    g, u = x @ w_in[:, :h], x @ w_in[:, h:]
    a, slope = g.clamp(min=0), (g > 0).double()
    hid, da = a * u, dy @ w_out.t()
    dgu = torch.cat((da * u * slope, da * a), 1)
    # G and U are off by 2^-11 of the largest of their 32 columns: what that changes dG and dU by
    pad = -h % 32
    top = lambda t: torch.nn.functional.pad(t.abs(), (0, pad)).view(len(t), -1, 32).amax(2).repeat_interleave(32, 1)[:, :h]  # noqa: E731
    e = dgu.abs() + torch.cat((da.abs() * top(u) * slope, da.abs() * top(g)), 1) / 8
    # a G below 2^-25 may be kept as zero beside one above 2^-10: relu's slope there is either
    either = torch.cat((da * u * (g.abs() < top(g) * 2.0 ** -15), torch.zeros_like(da)), 1).abs()
    loose = (0.0, either @ w_in.abs().t(), x.abs().t() @ either, 0.0)
    got = (hid @ w_out, dgu @ w_in.t(), x.t() @ dgu, hid.t() @ dy)
    noise = (hid.square() @ w_out.square(), e.square() @ w_in.square().t(), x.square().t() @ e.square(), hid.square().t() @ dy.square())
    return got, [U * (r.abs() + 3.5 * n.sqrt()) + o + 1e-37 for r, n, o in zip(got, noise, loose)]


def _check(got, ref, tol):
    for k, (a, b, t) in enumerate(zip(got, ref, tol)):
        over = (a.double() - b).abs() - t
        assert float(over.max()) <= 0, (k, float(over.max()), int((over > 0).sum()))


@pytest.mark.parametrize("shape", [(1, 32, 40, 24), (5, 64, 100, 64), (8, 264, 72, 40), (200, 64, 100, 64), (300, 256, 1000, 256),
                                   (150, 640, 264, 96)], ids=str)
@pytest.mark.parametrize("power", [(40, 0), (0, 40), (30, -30), (-30, 30), (-30, -30), (-16, 18)], ids=str)
def test_magnitudes_far_from_one(cuda, shape, power):
    """G and U of 2^40 and 2^-30, in all of a row, and beside each other in neighbouring rows and columns."""
    from graphcuda_b200 import ops
    m, d, h, o = shape
    x, w_in, w_out = _randn(m, d), _randn(d, 2 * h, seed=1) / d ** 0.5, _randn(h, o, seed=2) / h ** 0.5
    dy = _randn(m, o, seed=3)
    w_in[:, :h] *= 2.0 ** power[0]
    w_in[:, h:] *= 2.0 ** power[1]
    x[::2] *= 2.0 ** 10
    w_in[:, 32:64] *= 2.0 ** -12
    t = [v.bfloat16() for v in (x, w_in, w_out, dy)]
    _check(_gradients(*t), *_relu_exact(*t))
    ops.check_gemm_flag(cuda)


@pytest.mark.parametrize("m", [1, 3, 9, 33, 64])
@pytest.mark.parametrize("shape", [(25, 68, 2336), (128, 76, 1416), (264, 1032, 40), (2048, 1111, 513)], ids=str)
def test_few_rows_round_their_outputs_alone(cuda, m, shape):
    """Up to 64 rows, A and the gradients of G and U are kept to 16 bits and more (two bf16 numbers): the outputs' own rounding is
    left, and, of gradients, what G and U are off by, 2^-12 of the largest of 32 columns."""
    d, h, o = shape
    t = [v.bfloat16() for v in (_randn(m, d), _randn(d, 2 * h, seed=1) / d ** 0.5, _randn(h, o, seed=2) / h ** 0.5, _randn(m, o, seed=3))]
    x, w_in, w_out, dy = (v.double() for v in t)
    g, u = x @ w_in[:, :h], x @ w_in[:, h:]
    a, slope = g.clamp(min=0), (g > 0).double()
    hid, da = a * u, dy @ w_out.t()
    dgu = torch.cat((da * u * slope, da * a), 1)
    pad = -h % 32
    top = lambda v: torch.nn.functional.pad(v.abs(), (0, pad)).view(m, -1, 32).amax(2).repeat_interleave(32, 1)[:, :h]  # noqa: E731
    e = torch.cat((da.abs() * top(u) * slope, da.abs() * top(g)), 1) / 8
    either = torch.cat((da * u * (g.abs() < top(g) * 2.0 ** -15), torch.zeros_like(da)), 1).abs()
    ref = (hid @ w_out, dgu @ w_in.t(), x.t() @ dgu, hid.t() @ dy)
    # two bf16 numbers: 2^-17 of the value; fp32 sums add as much
    parts = (hid.abs() @ w_out.abs(), dgu.abs() @ w_in.abs().t(), x.abs().t() @ dgu.abs(), hid.abs().t() @ dy.abs())
    noise = (0.0, (e.square() @ w_in.square().t()).sqrt(), (x.square().t() @ e.square()).sqrt(), 0.0)
    loose = (0.0, either @ w_in.abs().t(), x.abs().t() @ either, 0.0)
    tol = [U * (r.abs() + 3.5 * n) + 2.0 ** -16 * p + o + 1e-37 for r, n, p, o in zip(ref, noise, parts, loose)]
    _check(_gradients(*t), ref, tol)


@pytest.mark.parametrize("m", [1, 6, 200])
@pytest.mark.parametrize("h", [40, 100, 1032])
@pytest.mark.parametrize("value", [float("inf"), float("nan"), 2.0 ** 120])
def test_a_column_does_not_change_its_neighbours(cuda, m, h, value):
    """An infinite, NaN or huge G in one column, and a U whose first columns are huge: dWin of all other columns is what it is
    without them.  (The other G are above 65504, where fp16 without an exponent would be infinite.)"""
    d = o = 64
    x, w_in, w_out = _randn(m, d), _randn(d, 2 * h, seed=1) * 2.0 ** 14, _randn(h, o, seed=2) / h ** 0.5
    x[:, 0] = 1.0
    w_in[1:, [3, h]] = 0.0
    w_in[0, [3, h]] = 1.0
    t = [v.bfloat16() for v in (x, w_in, w_out, _randn(m, o, seed=3))]
    ref, tol = _relu_exact(*t)
    t[1][0, 3] = value  # G's column 3
    t[1][0, h] = value  # U's column 0, which lies behind G's last
    got = _gradients(*t)[2]
    keep = torch.ones(2 * h, dtype=torch.bool, device=cuda)
    finite = value == 2.0 ** 120
    keep[[0, 3, h, h + 3]] = False
    if finite:  # the 31 columns beside them share their exponent: 2^120 leaves nothing of them
        keep[:32] = keep[h:h + 32] = False
    _check([got[:, keep]], [ref[2][:, keep]], [tol[2][:, keep]])


@pytest.mark.parametrize("m", [1, 2, 7, 8, 9, 31, 33])
@pytest.mark.parametrize("shape", [(64, 96, 40), (1024, 4096, 1024), (1025, 1111, 513)], ids=str)
def test_few_rows(cuda, m, shape):
    """One row and a few, which may take another path than nine: forward alone, with what it keeps, in 16 and in 8 bits."""
    import graphcuda_b200 as gc
    d, h, o = shape
    x, w_in, w_out, dy = (v.bfloat16() for v in (_randn(m, d), _randn(d, 2 * h, seed=1) / d ** 0.5, _randn(h, o, seed=2) / h ** 0.5,
                                                 _randn(m, o, seed=3)))
    ref, tol = _relu_exact(x, w_in, w_out, dy)
    got = _gradients(x, w_in, w_out, dy)
    _check(got, ref, tol)
    _check([gc.gated_ffn(x, w_in, w_out, activation="relu")], ref[:1], tol[:1])
    x8, xs = gc.quantize_weight_fp8(x.t())
    w8, ws = gc.quantize_weight_fp8(w_in)
    got8 = gc.gated_ffn_fp8(x8, xs, w8, ws, w_out, activation="relu")
    gu = (x8.double() * xs.double()[:, None]) @ (w8.double() * ws.double()[:, None]).t()
    hid = gu[:, :h].clamp(min=0) * gu[:, h:]
    y = hid @ w_out.double()
    _check([got8], [y], [U * (y.abs() + 3.5 * (hid.square() @ w_out.double().square()).sqrt()) + 1e-37])
    # the rows of a larger call are those of a smaller one, whichever path it takes, up to rounding
    if m > 1:
        _check([gc.gated_ffn(x[1:2], w_in, w_out, activation="relu")], [ref[0][1:2]], [tol[0][1:2]])


@pytest.fixture
def give_memory_back():
    """What is kept across calls (scratch) must not come to lie in this test's large blocks, which could not be freed then."""
    yield
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


def test_offsets_beyond_32_bits(cuda, give_memory_back):
    """3.3 G elements of x and dy from first to last, 3.2 G of what is kept: the last rows are those of a call on them alone."""
    import graphcuda_b200 as gc
    m, pitch, d, h, o = 1_600_000, 2048, 64, 1000, 64
    wide = torch.zeros(m, pitch, dtype=torch.bfloat16, device=cuda)
    x = wide[:, 1024:1024 + d]
    tail = _randn(300, d).bfloat16()
    x[-300:] = tail
    w_in, w_out = ((_randn(d, 2 * h, seed=1) / 8).bfloat16().requires_grad_(), (_randn(h, o, seed=2) / 32).bfloat16().requires_grad_())
    dy = _randn(300, o, seed=3).bfloat16()
    wide_dy = torch.zeros(m, pitch, dtype=torch.bfloat16, device=cuda)[:, :o]
    wide_dy[-300:] = dy
    xr = x.detach().requires_grad_()
    y = gc.gated_ffn(xr, w_in, w_out)
    full = torch.autograd.grad(y, (xr, w_in, w_out), wide_dy)
    tr = tail.detach().requires_grad_()
    yt = gc.gated_ffn(tr, w_in, w_out)
    part = torch.autograd.grad(yt, (tr, w_in, w_out), dy)
    assert not y[:-300].any() and not full[0][:-300].any()
    # sums are cut elsewhere; the outputs' own rounding is 2^-9 either way
    for a, b in ((y[-300:], yt), (full[0][-300:], part[0]), *zip(full[1:], part[1:])):
        assert float((a - b).detach().float().abs().max()) <= 2.0 ** -7 * float(b.detach().float().abs().max())


@pytest.mark.parametrize("m", [1, 6, 9, 200, 3000])
@pytest.mark.parametrize("scale", [0, 20, -20])
def test_relu_of_next_to_nothing(cuda, m, scale):
    """A G of 2^-30 beside ones about 1 (times a power of two) is positive, one of zero and one below are not: their gradients are
    those of relu all the same."""
    d, h, o = 64, 96, 64
    x, w_in, w_out = _randn(m, d), _randn(d, 2 * h, seed=1) / 8, _randn(h, o, seed=2) / 8
    x[:, 0] = 1.0
    for column, value in ((1, 2.0 ** -30), (34, -2.0 ** -30), (70, 0.0), (95, 2.0 ** -40)):
        w_in[:, column] = 0.0
        w_in[0, column] = value
    w_in[:, :h] *= 2.0 ** scale
    t = [v.bfloat16() for v in (x, w_in, w_out, _randn(m, o, seed=3))]
    got = _gradients(*t)
    x, w_in, w_out, dy = (v.double() for v in t)
    g, u, da = x @ w_in[:, :h], x @ w_in[:, h:], dy @ w_out.t()
    dg = da * u * (g > 0)
    tol = U * ((x.t() @ dg).abs() + 3.5 * (x.square().t() @ (dg * 1.2).square()).sqrt()) + 1e-37
    cols = [1, 34, 70, 95]
    over = (got[2][:, cols].double() - (x.t() @ dg)[:, cols]).abs() - tol[:, cols]
    assert float(over.max()) <= 0
    assert bool((got[2][:, [34, 70]] == 0).all()) and bool((got[2][:, [1, 95]] != 0).any())


def test_large_workspaces_go_back(cuda):
    """What a call needs between its kernels is not held when it has ended, nor is what it kept for a backward pass that is over."""
    t = [v.bfloat16() for v in (_randn(60_000, 64), _randn(64, 1024, seed=1) / 8, _randn(512, 64, seed=2) / 16, _randn(60_000, 64, seed=3))]
    before = torch.cuda.memory_allocated()
    got = _gradients(*t)
    del got
    assert torch.cuda.memory_allocated() - before < 64 << 20


def test_buffers_are_as_large_as_asked_for(cuda):
    """Nothing is written behind what is kept and behind the workspace."""
    from graphcuda_b200 import _lib
    lib = _lib.lib()
    for m, h in ((1, 1), (8, 31), (33, 33), (129, 1000), (257, 40)):
        d = o = 64
        x, w_in, w_out = _randn(m, d).bfloat16(), _randn(d, 2 * h, seed=1).bfloat16(), _randn(h, o, seed=2).bfloat16()
        kept = torch.full((lib.gc_gated_ffn_saved_bytes(m, h) + 4096,), 0x5A, dtype=torch.uint8, device=cuda)
        ws_bytes = lib.gc_gated_ffn_workspace_bytes(m, d, h, o, 0)
        ws = torch.full((ws_bytes + 4096,), 0x5A, dtype=torch.uint8, device=cuda)
        y = torch.empty(m, o, dtype=torch.bfloat16, device=cuda)
        rc = lib.gc_gated_ffn_forward_bf16(x.data_ptr(), d, w_in.data_ptr(), 2 * h, w_out.data_ptr(), o, m, d, h, o,
                                           _lib.ACT_SILU, y.data_ptr(), o, kept.data_ptr(), ws.data_ptr(), ws_bytes,
                                           torch.cuda.current_stream().cuda_stream)
        assert rc == 0, lib.gc_last_error()
        assert bool((kept[-4096:] == 0x5A).all()) and bool((ws[ws_bytes:] == 0x5A).all())
