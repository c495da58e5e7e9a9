"""Rows by group times a weight per group, and their gradients, against 64 bits.

Tolerances.  The result's rounding is half a step of bf16 (2^-8 of it).  Sums are fp32; the tensor core truncates, which costs a sum of n
terms at most (n / 16 + 16) x 2^-23 of the sum of magnitudes (an accumulation takes 16 products at once), and parts of
16,384 rows and fewer are added to 2^-23 each."""
import pytest
import torch

import graphcuda_b200 as gc

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = 2.0 ** -8


def near(got, want, magnitude, terms):
    err = (got.double() - want).abs() - (want.abs() * HALF * 1.001 + magnitude * (terms / 16 + 16) * 2.0 ** -23)
    assert got.dtype == torch.bfloat16 and got.shape == want.shape
    assert not got.numel() or float(err.max()) <= 0, float(err.max())


def reference(x, w, dy, bounds):
    """y, dx, dw and their sums of magnitudes."""
    X, W, D = x.double(), w.double(), dy.double()
    out = [torch.zeros(dy.shape, dtype=torch.float64, device=DEV), torch.zeros(x.shape, dtype=torch.float64, device=DEV),
           torch.zeros(w.shape, dtype=torch.float64, device=DEV)]
    mag = [torch.zeros_like(t) for t in out]
    for g in range(w.size(0)):
        r = slice(bounds[g], bounds[g + 1])
        if bounds[g] >= bounds[g + 1]:
            continue
        for to, f in ((out, lambda t: t), (mag, torch.abs)):
            to[0][r] = f(X[r]) @ f(W[g])
            to[1][r] = f(D[r]) @ f(W[g]).t()
            to[2][g] = f(X[r]).t() @ f(D[r])
    return out, mag


def inputs(sizes, k, n, before=0, behind=0, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed + k * 31 + n)
    bounds = [before]
    for s in sizes:
        bounds.append(bounds[-1] + s)
    rows = bounds[-1] + behind
    randn = lambda *s: torch.randn(*s, generator=gen, device=DEV).bfloat16()  # noqa: E731
    return randn(rows, k), (randn(len(sizes), k, n) / max(k, 1) ** 0.5).bfloat16(), randn(rows, n), bounds


def step(x, w, offsets, dy):
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    y = gc.grouped_linear(x, w, offsets)
    return (y.detach(),) + torch.autograd.grad(y, (x, w), dy)


def check(x, w, dy, bounds, given=None):
    offsets = torch.tensor(bounds if given is None else given, dtype=torch.int32, device=DEV)
    got = step(x, w, offsets, dy)
    want, mag = reference(x, w, dy, bounds)
    k, n = w.shape[1:]
    longest = max([b - a for a, b in zip(bounds, bounds[1:])], default=0)
    for g, t, m, terms in zip(got, want, mag, (k, n, longest)):
        near(g, t, m, terms)
    with torch.no_grad():
        assert torch.equal(gc.grouped_linear(x, w, offsets), got[0])
    return got


GROUPS = [[1], [0, 3, 0], [5, 64, 1, 63, 65], [128, 0, 127, 129], [300, 7], [1000], [2] * 40, [0] * 33 + [10] + [0] * 40, [256, 512, 100]]


@pytest.mark.parametrize("sizes", GROUPS)
@pytest.mark.parametrize("k,n", [(8, 8), (64, 64), (100, 47), (33, 200), (256, 256), (264, 520), (1, 1)])
def test_step(sizes, k, n):
    check(*inputs(sizes, k, n))


@pytest.mark.parametrize("sizes,k,n", [([2600] * 20, 256, 256), ([2000, 0, 4500, 2603] * 5, 200, 256), ([700] * 30 + [9000], 264, 250),
                                       ([40] * 70, 512, 512), ([1300, 500], 1024, 1024), ([130, 3], 2048, 1024)])
def test_parts_and_tiles_of_all_sorts(sizes, k, n):
    """Groups cut into parts and groups left whole, tiles of each shape."""
    check(*inputs(sizes, k, n))


@pytest.mark.parametrize("before,behind", [(0, 9), (3, 0), (70, 300)])
@pytest.mark.parametrize("k,n", [(64, 128), (47, 100), (256, 512)])
def test_rows_of_no_group(before, behind, k, n):
    x, w, dy, bounds = inputs([20, 0, 200, 1], k, n, before, behind)
    x[:before], x[bounds[-1]:], dy[:before], dy[bounds[-1]:] = torch.nan, torch.inf, torch.inf, torch.nan
    got = check(x, w, dy, bounds)
    for t in got[:2]:
        assert not t[:before].any() and not t[bounds[-1]:].any()


@pytest.mark.parametrize("sizes,k,n", [([40_000, 0, 3, 20_000], 64, 48), ([70_001], 128, 128), ([1, 30_000, 2000], 300, 260),
                                       ([5000] * 9, 256, 256), ([3000, 5000], 2048, 1024)])
def test_many_rows(sizes, k, n):
    check(*inputs(sizes, k, n))


def test_many_groups():
    gen = torch.Generator().manual_seed(3)
    check(*inputs(torch.randint(0, 40, (700,), generator=gen).tolist(), 64, 72))
    check(*inputs(torch.randint(0, 3, (300,), generator=gen).tolist(), 136, 40, 1, 5))


@pytest.mark.parametrize("k,n", [(2048, 2048), (520, 4000)])
def test_few_rows_for_many_weights(k, n):
    check(*inputs([1, 0, 2, 1, 0, 0, 7, 3], k, n))


def test_what_is_no_number_stays_in_its_group():
    x, w, dy, bounds = inputs([70, 100, 30], 96, 80)
    fine = step(x, w, torch.tensor(bounds, dtype=torch.int32, device=DEV), dy)
    for bad in (torch.nan, torch.inf):
        x2, w2, dy2 = x.clone(), w.clone(), dy.clone()
        x2[75:80], dy2[100], w2[1, 5] = bad, bad, bad
        got = step(x2, w2, torch.tensor(bounds, dtype=torch.int32, device=DEV), dy2)
        for g, f in zip(got[:2], fine[:2]):
            assert torch.equal(g[:70], f[:70]) and torch.equal(g[170:], f[170:])
        assert torch.equal(got[2][0], fine[2][0]) and torch.equal(got[2][2], fine[2][2])
        assert not got[0][75].isfinite().any() and not got[1][100].isfinite().any() and not got[2][1].isfinite().all()


@pytest.mark.parametrize("given,read", [([0, 5, 3, 90], [0, 5, 5, 60]), ([-4, 10, 10, 60], [0, 10, 10, 60]), ([70, 80, 90, 99], [60, 60, 60, 60]),
                                        ([30, 20, 10, 0], [30, 30, 30, 30])])
def test_offsets_that_are_none(given, read):
    """Read as the nearest that are: inside the rows, not decreasing."""
    x, w, dy, _ = inputs([20, 20, 20], 64, 40)
    check(x, w, dy, read, given)


def test_strides_and_alignment():
    x, w, dy, bounds = inputs([37, 0, 90, 12], 72, 56)
    offsets = torch.tensor(bounds, dtype=torch.int32, device=DEV)
    want = step(x, w, offsets, dy)

    def inside(t, off, more):
        wide = torch.full(t.shape[:-1] + (t.shape[-1] + off + more,), torch.nan, device=DEV, dtype=t.dtype)
        view = wide[..., off:off + t.shape[-1]]
        view.copy_(t)
        return view

    for off, more in ((0, 8), (8, 0), (3, 1), (0, 5)):
        got = step(inside(x, off, more), inside(w, off, more), offsets, inside(dy, off, more))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    turned = (x.t().contiguous().t(), w.transpose(1, 2).contiguous().transpose(1, 2), offsets, dy.t().contiguous().t())
    assert all(torch.equal(a, b) for a, b in zip(step(*turned), want))
    every = torch.stack((w, w), 1).flatten(0, 1)[::2]
    assert all(torch.equal(a, b) for a, b in zip(step(x, every, offsets, dy), want))
    spread = torch.stack((offsets, offsets), 1).flatten()[::2]
    assert all(torch.equal(a, b) for a, b in zip(step(x, w, spread, dy), want))
    y = gc.grouped_linear(x.detach().requires_grad_(), w, offsets)
    (dx,) = torch.autograd.grad(y.sum(), [y.grad_fn.next_functions[0][0].variable])  # an expanded gradient
    assert torch.equal(dx, step(x, w, offsets, torch.ones_like(dy))[1])


def test_only_the_gradients_that_are_asked_for():
    x, w, dy, bounds = inputs([30, 50], 64, 40)
    offsets = torch.tensor(bounds, dtype=torch.int32, device=DEV)
    _, dx, dw = step(x, w, offsets, dy)
    a = x.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(gc.grouped_linear(a, w, offsets), a, dy)[0], dx)
    b = w.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(gc.grouped_linear(x, b, offsets), b, dy)[0], dw)


def test_agrees_with_differences():
    """A step of one element: the loss is linear in x and in w, so a difference is the gradient up to the results' rounding."""
    x, w, dy, bounds = inputs([3, 0, 4], 16, 8)
    offsets = torch.tensor(bounds, dtype=torch.int32, device=DEV)
    y, dx, dw = step(x, w, offsets, dy)
    loss = lambda a, b: float((gc.grouped_linear(a, b, offsets).double() * dy.double()).sum())  # noqa: E731
    slack = float((y.double().abs() + 8).mul(dy.double().abs()).sum()) * 2 * HALF
    for at in ((0, 0), (2, 15), (6, 7)):
        up = x.clone()
        up[at] += 64
        h = float(up[at] - x[at])
        assert abs((loss(up, w) - loss(x, w)) / h - float(dx[at])) <= abs(float(dx[at])) * 3 * HALF + slack * 9 / h
    for at in ((0, 3, 2), (2, 15, 7)):
        up = w.clone()
        up[at] += 64
        h = float(up[at] - w[at])
        assert abs((loss(x, up) - loss(x, w)) / h - float(dw[at])) <= abs(float(dw[at])) * 3 * HALF + slack * 9 / h
    assert not dw[1].any()


def test_nothing_to_do():
    for sizes, k, n in (([0, 0], 16, 8), ([], 16, 8), ([3, 4], 0, 8), ([3, 4], 16, 0), ([3, 4], 0, 0)):
        x, w, dy, bounds = inputs(sizes, k, n, behind=0 if sizes else 5)
        y, dx, dw = step(x, w, torch.tensor(bounds, dtype=torch.int32, device=DEV), dy)
        assert y.shape == dy.shape and dx.shape == x.shape and dw.shape == w.shape
        assert not y.any() and not dx.any() and not dw.any()


def test_same_bits_every_time():
    x, w, dy, bounds = inputs([3000, 1, 7000, 250], 256, 136)
    offsets = torch.tensor(bounds, dtype=torch.int32, device=DEV)
    first = step(x, w, offsets, dy)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(step(x, w, offsets, dy), first))


def test_refusals():
    x, w, dy, bounds = inputs([3, 4], 16, 8)
    off = torch.tensor(bounds, dtype=torch.int32, device=DEV)
    for args in ((x.float(), w, off), (x, w.float(), off), (x[0], w, off), (x, w[0], off), (x[:, :8], w, off), (x, w, off.long()), (x, w, off[:2]),
                 (x, w, off.cpu()), (x, w.cpu(), off), (x, w, off[None])):
        with pytest.raises(RuntimeError):
            gc.grouped_linear(*args)
    a = x.detach().requires_grad_()
    y = gc.grouped_linear(a, w, off)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(y, a, dy, create_graph=True)
    y = gc.grouped_linear(a, w, off)
    off.add_(0)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(y, a, dy)


def test_recorded_in_a_graph_with_other_groups_every_time_and_on_another_stream():
    x, w, dy, bounds = inputs([300, 20, 0, 500], 128, 104)
    other = [0, 10, 400, 400, 820]
    off = torch.tensor(bounds, dtype=torch.int32, device=DEV)
    want = step(x, w, off, dy)
    want_other = step(x, w, torch.tensor(other, dtype=torch.int32, device=DEV), dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x, w, off, dy)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    held = off.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(x, w, held, dy)
    for _ in range(2):
        for o, t in ((bounds, want), (other, want_other)):
            held.copy_(torch.tensor(o, dtype=torch.int32, device=DEV))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, t))


def test_traced():
    x, w, dy, bounds = inputs([30, 50], 64, 40)
    off = torch.tensor(bounds, dtype=torch.int32, device=DEV)
    traced = torch.jit.trace(lambda a: gc.grouped_linear(a, w, off), (x,), check_trace=False)
    a, b = dy.new_tensor(x.flip(0).tolist()).requires_grad_(), x.flip(0).detach().requires_grad_()
    got, want = traced(a), gc.grouped_linear(b, w, off)
    assert torch.equal(got, want) and torch.equal(torch.autograd.grad(got, a, dy)[0], torch.autograd.grad(want, b, dy)[0])


def test_module_trains_with_masters():
    torch.manual_seed(0)
    x, w, dy, bounds = inputs([30, 50], 64, 40)
    off = torch.tensor(bounds, dtype=torch.int32, device=DEV)
    layer = gc.GroupedLinear(64, 40, 2).to(DEV)
    opt = gc.FusedAdamW(layer.parameters(), lr=1e-2)
    before = layer.weight.detach().clone()
    layer(x, off).backward(dy)
    assert torch.equal(layer.weight.grad, step(x, before, off, dy)[2])
    opt.step()
    assert not torch.equal(layer.weight, before)
