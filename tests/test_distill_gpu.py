"""Distillation loss against its formula in 64 bits.

Tolerances.  A probability comes from one exponential (2^-21 with its argument's rounding, whose effect x 2^-x stays below 2^-22)
over a sum whose chain has at most some 40 terms (40 x 2^-24): 4e-6 of the gradient's factor, and the output's own rounding,
eps / 2 of the value.  A row's loss is a mean of differences of logarithms, each exact to 2^-21 of the largest one that occurs,
and of the list's sums (k x 2^-24)."""
import pytest
import torch

import graphcuda_b200 as gc

pytestmark = pytest.mark.gpu
DEV = "cuda"


def formula(logits, top, index, mask, temperature, scale):
    """(loss, dlogits, largest difference of logarithms) in float64."""
    z = torch.log_softmax(logits.double() / temperature, 1)
    C = z.size(1)
    there = (index >= 0) & (index < C) & (top != -torch.inf)
    counts = there.any(1)
    if mask is not None:
        counts &= mask.bool()
    loss, d, most = 0.0, torch.zeros_like(z), 1.0
    for r in counts.nonzero()[:, 0].tolist():
        c, t = index[r][there[r]].long(), top[r][there[r]].double() / temperature
        log_p = torch.log_softmax(t, 0)
        p = log_p.exp()
        term = log_p - z[r][c]
        loss = loss + torch.where(p > 0, p * term, 0.0).sum()
        finite = term[term.isfinite()]
        if finite.numel():
            most = max(most, float(finite.abs().max()), float((t.max() - t).max()), float((z[r].max() - z[r][c])[term.isfinite()].max()))
        row = z[r].exp()
        row.index_add_(0, c, -p)
        d[r] = row
    return loss * temperature ** 2 * scale, d * (temperature * scale), most


def check(logits, top, index, mask=None, temperature=1.0, scale=0.37, grad=1.0):
    x = logits.detach().requires_grad_()
    loss = gc.distill_loss(x, top, index, mask, temperature, scale=scale)
    (dx,) = torch.autograd.grad(loss, x, torch.tensor(grad, device=DEV))
    want, dwant, most = formula(logits, top, index, mask, temperature, scale)
    rows, k = max(1, logits.size(0)), top.size(1)
    tol = temperature ** 2 * scale * rows * most * (2 ** -20 + k * 2.0 ** -24) + abs(float(want)) * 2.0 ** -23
    assert abs(float(loss.detach()) - float(want)) <= tol, (loss, want, tol)
    dwant = dwant * grad
    eps = torch.finfo(logits.dtype).eps
    err = (dx.double() - dwant).abs() - (dwant.abs() * eps / 2 * 1.001 + abs(grad) * temperature * scale * 4e-6)
    assert dx.dtype == logits.dtype and dx.shape == logits.shape and float(err.max()) <= 0, float(err.max())
    with torch.no_grad():
        assert abs(float(gc.distill_loss(logits, top, index, mask, temperature, scale=scale)) - float(want)) <= tol
    return loss, dx


def make(M, C, k, seed=0, dtype=torch.float32, top_dtype=None, index_dtype=torch.int64, distinct=True):
    g = torch.Generator(device=DEV).manual_seed(seed)
    logits = (2 * torch.randn(M, C, generator=g, device=DEV)).to(dtype)
    teacher = 0.5 * logits.float() + 2 * torch.randn(M, C, generator=g, device=DEV)
    if distinct and k <= C:
        top, index = teacher.topk(k, 1)
    else:
        index = torch.randint(0, C, (M, k), generator=g, device=DEV)
        top = teacher.gather(1, index)
    return logits, top.to(top_dtype or dtype), index.to(index_dtype)


SIZES = [(1, 1, 1), (1, 2, 1), (3, 2, 2), (5, 7, 3), (33, 47, 8), (100, 256, 32), (100, 256, 33), (64, 257, 5), (9, 1000, 300),
         (130, 31, 31), (3, 4096, 64), (5, 4097, 1024), (2, 200_001, 50), (1, 8193, 7), (147, 12_345, 10), (149, 12_345, 10),
         (300, 5000, 10), (2708, 7, 3),
         # one pass: in rings of short segments and of long ones, rows of whole segments and not, up to the ring's length
         (148, 4096, 5), (700, 4099, 40), (601, 12_288, 3), (200, 18_432, 100), (149, 18_433, 256), (310, 50_688, 64), (150, 101_376, 12), (150, 101_377, 12)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,C,k", SIZES)
def test_loss_and_gradient(M, C, k, dtype):
    check(*make(M, C, k, seed=M + C, dtype=dtype), temperature=2.0)


@pytest.mark.parametrize("top_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("index_dtype", [torch.int64, torch.int32])
@pytest.mark.parametrize("temperature", [0.5, 1.0, 7.0])
def test_types_and_temperatures(top_dtype, index_dtype, temperature):
    for C, k in ((40, 5), (700, 40), (9000, 100)):
        check(*make(20, C, k, seed=C, top_dtype=top_dtype, index_dtype=index_dtype), temperature=temperature, grad=-2.5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,C", [(40, 10), (40, 47), (40, 300), (40, 5001), (40, 20_000), (160, 9000), (150, 40_001)])
def test_lists_with_holes_and_rows_that_do_not_count(M, C, dtype):
    k = 8
    logits, top, index = make(M, C, k, seed=C, dtype=dtype)
    g = torch.Generator(device=DEV).manual_seed(C)
    index[torch.rand(M, k, generator=g, device=DEV) < 0.4] = -1
    index[3] = -1                       # nothing
    index[4] = C + 5                    # no classes
    index[5, 0], index[5, 1] = 2 ** 40, -2 ** 40
    top[6] = -torch.inf                 # no entries either
    top[7, ::2] = -torch.inf
    mask = torch.rand(M, generator=g, device=DEV) < 0.7
    mask[3:9] = True
    mask[10], mask[11] = False, False
    logits[10] = torch.nan              # what is not selected may hold anything
    top[11] = torch.inf
    logits[3] = torch.nan
    top[index < 0] = torch.nan
    for m in (mask, mask.to(torch.uint8)):
        x = logits.detach().requires_grad_()
        loss = gc.distill_loss(x, top, index, m, 3.0, scale=0.1)
        (dx,) = torch.autograd.grad(loss, x)
        keep = torch.ones(M, dtype=torch.bool, device=DEV)
        keep[[3, 10, 11]] = False
        want, dwant, _ = formula(logits[keep], top[keep], index[keep], mask[keep], 3.0, 0.1)
        assert abs(float(loss.detach()) - float(want)) <= 9 * 0.1 * M * 30 * 2.0 ** -19
        err = (dx[keep].double() - dwant).abs() - (dwant.abs() * torch.finfo(dtype).eps / 2 * 1.001 + 0.3 * 4e-6)
        assert float(err.max()) <= 0
        assert not dx[~keep].any() and not dx[6].any() and not dx[4].any() and not dx[~mask].any()


@pytest.mark.parametrize("M,C,k", [(17, 12, 9), (17, 200, 32), (17, 3000, 200), (17, 7000, 1000), (150, 9000, 300), (150, 45_000, 1024)])
def test_an_index_more_than_once(M, C, k):
    logits, top, index = make(M, C, k, seed=k, distinct=False)
    index[0] = 5
    index[1, ::2] = 1
    check(logits, top, index, temperature=2.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,C", [(12, 30), (12, 1000), (12, 30_011), (148, 6000), (148, 30_011)])
def test_masked_classes(M, C, dtype):
    """Classes at -inf or at the type's lowest value have no probability; a row of lowest values alone is uniform."""
    logits, top, index = make(M, C, 4, seed=C, dtype=dtype)
    low = torch.finfo(dtype).min
    g = torch.Generator(device=DEV).manual_seed(1)
    out = torch.rand(M, C, generator=g, device=DEV) < 0.5
    out.scatter_(1, index, False)
    logits[:6][out[:6]] = -torch.inf
    logits[6:][out[6:]] = low
    logits[11] = low
    for temperature in (0.25, 1.0, 4.0):
        check(logits, top, index, temperature=temperature)
    logits[0, index[0, 1]] = -torch.inf  # a class that the teacher gives a probability: infinitely far
    x = logits.detach().requires_grad_()
    loss = gc.distill_loss(x, top, index)
    (dx,) = torch.autograd.grad(loss, x)
    assert float(loss.detach()) == float("inf") and bool(dx.isfinite().all())


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("M,C", [(6, 30), (6, 1000), (6, 30_011), (148, 6000), (148, 30_011)])
def test_what_is_no_number_stays_in_its_row(M, C, bad):
    logits, top, index = make(M, C, 4, seed=C)
    logits[2, C // 2] = bad
    top[4, 1] = bad
    x = logits.detach().requires_grad_()
    loss = gc.distill_loss(x, top, index)
    (dx,) = torch.autograd.grad(loss, x)
    assert torch.isnan(loss)
    fine = [r for r in range(M) if r not in (2, 4)]
    assert bool(dx[fine].isfinite().all())
    assert torch.isnan(dx[2]).any() and torch.isnan(dx[4]).any()
    want = formula(logits[fine], top[fine], index[fine], None, 1.0, 1 / M)[1]
    assert float((dx[fine].double() - want).abs().max()) <= 1 / M * 4e-6 + 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_alignment(dtype):
    for M, C in ((11, 47), (11, 301), (11, 9001), (148, 9001), (148, 20_000)):
        logits, top, index = make(M, C, 6, seed=C, dtype=dtype)
        for before, after in ((0, 1), (0, 3), (1, 0), (3, 2), (8, 8)):
            wide = torch.full((M, before + C + after), torch.nan, device=DEV, dtype=dtype)
            wide[:, before:before + C] = logits
            check(wide[:, before:before + C], top, index)
        check(logits.t().contiguous().t(), top.t().contiguous().t(), index.t().contiguous().t())
        wide_top, wide_index = torch.cat((top, top), 1), torch.cat((index, index), 1)
        check(logits, wide_top[:, 3:9], wide_index[:, 3:9])
        check(logits[:1], top[:1], index[:1])
        check(logits[::2], top[::2], index[::2])


def test_padded_logits_give_a_gradient_that_the_layer_below_takes_as_it_is():
    buf = torch.randn(64, 48, device=DEV)
    logits, top, index = buf[:, :47], *make(64, 47, 5)[1:]
    before = gc._lib.host.zero_padded_count()
    _, dx = check(logits, top, index)
    assert dx.stride() == (48, 1) and gc._lib.host.zero_padded_count() == before + 1
    whole = gc._lib.host.zero_padded_base(dx, 48)
    assert whole is not None and not whole[:, 47].any()


def test_agrees_with_differences():
    logits, top, index = make(3, 11, 4, seed=5)
    x = logits.detach().requires_grad_()
    (dx,) = torch.autograd.grad(gc.distill_loss(x, top, index, None, 1.5, scale=1.0), x)
    h = 2.0 ** -5
    for r in range(3):
        for c in range(11):
            step = torch.zeros_like(logits)
            step[r, c] = h
            up, down = (float(gc.distill_loss(logits + s * step, top, index, None, 1.5, scale=1.0)) for s in (1, -1))
            # third derivative of a log-sum-exp below 1 / T; the losses themselves are off by 1e-5 each
            assert abs((up - down) / (2 * h) - float(dx[r, c])) <= h * h / 6 * 1.5 + 2e-5 / h


def test_default_scale_and_nothing_to_do():
    logits, top, index = make(10, 20, 3)
    mask = torch.zeros(10, dtype=torch.bool, device=DEV)
    mask[:4] = True
    assert torch.equal(gc.distill_loss(logits, top, index, mask), gc.distill_loss(logits, top, index, mask, scale=0.25))
    assert torch.equal(gc.distill_loss(logits, top, index), gc.distill_loss(logits, top, index, scale=0.1))
    for args in ((logits[:0], top[:0], index[:0]), (logits, top[:, :0], index[:, :0]), (logits, top, index, mask & False)):
        x = args[0].detach().requires_grad_()
        loss = gc.distill_loss(x, *args[1:])
        (dx,) = torch.autograd.grad(loss, x)
        assert float(loss) == 0 and dx.shape == x.shape and not dx.any()


@pytest.mark.parametrize("M,C,k", [(200, 9000, 20), (300, 47, 8), (300, 47, 40), (70, 1000, 200), (9, 4096, 1000)])
def test_a_gradient_that_is_not_one_and_gradients_of_their_own(M, C, k):
    """Rows may have their gradient before the loss's is known; what is handed out is changed by no later backward pass."""
    logits, top, index = make(M, C, k, distinct=C != 1000)
    x = logits.detach().requires_grad_()
    loss = gc.distill_loss(x, top, index, None, 2.0)
    first = torch.autograd.grad(loss, x, retain_graph=True)[0]
    kept = first.clone()
    first.zero_()
    third = torch.autograd.grad(loss, x, torch.tensor(3.0, device=DEV), retain_graph=True)[0]
    again = torch.autograd.grad(loss, x)[0]
    assert not first.any() and torch.equal(again, kept)
    assert float((third - 3 * kept).abs().max()) <= float(kept.abs().max()) * 3 * 2.0 ** -22
    check(logits, top, index, temperature=2.0, grad=3.0)
    half = logits.detach().requires_grad_()
    (0.5 * gc.distill_loss(half, top, index, None, 2.0)).backward()
    assert float((half.grad - 0.5 * kept).abs().max()) <= float(kept.abs().max()) * 2.0 ** -22


@pytest.mark.parametrize("M,C,k", [(500, 20_000, 30), (200, 60_000, 30), (1000, 47, 8), (300, 1000, 300), (60, 6000, 600)])
def test_same_bits_every_time_and_backward_twice(M, C, k):
    logits, top, index = make(M, C, k, dtype=torch.bfloat16, distinct=k < 100)
    x = logits.detach().requires_grad_()
    losses, grads = [], []
    for _ in range(3):
        loss = gc.distill_loss(x, top, index)
        losses.append(loss.detach())
        grads += [torch.autograd.grad(loss, x, retain_graph=True)[0], torch.autograd.grad(loss, x)[0]]
    assert all(torch.equal(l, losses[0]) for l in losses) and all(torch.equal(g, grads[0]) for g in grads)


def test_refusals():
    logits, top, index = make(4, 10, 3)
    for args in ((logits.double(), top, index), (logits.half(), top, index), (logits[0], top, index), (logits, top[:3], index[:3]),
                 (logits, top, index[:, :2]), (logits, top, index.float()), (logits, top.cpu(), index), (logits, top, index.cpu()),
                 (logits[:, :0], top, index), (logits, top, index, torch.ones(3, dtype=torch.bool, device=DEV)),
                 (logits, top, index, torch.ones(4, device=DEV)), (logits, top, index, torch.ones(4, dtype=torch.bool)),
                 (logits, top, index, None, 0.0), (logits, top, index, None, -1.0), (logits, top, index, None, float("nan"))):
        with pytest.raises(RuntimeError):
            gc.distill_loss(*args, scale=1.0)
    with pytest.raises(RuntimeError, match="1024"):
        gc.distill_loss(logits, top[:, :1].expand(4, 1025), index[:, :1].expand(4, 1025))
    with pytest.raises(RuntimeError, match="teacher"):
        gc.distill_loss(logits, top.detach().requires_grad_(), index)
    x = logits.detach().requires_grad_()
    loss = gc.distill_loss(x, top, index)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(loss, x, create_graph=True)
    loss = gc.distill_loss(x.clone(), top, index)
    top.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()


def test_recorded_in_a_graph_and_on_another_stream():
    logits, top, index = make(300, 9000, 12)
    x = logits.detach().requires_grad_()
    want = gc.distill_loss(x, top, index, None, 2.0)
    (dwant,) = torch.autograd.grad(want, x)
    want = want.detach()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = logits.detach().requires_grad_()
        got = gc.distill_loss(y, top, index, None, 2.0, scale=1 / 300)
        (dgot,) = torch.autograd.grad(got, y)
        got = got.detach()
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(dgot, dwant)
    graph = torch.cuda.CUDAGraph()
    z = torch.zeros_like(logits).requires_grad_()
    with torch.cuda.graph(graph):
        loss = gc.distill_loss(z, top, index, None, 2.0, scale=1 / 300)
        (dz,) = torch.autograd.grad(loss, z)
        loss = loss.detach()
    for _ in range(2):
        with torch.no_grad():
            z.copy_(logits)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(loss, want) and torch.equal(dz, dwant)
        with torch.no_grad():
            z.zero_()
        graph.replay()


def test_traced():
    logits, top, index = make(30, 50, 5)
    f = torch.jit.trace(lambda z: gc.distill_loss(z, top, index, None, 2.0, scale=0.1), (logits,), check_trace=False)
    other = make(30, 50, 5, seed=9)[0].requires_grad_()
    plain = other.detach().requires_grad_()
    got, want = f(other), gc.distill_loss(plain, top, index, None, 2.0, scale=0.1)
    assert torch.equal(got, want)
    assert torch.equal(torch.autograd.grad(got, other)[0], torch.autograd.grad(want, plain)[0])
