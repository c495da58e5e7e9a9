"""Products with weights of 4 bits against their formulas in 64 bits.

Tolerances.  Sums are fp32, of which the tensor core's chain and the groups' together have at most in / 32 + 32 terms, each off by 2^-23
of the sum of magnitudes.  The result's own rounding is half a step of bf16, 2^-8 of it.  Above 128 rows a weight's rounding
is another 2^-8 of it at worst; in the block above 64 rows those of both weights and of the hidden row, to fp16, are 2^-11, and what
fp16 cannot hold of a hidden row beside its bound."""
import pytest
import torch

import graphcuda_b200 as gc
from graphcuda_b200.models import ResidualGCN

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = 2.0 ** -8


def weight(k, n, group=64, zeros=False, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + k * 7 + n)
    codes = torch.randint(0, 16, (k, n), generator=g, device=DEV, dtype=torch.uint8)
    groups = -(-k // group)
    scale = (torch.rand(groups, n, generator=g, device=DEV) + 0.5).bfloat16() / max(k, 1) ** 0.5 / 5
    zero = torch.randint(0, 16, (groups, n), generator=g, device=DEV, dtype=torch.uint8) if zeros else None
    return gc.Int4Weight.from_codes(codes, scale.bfloat16(), zero, group=group)


def rows(m, k, seed=0):
    return torch.randn(m, k, generator=torch.Generator(device=DEV).manual_seed(seed + m + k), device=DEV).bfloat16()


def near(got, want, slack):
    err = (got.double() - want).abs() - (want.abs() * HALF * 1.001 + slack)
    assert float(err.max()) <= 0, float(err.max())


def check_linear(x, w):
    got = gc.linear_int4(x, w)
    assert got.shape == (x.size(0), w.out_features) and got.dtype == torch.bfloat16
    X, W = x.double(), w.dequantize().double()
    slack = (X.abs() @ W.abs()) * ((w.in_features / 32 + 32) * 2.0 ** -23 + (HALF if x.size(0) > 128 else 0))
    near(got, X @ W, slack + 1e-30)
    return got


ROWS = [1, 2, 4, 5, 8, 9, 16, 17, 32, 33, 64, 65, 96, 97, 128, 129]


@pytest.mark.parametrize("m", ROWS)
@pytest.mark.parametrize("k,n", [(1, 1), (40, 17), (128, 16), (129, 300), (1433, 47), (2048, 512), (5000, 40)])
def test_linear(m, k, n):
    for group, zeros in ((32, True), (64, False), (128, True)):
        check_linear(rows(m, k), weight(k, n, group, zeros))


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
def test_wide_layers(group, zeros):
    for m, k, n in ((1, 2048, 8192), (5, 8192, 2050), (16, 16_384, 1024), (40, 1024, 9000), (120, 4096, 700), (1, 64, 40_000)):
        check_linear(rows(m, k), weight(k, n, group, zeros))


def test_zero_points_are_exact_however_large_the_inputs():
    """A code equal to its zero point has no say, whatever it is multiplied with."""
    w = gc.Int4Weight.from_codes(torch.full((256, 32), 11, dtype=torch.uint8, device=DEV),
                                 torch.ones(4, 32, dtype=torch.bfloat16, device=DEV),
                                 torch.full((4, 32), 11, dtype=torch.uint8, device=DEV), group=64)
    for m in (1, 20, 100, 300):
        x = rows(m, 256) * 1e30
        assert not gc.linear_int4(x, w).any()


def act64(name, g):
    if name == "silu":
        return g * torch.sigmoid(g), torch.sigmoid(g) * (1 + g * (1 - torch.sigmoid(g)))
    if name == "gelu":
        cdf = torch.special.erfc(-g * 0.5 ** 0.5) / 2
        return g * cdf, cdf + g * torch.exp(-g * g / 2) * 0.3989422804014327
    return g.clamp(min=0), (g > 0).double()


def check_block(x, w_in, w_out, act):
    got = gc.gated_ffn_int4(x, w_in, w_out, activation=act)
    m, h = x.size(0), w_out.in_features
    X, Wi, Wo = x.double(), w_in.dequantize().double(), w_out.dequantize().double()
    G, U = (X @ Wi).split(h, 1)
    a, slope = act64(act, G)
    hidden = a * U
    many = 2.0 ** -11 if m > 64 else 0
    # of the first product, the activation (1e-5 of its input), the hidden row (16 bits, or a step of fp16), the second
    first = (X.abs() @ Wi.abs()) * ((w_in.in_features / 32 + 32) * 2.0 ** -23 + many)
    eg, eu = first.split(h, 1)
    # slopes of the activations are below 1.13, and near g the one at g moves by at most 1.1 times the distance
    dh = (slope.abs() + 1.1 * eg) * eg * U.abs() + a.abs() * eu + eg * eu * 1.13 + 1e-5 * G.abs() * U.abs()
    dh += (hidden.abs() + dh) * (many or 2.0 ** -16)
    if many:  # half of fp16's smallest number, 2^-25, where 2^15 stands for the bound: |x|^2 D w^2 in powers of two (x by up to 32 more), 15 steps of the largest scale for w
        dh += 2.0 ** -26 * X.square().sum(1, keepdim=True) * w_in.in_features * Wi.abs().max() ** 2
        # the bound is 2^-85 at least, so that 2^-24 of fp16 stands for 2^-124; the hidden row's own range, fp32's, ends at 2^-126
        dh += 2.0 ** -124
    second = (hidden.abs() @ Wo.abs()) * ((h / 32 + 32) * 2.0 ** -23 + many)
    near(got, hidden @ Wo, second + dh @ Wo.abs() * (1 + HALF) + 1e-30)
    return got, hidden @ Wo


@pytest.mark.parametrize("m", ROWS)
@pytest.mark.parametrize("d,h,o", [(1, 1, 1), (40, 24, 16), (100, 267, 47), (256, 1024, 256), (129, 15, 300)])
def test_block(m, d, h, o):
    for act, group, zeros in (("silu", 32, True), ("gelu", 64, False), ("relu", 128, True)):
        check_block(rows(m, d), weight(d, 2 * h, group, zeros), weight(h, o, group, zeros, seed=1), act)


def test_wide_blocks_and_mixed_groups():
    check_block(rows(1, 2048), weight(2048, 16_384, 64), weight(8192, 2048, 32, True), "silu")
    check_block(rows(7, 1024), weight(1024, 2 * 4001, 128, True), weight(4001, 520, 64), "gelu")


def rms(got, want):
    return float((got.double() - want).norm() / want.norm())


def test_errors_on_average():
    """Of roundings spread evenly over a step: 2^-8 / sqrt(3) each at most."""
    one = HALF / 3 ** 0.5
    x, w = rows(2000, 512), weight(512, 256)
    want = x.double() @ w.dequantize().double()
    assert rms(gc.linear_int4(x[:128], w), want[:128]) <= one and rms(gc.linear_int4(x, w), want) <= one * 2 ** 0.5
    wi, wo = weight(512, 1024, 32), weight(512, 200, 32, seed=1)
    for m, n in ((64, 1), (2000, 1.09)):  # result; and both halves of the first weight (1.5 for the slope), the second's, the hidden row's, an eighth each
        assert rms(*check_block(x[:m], wi, wo, "silu")) <= one * n ** 0.5


def test_strides_and_alignment():
    for k in (48, 200, 333):
        w, wi, wo = weight(k, 40), weight(k, 48), weight(24, 30)
        for m in (1, 6, 20, 90, 250):
            wide = torch.full((m, k + 9), torch.nan, device=DEV, dtype=torch.bfloat16)
            for off in (0, 1, 8, 9):
                wide[:] = torch.nan
                x = wide[:, off:off + k]
                x.copy_(rows(m, k))
                assert torch.equal(check_linear(x, w), gc.linear_int4(x.contiguous(), w))
                assert torch.equal(gc.gated_ffn_int4(x, wi, wo), gc.gated_ffn_int4(x.contiguous(), wi, wo))
            check_linear(rows(m, k).t().contiguous().t(), w)
            check_linear(rows(1, k).expand(m, k), w)


def test_what_is_no_number_stays_in_its_row():
    w, wi, wo = weight(200, 40, zeros=True), weight(200, 96), weight(48, 24)
    for m in (3, 12, 100, 250):
        x = rows(m, 200)
        fine_l, fine_b = gc.linear_int4(x, w), gc.gated_ffn_int4(x, wi, wo)
        for bad in (float("nan"), float("inf")):
            y = x.clone()
            y[1, 77] = bad
            for f, fine in ((lambda t: gc.linear_int4(t, w), fine_l), (lambda t: gc.gated_ffn_int4(t, wi, wo), fine_b)):
                got = f(y)
                keep = [i for i in range(m) if i != 1]
                assert torch.equal(got[keep], fine[keep]) and not got[1].isfinite().any()


def test_nothing_to_do():
    w = weight(64, 24)
    assert gc.linear_int4(rows(0, 64), w).shape == (0, 24)
    assert gc.linear_int4(rows(3, 64), weight(64, 0)).shape == (3, 0)
    for m in (3, 20, 300):
        none = gc.linear_int4(rows(m, 0), weight(0, 24))
        assert none.shape == (m, 24) and not none.any()
        assert not gc.gated_ffn_int4(rows(m, 0), weight(0, 48), weight(24, 8)).any()
        assert not gc.gated_ffn_int4(rows(m, 64), weight(64, 0), weight(0, 8)).any()
    assert gc.gated_ffn_int4(rows(0, 64), weight(64, 48), weight(24, 8)).shape == (0, 8)


def test_same_bits_every_time_and_in_any_company():
    w, wi, wo = weight(3000, 700), weight(3000, 1000), weight(500, 260)
    for m in (1, 8, 64, 100, 300):
        x = rows(m, 3000)
        for f in (lambda t: gc.linear_int4(t, w), lambda t: gc.gated_ffn_int4(t, wi, wo)):
            first = f(x)
            assert all(torch.equal(f(x), first) for _ in range(4))


def test_refusals():
    x, w = rows(3, 64), weight(64, 48)
    for bad in (x.float(), x[0], x[:, :63], x.cpu()):
        with pytest.raises(RuntimeError):
            gc.linear_int4(bad, w)
        with pytest.raises(RuntimeError):
            gc.gated_ffn_int4(bad, w, weight(24, 8))
    for wo in (weight(48, 8), weight(23, 8)):
        with pytest.raises(RuntimeError):
            gc.gated_ffn_int4(x, w, wo)
    with pytest.raises(RuntimeError):
        gc.linear_int4(x, w.cpu())
    for change in (lambda t: setattr(t, "records", t.records[:2]), lambda t: setattr(t, "records", t.records.to(torch.int8)),
                   lambda t: setattr(t, "group", 32), lambda t: setattr(t, "out_features", 480), lambda t: setattr(t, "zero_points", True)):
        t = weight(64, 48)
        change(t)
        with pytest.raises(RuntimeError, match="Int4Weight"):
            gc.linear_int4(x, t)
    with pytest.raises(RuntimeError, match="gradient"):
        gc.linear_int4(x.clone().requires_grad_(), w)
    with pytest.raises(RuntimeError, match="gradient"):
        gc.gated_ffn_int4(x.clone().requires_grad_(), w, weight(24, 8))


@pytest.mark.parametrize("m", [1, 20, 100, 300])
def test_recorded_in_a_graph_and_on_another_stream(m):
    x, w, wi, wo = rows(m, 1000), weight(1000, 300), weight(1000, 512), weight(256, 130)
    calls = (lambda t: gc.linear_int4(t, w), lambda t: gc.gated_ffn_int4(t, wi, wo))
    want = [f(x) for f in calls]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [f(x) for f in calls]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    z = torch.zeros_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [f(z) for f in calls]
    for _ in range(2):
        z.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        z.zero_()
        graph.replay()


def test_traced():
    x, w, wi, wo = rows(5, 96), weight(96, 40), weight(96, 48), weight(24, 16)
    for f in (lambda t: gc.linear_int4(t, w), lambda t: gc.gated_ffn_int4(t, wi, wo)):
        traced = torch.jit.trace(f, (x,), check_trace=False)
        y = rows(5, 96, seed=3)
        assert torch.equal(traced(y), f(y)) and not torch.equal(traced(y), f(x))


def test_a_model_served_in_4_bits():
    """The served model is the source with its blocks' weights replaced by what their codes stand for, bit for bit in its graph layers
    and within the blocks' roundings otherwise; and it keeps its own weights."""
    torch.manual_seed(0)
    n = 300
    edges = torch.randint(0, n, (2, 1500), device=DEV)
    adj = gc.normalized_adjacency(edges, n)
    x = torch.randn(n, 20, device=DEV)
    model = ResidualGCN(20, 64, 2, 7).to(DEV)
    served = model.for_serving(bits=4)
    assert served.for_serving() is served and served.bits == 4
    with pytest.raises(RuntimeError):
        served.for_serving(8)
    got = served(x, adj, log_softmax=False)
    with torch.no_grad():
        for block, other in zip(served.blocks, model.blocks):
            other.ffn.w_in.copy_(block.ffn.w_in.dequantize())
            other.ffn.w_out.copy_(block.ffn.w_out.dequantize())
        want = model(x, adj, log_softmax=False)
        assert torch.equal(served(x, adj, log_softmax=False), got)
    assert not got.requires_grad
    # two blocks' roundings, 4e-3 of a block's addition to the stream each, and no more
    assert float((got - want).norm() / want.norm()) <= 2e-2
    pred, counts = served.evaluate(x, adj, torch.zeros(n, dtype=torch.int64, device=DEV))
    assert torch.equal(pred, got.argmax(1)) and int(counts[0, 1]) == n


@pytest.mark.parametrize("x_size,in_size,out_size", [(1e-30, 1.0, 1.0), (1e18, 1e-18, 1.0), (1e-20, 1e12, 1e25), (1e10, 1e-25, 1e20), (1e30, 1e-25, 1e-5)])
def test_block_over_the_range_of_its_types(x_size, in_size, out_size):
    # rows, outputs and groups of very different sizes: many rows go through fp16 with exponents of their own
    torch.manual_seed(5)
    def sized(k, n, size):
        codes = torch.randint(0, 16, (k, n), dtype=torch.uint8, device=DEV)
        scale = size * 2.0 ** torch.randint(-6, 7, (1, n), device=DEV) * (0.5 + torch.rand(k // 32, n, device=DEV))
        return gc.Int4Weight.from_codes(codes, scale.bfloat16(), torch.randint(0, 16, scale.shape, dtype=torch.uint8, device=DEV), group=32)
    x = (torch.randn(150, 96, device=DEV) * x_size * 2.0 ** torch.randint(-20, 1, (150, 1), device=DEV)).bfloat16()
    check_block(x, sized(96, 2 * 64, in_size), sized(64, 40, out_size), "relu")
