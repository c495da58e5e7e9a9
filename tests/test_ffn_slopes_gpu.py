"""relu's slope in the gated block: one or the other only where the sign of G is within a float32 sum's rounding; and a few rows
through a recorded call.

Tolerances as in test_ffn_range_gpu.py: u = 2^-8 for an operand's rounding, u / sqrt(3) times the root of the summed squares for
sums, six of those (3.5 u), u of the output itself; G and U are kept to 2^-11 of the largest of their 32 columns, an eighth of u."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -8 * 1.01


def _randn(*s, seed=0):
    return torch.randn(*s, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


@pytest.mark.parametrize("m", [1, 6, 50, 200, 3000])
@pytest.mark.parametrize("shape", [(64, 96, 64), (100, 267, 47), (256, 1032, 40)], ids=str)
@pytest.mark.parametrize("spread", [0, 10, 16, 24, 40])
def test_slopes_of_columns_of_all_sizes(cuda, m, shape, spread):
    """Columns of G that are powers of two apart, up to 2^-spread of their neighbours: what is positive has slope one, what is
    not has zero.  The rows of dWin that belong to G say so, column by column."""
    import graphcuda_b200 as gc
    d, h, o = shape
    x, w_in, w_out, dy = _randn(m, d), _randn(d, 2 * h, seed=1) / d ** 0.5, _randn(h, o, seed=2) / h ** 0.5, _randn(m, o, seed=3)
    w_in[:, :h] *= 2.0 ** -(torch.arange(h, device=cuda) * 7 % (spread + 1)).float()
    x, w_in, w_out, dy = (t.bfloat16() for t in (x, w_in, w_out, dy))
    leaves = [t.requires_grad_() for t in (x, w_in, w_out)]
    got, = torch.autograd.grad(gc.gated_ffn(*leaves, activation="relu"), leaves[1:2], dy)
    x, w_in, w_out, dy = (t.detach().double() for t in (x, w_in, w_out, dy))
    g, u, da = x @ w_in[:, :h], x @ w_in[:, h:], dy @ w_out.t()
    dg = da * u * (g > 0)
    pad = -h % 32
    top = torch.nn.functional.pad(u.abs(), (0, pad)).view(m, -1, 32).amax(2).repeat_interleave(32, 1)[:, :h]
    e = dg.abs() + da.abs() * top * (g > 0) / 8
    # a sum of d products in float32 is off by d 2^-23 of their magnitudes at most: the sign is open below that
    open_sign = (da * u * (g.abs() <= d * 2.0 ** -23 * (x.abs() @ w_in[:, :h].abs()))).abs()
    ref = x.t() @ dg
    tol = U * (ref.abs() + 3.5 * (x.square().t() @ e.square()).sqrt()) + x.abs().t() @ open_sign + 1e-37
    assert float(((got[:, :h].double() - ref).abs() - tol).max()) <= 0


@pytest.mark.parametrize("m", [1, 2, 4, 8])
def test_few_rows_recorded(cuda, m):
    """The second of the two launches begins before the first has ended: replayed, with new inputs, as called."""
    import graphcuda_b200 as gc
    d, h, o = 256, 1024, 256
    make = lambda s: [t.bfloat16() for t in (_randn(m, d, seed=s), _randn(d, 2 * h, seed=s + 1) / 16, _randn(h, o, seed=s + 2) / 32)]  # noqa: E731
    static = make(0)
    w8, ws = gc.quantize_weight_fp8(static[1])
    x8, xs = gc.quantize_weight_fp8(static[0].t())

    def calls():
        with torch.no_grad():
            return gc.gated_ffn(*static), gc.gated_ffn_fp8(x8, xs, w8, ws, static[2])

    calls()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = calls()
    for s in (10, 20, 30):
        for a, b in zip(static, make(s)):
            a.copy_(b)
        for a, b in zip((w8, ws, x8, xs), (*gc.quantize_weight_fp8(static[1]), *gc.quantize_weight_fp8(static[0].t()))):
            a.copy_(b)
        for _ in range(3):
            graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, calls()))
