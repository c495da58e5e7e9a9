"""The 8-bit forms as a server has them: inside a trace, frozen beside a model that trains on, and without a gradient."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _poison(*like):
    """What fresh memory holds from here on."""
    junk = [torch.full((t.numel() * t.element_size() // 4 + 64,), float("nan"), device=t.device) for t in like for _ in range(4)]
    del junk


class _Traced(torch.nn.Module):
    """Norm and block with a residual that is no input of the trace."""

    def __init__(self, norm, ffn, residual):
        super().__init__()
        self.norm, self.ffn, self.residual = norm, ffn, residual

    def forward(self, x):
        got = self.norm.fp8(x, self.residual)
        return (self.ffn(got[0], got[1]), *got)


@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("rows", [1, 7, 300])
def test_traced_eight_bit_forms_run_on_new_inputs(cuda, rows, add):
    import graphcuda_b200 as gc
    torch.manual_seed(0)
    norm, ffn = gc.RMSNorm(96).to(cuda), gc.GatedFFN(96, 160, 40).to(cuda).for_serving()
    xs = [torch.randn(rows, 96, device=cuda).bfloat16() for _ in range(3)]
    model = _Traced(norm, ffn, torch.randn(rows, 96, device=cuda) if add else None)
    with torch.no_grad():
        traced = torch.jit.trace(model, (xs[0],), check_trace=False)
        for x in xs:
            expect = model(x)
            _poison(*expect)
            got = traced(x)
            assert len(got) == len(expect) == (4 if add else 3)
            assert all(a.dtype == b.dtype and torch.equal(a.float(), b.float()) for a, b in zip(got, expect))


def test_a_trace_has_no_gradient_either(cuda):
    """What raises outside of a trace raises while it is taken."""
    import graphcuda_b200 as gc
    x, w = torch.randn(4, 32, device=cuda), torch.ones(32, device=cuda, requires_grad=True)
    w8, ws = gc.quantize_weight_fp8(torch.randn(32, 48, device=cuda))
    w_out = torch.randn(24, 16, device=cuda).bfloat16().requires_grad_()
    x8, xs = gc.rms_norm_fp8(x, w.detach())
    with pytest.raises(RuntimeError, match="no gradient"):
        torch.jit.trace(lambda t: gc.rms_norm_fp8(t, w)[1], (x,), check_trace=False)
    with pytest.raises(RuntimeError, match="no gradient"):
        torch.jit.trace(lambda s: gc.gated_ffn_fp8(x8, s, w8, ws, w_out), (xs,), check_trace=False)


def _setup(cuda, seed=0):
    from graphcuda_b200 import normalized_adjacency, synth
    from graphcuda_b200.models import ResidualGCN
    n, f, classes = 400, 40, 5
    edges = synth.symmetrize(synth.preferential_attachment_edges(n, 4 * n, seed))
    adj = normalized_adjacency(edges.to(cuda), n, symmetric=True)
    torch.manual_seed(seed)
    model = ResidualGCN(f, 48, 3, classes, hidden=80).to(cuda)
    return adj, model, torch.randn(n, f, device=cuda), torch.randint(0, classes, (n,), device=cuda)


def test_traced_served_model_runs_on_new_inputs(cuda):
    adj, model, X, _ = _setup(cuda)
    served = model.for_serving()

    class Answer(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.model = served

        def forward(self, x):
            return self.model(x, adj, log_softmax=False)

    with torch.no_grad():
        traced = torch.jit.trace(Answer(), (X,), check_trace=False)
        for seed in range(3):
            x = torch.randn(X.shape, generator=torch.Generator().manual_seed(seed)).to(cuda)
            expect = served(x, adj, log_softmax=False)
            _poison(expect, x)
            assert torch.equal(traced(x), expect)


def test_served_model_is_that_of_its_moment(cuda):
    """The source trains on: the served model answers as it did."""
    from graphcuda_b200 import FusedAdamW, log_softmax_nll_loss
    adj, model, X, y = _setup(cuda, seed=1)
    opt = FusedAdamW(model.parameters(), lr=1e-2)
    served = model.for_serving()
    before = served(X, adj, log_softmax=False)
    for _ in range(3):
        opt.zero_grad(set_to_none=True)
        log_softmax_nll_loss(model(X, adj, log_softmax=False), y, scale=1.0 / len(y)).backward()
        opt.step()
    assert torch.equal(served(X, adj, log_softmax=False), before)
    later = model.for_serving()(X, adj, log_softmax=False)
    assert not torch.equal(later, before)
    # nor does what is done to the served model reach its source
    kept = [p.detach().clone() for p in model.parameters()]
    for t in (*served.parameters(), *served.buffers()):
        t.data.zero_()
    assert all(torch.equal(a, b) for a, b in zip(kept, model.parameters()))
    assert not any(p.requires_grad for p in served.parameters())


def test_served_model_holds_one_set_of_weights(cuda):
    """Smaller than its source, by half of the first products' weights: nothing is kept that no call reads."""
    _, model, _, _ = _setup(cuda)
    served = model.for_serving()
    size = lambda m: sum(t.numel() * t.element_size() for t in (*m.parameters(), *m.buffers()))  # noqa: E731
    w_in = sum(b.ffn.w_in.numel() for b in model.blocks)
    scales = sum(b.ffn.w_in.size(1) * 4 for b in model.blocks)
    assert size(served) == size(model) - w_in + scales
    again = served.for_serving()
    assert all(torch.equal(a.float(), b.float()) for a, b in zip(again.state_dict().values(), served.state_dict().values()))


def test_an_eight_bit_operand_with_a_gradient_is_refused(cuda):
    """A cast to 8 bits is differentiable to torch: the block would drop what comes back."""
    import graphcuda_b200 as gc
    x = torch.randn(4, 32, device=cuda, requires_grad=True)
    w = torch.randn(32, 48, device=cuda, requires_grad=True)
    w8, ws = gc.quantize_weight_fp8(w)
    w_out, ones = torch.randn(24, 16, device=cuda).bfloat16(), torch.ones(4, device=cuda)
    x8, wx8 = x.to(torch.float8_e4m3fn), w.t().to(torch.float8_e4m3fn)
    assert x8.requires_grad and wx8.requires_grad and not w8.requires_grad
    for a, b in ((x8, w8), (x8.detach(), wx8)):
        with pytest.raises(RuntimeError, match="no gradient"):
            gc.gated_ffn_fp8(a, ones, b, ws, w_out)
        with torch.no_grad():
            gc.gated_ffn_fp8(a, ones, b, ws, w_out)
