"""Products per kind of vertex, a deep model, its answers kept and learnt by a small one, 4-bit serving: together, as one uses them.

Tolerances are beside the comparisons; a rounding to bf16 is off by 2^-8 of the value at most."""
import numpy as np
import pytest
import torch

import graphcuda_b200 as gc
from graphcuda_b200.models import GCN, ResidualGCN
from tests.test_planetoid import _write

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
HALF = 2.0 ** -8
KINDS = [130, 0, 201, 69]
N, IN, WIDTH, CLASSES, TOP = 400, 50, 64, 300, 20


class Kinds(torch.nn.Module):
    """Vertices sorted by kind, each kind with features of its own meaning."""

    def __init__(self):
        super().__init__()
        self.embed = gc.GroupedLinear(IN, WIDTH, len(KINDS))
        self.gcn = ResidualGCN(WIDTH, WIDTH, 2, CLASSES)

    def forward(self, x, offsets, adj):
        return self.gcn(self.embed(x, offsets).float(), adj, log_softmax=False)


@pytest.fixture
def graph():
    torch.manual_seed(3)
    adj = gc.normalized_adjacency(torch.randint(0, N, (2, 6 * N), device=DEV), N, symmetric=True)
    offsets = torch.tensor([0, *np.cumsum(KINDS)], dtype=torch.int32, device=DEV)
    return torch.randn(N, IN, device=DEV).bfloat16(), offsets, adj, torch.randint(0, CLASSES, (N,), device=DEV)


def test_a_small_model_learns_what_a_deep_one_answers_and_both_are_served(graph):
    x, offsets, adj, labels = graph
    teacher = Kinds().to(DEV)
    opt = gc.FusedAdamW(teacher.parameters(), lr=0.003)
    for _ in range(5):
        opt.zero_grad(set_to_none=True)
        gc.log_softmax_nll_loss(teacher(x, offsets, adj), labels).backward()
        grad = teacher.embed.weight.grad
        assert grad.dtype == torch.bfloat16 and grad[0].any() and not grad[1].any()  # the second kind has no vertex
        opt.step()
    with torch.no_grad():
        top, index = teacher(x, offsets, adj).topk(TOP)
    student = GCN([WIDTH, 16, CLASSES]).to(DEV)
    embed = gc.GroupedLinear(IN, WIDTH, len(KINDS)).to(DEV)
    opts = [gc.FusedAdam(student.parameters(), lr=0.01), gc.FusedAdamW(embed.parameters(), lr=0.003)]
    for _ in range(5):
        for o in opts:
            o.zero_grad(set_to_none=True)
        logits = student(embed(x, offsets).float(), adj, log_softmax=False)
        loss = gc.distill_loss(logits, top, index, temperature=2.0)
        loss.backward()
        q = torch.log_softmax(logits.detach().double() / 2, 1).gather(1, index)
        p = torch.softmax(top.double() / 2, 1)
        want = 4 * (p * (p.log() - q)).sum() / N
        # sums of 300 exponentials and 20 products, logarithms of size below 10: some 400 steps of 2^-24 of the parts' magnitudes
        slack = 4 * (p * (p.log().abs() + q.abs() + 1)).sum() / N * 400 * 2.0 ** -24
        assert abs(float(loss.detach()) - float(want)) <= float(slack)
        for o in opts:
            o.step()
    assert all(torch.isfinite(p).all() for m in (student, embed) for p in m.parameters())

    # 4 bits against the same model with weights that 4 bits hold: both round the norm's output, the hidden row and the two outputs
    # of each of 2 blocks to bf16, one of them the weights, twice; norms and sums pass relative errors on at their size
    served = teacher.gcn.for_serving(bits=4)
    plain = teacher.gcn
    with torch.no_grad():
        for block, small in zip(plain.blocks, served.blocks):
            for name in ("w_in", "w_out"):
                weight = getattr(small.ffn, name).dequantize()
                getattr(block.ffn, name).copy_(weight)
        h = teacher.embed(x, offsets).float()
        got, want = served(h, adj, log_softmax=False).double(), plain(h, adj, log_softmax=False).double()
    assert ((got - want).norm() / want.norm()) <= 2 * 2 * 6 * HALF
    gc.ops.check_gemm_flag(DEV)


def test_gradient_through_a_product_per_kind_and_the_loss(graph):
    x, offsets, _, labels = graph
    torch.manual_seed(4)
    w = (torch.randn(len(KINDS), IN, CLASSES, device=DEV) / IN ** 0.5).bfloat16().requires_grad_()
    xs = x.clone().requires_grad_()
    top, index = torch.randn(N, CLASSES, device=DEV).topk(TOP)
    mask = torch.rand(N, device=DEV) < 0.7
    gc.distill_loss(gc.grouped_linear(xs, w, offsets), top, index, mask, 1.5, scale=1.0).backward()
    X, W = x.double().requires_grad_(), w.detach().double().requires_grad_()
    bounds = offsets.tolist()
    Z = torch.cat([X[a:b] @ W[g] for g, (a, b) in enumerate(zip(bounds, bounds[1:]))])
    p = torch.softmax(top.double() / 1.5, 1)
    (1.5 ** 2 * (p * (p.log() - torch.log_softmax(Z / 1.5, 1).gather(1, index))).sum(1)[mask].sum()).backward()
    with torch.no_grad():
        # z is rounded: q moves by at most 2 |dz| / 1.5 of itself (and z's own sums by 64 * 2^-24); dz = 1.5 (q - p) is rounded again
        q = torch.softmax(Z / 1.5, 1)
        dz = 1.5 * (q - torch.zeros_like(Z).scatter_add_(1, index, p)) * mask[:, None]
        moved = (2 / 1.5 * Z.abs().amax(1, keepdim=True) * HALF * 1.1 + 1e-5) * 1.5 * q * mask[:, None]
        off = moved + (dz.abs() + moved) * HALF + 1e-7
        for g, (a, b) in enumerate(zip(bounds, bounds[1:])):
            slack = X[a:b].abs().T @ off[a:b]
            assert ((w.grad[g].double() - W.grad[g]).abs() <= slack * 1.01 + W.grad[g].abs() * HALF + 1e-6).all()
            slack = off[a:b] @ W[g].abs().T
            assert ((xs.grad[a:b].double() - X.grad[a:b]).abs() <= slack * 1.01 + X.grad[a:b].abs() * HALF + 1e-6).all()


def _everything(x, w, offsets, top, index, int4, block):
    leaf, weights = x.detach().requires_grad_(), w.detach().requires_grad_()
    loss = gc.distill_loss(gc.grouped_linear(leaf, weights, offsets), top, index, None, 2.0, scale=1.0)
    dx, dw = torch.autograd.grad(loss, (leaf, weights))
    return [loss.detach(), dx, dw, gc.linear_int4(x, int4), gc.gated_ffn_int4(x, *block), gc.linear_int4(x[:40], int4),
            gc.gated_ffn_int4(x[:20], *block), gc.linear_int4(x[:3], int4), gc.gated_ffn_int4(x[:3], *block)]


def _inputs(graph, seed):
    torch.manual_seed(seed)
    x, offsets = torch.randn(N, 264, device=DEV).bfloat16(), graph[1]
    weight = lambda k, n: gc.quantize_weight_int4((torch.randn(k, n, device=DEV) / k ** 0.5).bfloat16(), group=64)
    return (x, torch.randn(len(KINDS), 264, CLASSES, device=DEV).bfloat16() / 16, offsets, *torch.randn(N, CLASSES, device=DEV).topk(TOP),
            weight(264, 1000), (weight(264, 2 * 328), weight(328, 200)))


def test_two_streams_at_once_give_the_bits_of_one(graph):
    inputs = [_inputs(graph, s) for s in (1, 2)]
    want = [_everything(*i) for i in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in inputs]
    got = [[], []]
    for _ in range(10):
        for k, (i, s) in enumerate(zip(inputs, streams)):
            with torch.cuda.stream(s):
                got[k].append(_everything(*i))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for k in (0, 1) for run in got[k] for a, b in zip(run, want[k]))


def test_two_recorded_steps_replayed_at_once_give_the_bits_of_eager_ones(graph):
    inputs = [_inputs(graph, s) for s in (1, 2)]
    want = [_everything(*i) for i in inputs]
    graphs, got = [], []
    for i in inputs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got.append(_everything(*i))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in inputs]
    torch.cuda.synchronize()
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))


def test_script_serves_in_4_bits_and_distils(tmp_path, capsys):
    from graphcuda_b200.train_planetoid import main
    ids = list(range(200, 260))
    np.random.default_rng(5).shuffle(ids)
    _write(str(tmp_path), "toy", n_train=20, n_other=180, test_ids=ids, n_feat=50, n_cls=4, seed=7)
    history = main(["--raw", str(tmp_path), "--name", "toy", "--epochs", "3", "--layers", "2", "--hidden", "32", "--optimizer", "adamw",
                    "--seed", "11", "--serve", "--serve-bits", "4", "--distill", "16"])["history"]
    out = capsys.readouterr().out
    assert "Served in 4 bits | Train Acc:" in out and "Distilled epoch 003 | Loss:" in out
    served, lines = [h for h in history if h.get("served")], [h for h in history if h.get("distilled")]
    assert len(served) == 1 and len(lines) == 3 and all(h["loss"] >= 0 for h in lines)
