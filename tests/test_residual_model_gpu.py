"""The deep model that runs the norm, the gated block and AdamW together: against its formula, in training, recorded,
served in 8 bits, and through the training command."""
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

N, F, WIDTH, LAYERS, CLASSES = 600, 50, 48, 3, 7


def _setup(cuda, seed=0):
    from graphcuda_b200 import normalized_adjacency, synth
    from graphcuda_b200.models import ResidualGCN
    e = synth.preferential_attachment_edges(N, 4 * N, seed)
    edges = synth.symmetrize(e)
    adj = normalized_adjacency(edges.to(cuda), N, symmetric=True)
    torch.manual_seed(seed)
    model = ResidualGCN(F, WIDTH, LAYERS, CLASSES, hidden=80).to(cuda)
    g = torch.Generator().manual_seed(seed)
    y = torch.randint(0, CLASSES, (N,), generator=g).to(cuda)
    # features that tell the classes apart
    X = (torch.randn(N, F, generator=g).to(cuda) + 3 * torch.nn.functional.one_hot(y, F).float())
    return adj, edges, model, X, y


def _dense(edges):
    A = torch.eye(N, dtype=torch.float64)
    A[edges[0], edges[1]] = 1
    d = A.sum(0).rsqrt()
    return d[:, None] * A * d


def test_forward_is_the_formula(cuda):
    adj, edges, model, X, _ = _setup(cuda)
    A, w = _dense(edges), {k: v.detach().cpu().double() for k, v in model.state_dict().items()}
    norm = lambda h, k: h / (h.square().mean(1, keepdim=True) + 1e-6).sqrt() * w[k + ".weight"]  # noqa: E731
    h = A @ X.cpu().double() @ w["conv_in.weights"]
    for i in range(LAYERS):
        p = f"blocks.{i}."
        h = h + A @ norm(h, p + "norm_conv") @ w[p + "conv.weights"]
        gu = norm(h, p + "norm_ffn") @ w[p + "ffn.w_in"]
        g, u = gu.chunk(2, 1)
        h = h + (g * torch.sigmoid(g) * u) @ w[p + "ffn.w_out"]
    ref = A @ norm(h, "norm_out") @ w["conv_out.weights"]
    with torch.no_grad():
        got = model(X, adj, log_softmax=False)
    # three roundings to bfloat16 per block (its input, hidden row and output), 2^-8 each, in an addition to the stream
    assert float((got.cpu().double() - ref).norm() / ref.norm()) < 3 * LAYERS * 2.0 ** -8
    served = model.for_serving()(X, adj, log_softmax=False)
    assert float((served.cpu().double() - ref).norm() / ref.norm()) < 2 * LAYERS * 2.0 ** -4


@pytest.mark.parametrize("bits", [32, 8])
def test_trains_recorded_and_serves(cuda, bits):
    from graphcuda_b200 import FusedAdamW, GraphedTrainStep, log_softmax_nll_loss, ops
    adj, _, model, X, y = _setup(cuda, seed=1)
    opt = FusedAdamW(model.parameters(), lr=3e-3, state_bits=bits)
    with torch.no_grad():
        first = log_softmax_nll_loss(model(X, adj, log_softmax=False), y, scale=1.0 / N).item()
    step = GraphedTrainStep(model, adj, X, y, opt, warmup=2)
    for _ in range(60):
        loss = step.step()
    assert loss.item() < 0.2 * first and opt.steps_taken() == 62
    pred, counts = model.evaluate(X, adj, y)
    accuracy = int(counts[0, 0]) / N
    assert accuracy > 0.95 and torch.equal(pred, model(X, adj).argmax(1))
    served = model.for_serving()
    _, counts = served.evaluate(X, adj, y)
    assert int(counts[0, 0]) / N > accuracy - 0.03
    ops.check_gemm_flag(cuda)


def test_recorded_steps_are_the_eager_ones(cuda):
    from graphcuda_b200 import FusedAdamW, GraphedTrainStep, log_softmax_nll_loss
    adj, _, eager, X, y = _setup(cuda, seed=2)
    _, _, graphed, _, _ = _setup(cuda, seed=2)
    a, b = FusedAdamW(eager.parameters(), lr=1e-3), FusedAdamW(graphed.parameters(), lr=1e-3)
    step = GraphedTrainStep(graphed, adj, X, y, b, warmup=1)
    for _ in range(4):
        step.step()
    for _ in range(5):
        a.zero_grad(set_to_none=True)
        log_softmax_nll_loss(eager(X, adj, log_softmax=False), y, scale=1.0 / N).backward()
        a.step()
    assert all(torch.equal(p, q) for p, q in zip(eager.parameters(), graphed.parameters()))


def test_training_command(cuda, golden_dir, capsys):
    from graphcuda_b200 import train_planetoid
    raw = os.path.join(golden_dir, "cora_raw")
    r = train_planetoid.main(["--raw", raw, "--layers", "2", "--hidden", "32", "--optimizer", "adamw", "--epochs", "30",
                              "--seed", "3", "--state-bits", "8", "--graph", "--serve"])
    best = max(h["test"] for h in r["history"])
    assert best > 0.65 and r["history"][-1]["served"] and r["history"][-1]["test"] > best - 0.1
    assert "Served in 8 bits" in capsys.readouterr().out
    for bad in (["--layers", "2"], ["--serve"]):
        with pytest.raises(SystemExit):
            train_planetoid.main(["--raw", raw] + bad)
