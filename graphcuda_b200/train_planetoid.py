"""The reference's training script (tests/gcn/graphcuda_impl.py) on this library, without torch_geometric:

    python -m graphcuda_b200.train_planetoid --raw <reference tree>/data/Cora/raw --name cora

Same flow and the same printed lines: a 2-layer GCN (hidden 16), SGD with lr 1 (line 45), 20 epochs of
train() (lines 51-58) each followed by test() (lines 60-69), epoch time = the train step only (lines 78-82).
Differences: the raw files are parsed by graphcuda_b200.planetoid, the adjacency is normalised on the GPU
(normalized_adjacency replaces lines 27-38), log_softmax + nll_loss is the fused kernel, the optimizer step is one
launch, test() is GCN.evaluate (fused argmax / accuracy counts), and ``--graph`` replays the whole train step as
one CUDA graph.  ``--optimizer adam`` gives the Adam lr 0.01 configuration this library is benchmarked on.

Beyond the script, a deep model: ``--layers 8 --hidden 64 --optimizer adamw [--state-bits 8] [--serve]`` trains
models.ResidualGCN (norms, gated feed-forward blocks) with FusedAdamW; ``--serve`` evaluates it in 8 bits at the end.
"""
from __future__ import annotations

import argparse
import time

import torch

from . import ops


def main(argv=None) -> dict:
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--raw", required=True, help="directory holding ind.<name>.* files")
    ap.add_argument("--name", default="cora")
    ap.add_argument("--epochs", type=int, default=20)
    ap.add_argument("--hidden", type=int, default=16)
    ap.add_argument("--layers", type=int, default=None, help="a residual model of this many blocks, --hidden wide")
    ap.add_argument("--optimizer", choices=["sgd", "adam", "adamw"], default="sgd")
    ap.add_argument("--lr", type=float, default=None,
                    help="default: 1 for sgd (the script's value), 0.01 for adam, 0.003 for adamw")
    ap.add_argument("--state-bits", type=int, choices=[8, 32], default=32, help="of the moments that adamw keeps")
    ap.add_argument("--serve", action="store_true", help="with --layers: evaluate in 8 bits at the end")
    ap.add_argument("--seed", type=int, default=None)
    ap.add_argument("--graph", action="store_true", help="record the train step once and replay it as a CUDA graph")
    ap.add_argument("--precision", default=None)
    args = ap.parse_args(argv)

    import graphcuda_b200 as gc
    from graphcuda_b200.models import GCN, ResidualGCN
    from graphcuda_b200.planetoid import load_planetoid_raw

    if not torch.cuda.is_available():
        raise SystemExit("graphcuda_b200 has no CPU path: a CUDA device is required")
    device = torch.device("cuda")
    if args.seed is not None:
        torch.manual_seed(args.seed)
    data = load_planetoid_raw(args.raw, args.name).to(device)
    adj = gc.normalized_adjacency(data.edge_index, data.num_nodes, symmetric=True)
    if args.layers is None:
        if args.serve:
            ap.error("--serve needs --layers")
        model = GCN([data.num_node_features, args.hidden, data.num_classes], precision=args.precision).to(device)
    else:
        if args.optimizer != "adamw":
            ap.error("--layers: the feed-forward blocks' bfloat16 weights need --optimizer adamw")
        model = ResidualGCN(data.num_node_features, args.hidden, args.layers, data.num_classes,
                            precision=args.precision).to(device)
    lr = args.lr if args.lr is not None else {"sgd": 1.0, "adam": 0.01, "adamw": 0.003}[args.optimizer]
    if args.optimizer == "adamw":
        opt = gc.FusedAdamW(model.parameters(), lr=lr, state_bits=args.state_bits)
    else:
        opt = (gc.FusedSGD if args.optimizer == "sgd" else gc.FusedAdam)(model.parameters(), lr=lr)
    masks = [data.train_mask, data.val_mask, data.test_mask]
    n_train = int(data.train_mask.sum())
    print(f"Model is on device: {next(model.parameters()).device}")
    print(f"Data.x is on device: {data.x.device}")
    print(f"Data.edge_index is on device: {data.edge_index.device}")

    def train_eager():
        model.train()
        opt.zero_grad(set_to_none=True)
        loss = gc.log_softmax_nll_loss(model(data.x, adj, log_softmax=False), data.y, data.train_mask,
                                       scale=1.0 / n_train)
        loss.backward()
        opt.step()
        return loss

    def test():
        model.eval()
        _, counts = model.evaluate(data.x, adj, data.y, masks)
        c = counts.cpu()
        return [int(c[i, 0]) / max(int(c[i, 1]), 1) for i in range(3)]

    accs = test()
    print(f"Epoch 000 | Train Acc: {accs[0]:.4f} | Val Acc: {accs[1]:.4f} | Test Acc: {accs[2]:.4f}")
    history = [dict(epoch=0, train=accs[0], val=accs[1], test=accs[2])]
    graphed = None
    total = 0.0
    for epoch in range(1, args.epochs + 1):
        torch.cuda.synchronize()
        t0 = time.time()
        if args.graph and graphed is None:
            # Recorded before the model is ever trained on the default stream.  The constructor runs one eager
            # step on the capture's side stream (plans get built there); that step is this epoch's update.
            graphed = gc.GraphedTrainStep(model, adj, data.x, data.y, opt, row_mask=data.train_mask, warmup=1)
            loss = graphed.warmup_loss
        elif graphed is not None:
            loss = graphed.step()
        else:
            loss = train_eager()
        loss_value = loss.item()  # like the script's loss.item(): waits for the step
        dt = time.time() - t0
        ops.check_gemm_flag(data.x.device)  # the step is complete: a tensor-core wait that ran out would show now
        total += dt
        accs = test()
        history.append(dict(epoch=epoch, time=dt, loss=loss_value, train=accs[0], val=accs[1], test=accs[2]))
        print(f"Epoch {epoch:03d} | Time: {dt:.4f}s | Loss: {loss_value:.4f} | "
              f"Train Acc: {accs[0]:.4f} | Val Acc: {accs[1]:.4f} | Test Acc: {accs[2]:.4f}")
    if args.serve:
        model.eval()
        _, counts = model.for_serving().evaluate(data.x, adj, data.y, masks)
        served = [int(a) / max(int(b), 1) for a, b in counts.cpu()]
        print(f"Served in 8 bits | Train Acc: {served[0]:.4f} | Val Acc: {served[1]:.4f} | Test Acc: {served[2]:.4f}")
        history.append(dict(epoch=args.epochs, served=True, train=served[0], val=served[1], test=served[2]))
    print(f"\nTotal training time for {args.epochs} epochs: {total:.4f} seconds")
    print(f"Average time per epoch (train): {total / max(args.epochs, 1):.6f} seconds")
    return dict(history=history, seconds=total)


if __name__ == "__main__":
    main()
