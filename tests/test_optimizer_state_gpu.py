"""What the optimizers leave behind beside the numbers: versions that autograd checks, masters that follow their parameters,
step counts under recording, random bits."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

HYPER = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)


def _randn(shape, seed, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to("cuda", dtype)


# ---- versions
@pytest.mark.parametrize("name", ["FusedSGD", "FusedAdam", "FusedAdamW", "FusedAdamW8"])
def test_a_step_between_forward_and_backward_is_told(cuda, name):
    import graphcuda_b200 as gc
    p = torch.nn.Parameter(_randn((40, 30), 0))
    q = torch.nn.Parameter(_randn((20,), 1))
    opt = getattr(gc, name.rstrip("8"))([p, q], lr=0.1, **(dict(state_bits=8) if name[-1] == "8" else {}))
    for _ in range(2):
        loss = (p * p).sum() + (q * q).sum()
        p.grad, q.grad = _randn((40, 30), 2), _randn((20,), 3)
        versions = p._version, q._version
        opt.step()
        assert p._version > versions[0] and q._version > versions[1]
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    p.grad = q.grad = None
    ((p * p).sum() + (q * q).sum()).backward()  # a new forward pass is fine


def test_a_step_between_the_blocks_passes_is_told(cuda):
    import graphcuda_b200 as gc
    block = gc.GatedFFN(32, 48, 16).to(cuda)
    norm = gc.RMSNorm(32, out_dtype=torch.bfloat16).to(cuda)
    opt = gc.FusedAdamW([*block.parameters(), *norm.parameters()], lr=0.1)
    x = _randn((9, 32), 0)
    block(norm(x)).float().sum().backward()
    for module, arg in ((block, x.bfloat16()), (norm, x)):
        y = module(arg)
        opt.step()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.float().sum().backward()


def test_everything_a_step_writes_has_a_new_version(cuda):
    import graphcuda_b200 as gc
    p, master, g = _randn(600, 0, torch.bfloat16), _randn(600, 0), _randn(600, 1, torch.bfloat16)
    m, v = (torch.zeros(600, dtype=torch.uint8, device=cuda) for _ in range(2))
    ms, vs = (torch.zeros(3, device=cuda) for _ in range(2))
    step = torch.zeros(2, dtype=torch.int64, device=cuda)
    written, read = (p, master, m, v, ms, vs, step), (g,)
    before = [t._version for t in written], [t._version for t in read]
    gc.adamw_step([p], [g], [m], [v], step, masters=[master], scales=([ms], [vs]), lr=0.1)
    assert all(t._version > b for t, b in zip(written, before[0])) and [t._version for t in read] == before[1]
    out = torch.zeros(600, device=cuda), torch.zeros(600, device=cuda)
    versions = [t._version for t in (*out, m, v, ms, vs)]
    gc.adamw_moments([m], [v], ([ms], [vs]), out=([out[0]], [out[1]]))
    assert all(t._version > b for t, b in zip(out, versions)) and [t._version for t in (m, v, ms, vs)] == versions[2:]
    with torch.inference_mode():  # such tensors have no versions
        p, g, m, v = torch.zeros(600, device=cuda), torch.ones(600, device=cuda), torch.zeros(600, device=cuda), torch.zeros(600, device=cuda)
        step = torch.zeros(2, dtype=torch.int64, device=cuda)
        gc.adamw_step([p], [g], [m], [v], step, lr=0.1)
        assert int(step[0]) == 1 and bool((p < 0).all())
