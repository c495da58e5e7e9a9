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


# ---- masters
SIZES = [(700,), (33,), (65, 64), (4097,)]


def _change(p, new, how):
    if how == "copy_":
        with torch.no_grad():
            p.copy_(new)
    elif how == "data":
        p.data.copy_(new)
    elif how == "swap":
        p.data = new.clone()
    else:  # one element of seven: the others keep what their masters have beyond bfloat16
        p.data.view(-1)[::7] = new.view(-1)[::7]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("how", ["copy_", "data", "swap", "some"])
def test_a_parameter_changed_between_steps_stays_changed(cuda, bits, how):
    """As with torch.optim: the next step starts from the value that the parameter has.  Beside it, an optimizer whose masters
    are changed by hand."""
    import graphcuda_b200 as gc
    sets = [[torch.nn.Parameter(_randn(s, i, torch.bfloat16)) for i, s in enumerate(SIZES)] for _ in range(2)]
    opts = [gc.FusedAdamW(ps, **HYPER, state_bits=bits, seed=5) for ps in sets]

    def step(t):
        for ps, opt in zip(sets, opts):
            for i, p in enumerate(ps):
                p.grad = _randn(p.shape, 10 * t + i, torch.bfloat16)
            opt.step()

    for t in range(3):
        step(t)
    for i, (p, q) in enumerate(zip(*sets)):
        master = opts[1].state[q]["master"]
        assert not torch.equal(master, q.detach().float())  # there is something to keep
        new = _randn(p.shape, 100 + i, torch.bfloat16)
        _change(p, new, how)
        changed = p.detach().view(torch.int16) != q.detach().view(torch.int16)
        assert changed.any()
        master.copy_(torch.where(changed, p.detach().float(), master))
        q.data.copy_(p.detach())
    for t in range(3, 5):
        step(t)
    for p, q in zip(*sets):
        assert torch.equal(p, q)
        assert all(torch.equal(opts[0].state[p][k], opts[1].state[q][k]) for k in opts[0].state[p])


def test_loaded_weights_stay_in_a_run_that_is_recorded(cuda):
    """A state dict loaded between replays of a recorded step."""
    import graphcuda_b200 as gc
    lin = gc.GatedFFN(32, 40, 24).to(cuda)
    for i, p in enumerate(lin.parameters()):
        p.grad = _randn(p.shape, i, torch.bfloat16)
    start = {k: v.clone() for k, v in lin.state_dict().items()}
    opt = gc.FusedAdamW(lin.parameters(), lr=1e-2, weight_decay=0.0)
    opt.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for _ in range(20):
        graph.replay()
    far = {k: (v.float() - start[k].float()).abs().max().item() for k, v in lin.state_dict().items()}
    assert min(far.values()) > 0.1
    lin.load_state_dict(start)
    graph.replay()
    for k, v in lin.state_dict().items():  # one step of a constant gradient: the learning rate, and bfloat16's rounding
        assert float((v.float() - start[k].float()).abs().max()) < 0.011 + float(start[k].abs().max()) * 2.0 ** -8


def test_lists_with_masters_take_the_masters_word(cuda):
    """adamw_step on lists: the masters are the parameters, whatever the bfloat16 tensors hold -- unless they are to follow."""
    import graphcuda_b200 as gc
    for follow in (False, True):
        master, g = _randn(900, 0), _randn(900, 1, torch.bfloat16)
        p = torch.full((900,), 3.0, dtype=torch.bfloat16, device=cuda)
        m, v = torch.zeros(900, device=cuda), torch.zeros(900, device=cuda)
        step = torch.zeros(2, dtype=torch.int64, device=cuda)
        expect = torch.full_like(master, 3.0) if follow else master.clone()
        gc.adamw_step([p], [g], [m], [v], step, masters=[master], **(dict(follow=True) if follow else {}), **HYPER)
        m2, v2, step2 = torch.zeros(900, device=cuda), torch.zeros(900, device=cuda), torch.zeros(2, dtype=torch.int64, device=cuda)
        gc.adamw_step([expect], [g.float()], [m2], [v2], step2, **HYPER)
        assert torch.equal(master, expect) and torch.equal(p, expect.bfloat16())


def test_following_takes_masters(cuda):
    import graphcuda_b200 as gc
    p, step = torch.zeros(300, device=cuda), torch.zeros(2, dtype=torch.int64, device=cuda)
    with pytest.raises(RuntimeError, match="masters"):
        gc.adamw_step([p], [p], [p.clone()], [p.clone()], step, lr=0.1, follow=True)
    assert not step.any()


# ---- recording
def test_a_first_step_is_not_recorded(cuda):
    """States made while a stream is captured would be zeros again at every replay."""
    import graphcuda_b200 as gc
    p, x = torch.nn.Parameter(_randn(500, 0)), torch.zeros(1, device=cuda)
    p.grad = _randn(500, 1)
    opt = gc.FusedAdamW([p], lr=0.1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x.add_(1)
        with pytest.raises(RuntimeError, match="before it is recorded"):
            opt.step()
    assert not opt.state[p]
    opt.step()
    assert opt.steps_taken() == 1


def test_a_count_that_parts_is_not_recorded(cuda):
    """Parameters that have always been updated together share a count; a copy of it made while a stream is captured would be
    the same count again at every replay."""
    import graphcuda_b200 as gc
    p, q, x = torch.nn.Parameter(_randn(500, 0)), torch.nn.Parameter(_randn(400, 1)), torch.zeros(1, device=cuda)
    p.grad, q.grad = _randn(500, 2), _randn(400, 3)
    opt = gc.FusedAdamW([p, q], lr=0.1)
    opt.step()
    q.grad = None
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x.add_(1)
        with pytest.raises(RuntimeError, match="before it is recorded"):
            opt.step()
    opt.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for _ in range(3):
        graph.replay()
    assert int(opt.state[p]["step"][0]) == 5 and int(opt.state[q]["step"][0]) == 1


# ---- random bits
def test_lists_round_by_bits_of_their_own(cuda):
    """Equal tensors and gradients in different groups, and in one group beside others: rounded differently, the first as a call
    on a list alone."""
    import graphcuda_b200 as gc
    n = 2048
    ps = [torch.nn.Parameter(_randn(n, 0)) for _ in range(3)]
    opt = gc.FusedAdamW([dict(params=[p]) for p in ps], **HYPER, state_bits=8, seed=11)
    codes = [[torch.zeros(n, dtype=torch.uint8, device=cuda)] for _ in range(2)]
    scales = [[torch.zeros(n // 256, device=cuda)] for _ in range(2)]
    step, alone = torch.zeros(2, dtype=torch.int64, device=cuda), ps[0].detach().clone()
    g = _randn(n, 1)
    for _ in range(2):
        for p in ps:
            p.grad = g.clone()
        opt.step()
        gc.adamw_step([alone], [g], *codes, step, scales=scales, seed=11, **HYPER)
    st = [opt.state[p] for p in ps]
    assert torch.equal(st[0]["exp_avg"], codes[0][0]) and torch.equal(st[0]["exp_avg_sq"], codes[1][0])
    for i in range(3):
        for j in range(i):
            for k in ("exp_avg", "exp_avg_sq"):
                assert float((st[i][k] != st[j][k]).float().mean()) > 0.2


# ---- more elements than the CTAs of a launch take in one pass
def test_8_bit_codes_of_a_large_tensor(cuda):
    """Chunks that a CTA comes to in its second and third pass, and the tensor behind: the codes of the formula."""
    import graphcuda_b200 as gc
    from test_adamw_gpu import _blocks, _host_step
    from test_adamw_gpu import HYPER as hyper
    sizes = (148 * 4 * 2048 * 2 + 777, 5000)
    gs = [_randn(n, i) for i, n in enumerate(sizes)]
    ps = [torch.zeros(n, device=cuda) for n in sizes]
    codes = [[torch.zeros(n, dtype=torch.uint8, device=cuda) for n in sizes] for _ in range(2)]
    scales = [[torch.zeros(-(-n // 256), device=cuda) for n in sizes] for _ in range(2)]
    step = torch.zeros(2, dtype=torch.int64, device=cuda)
    host = [(np.zeros_like(_blocks(g.cpu().numpy())),) * 2 for g in gs]
    for t in (1, 2):
        gc.adamw_step(ps, gs, *codes, step, scales=scales, seed=3, **hyper)
        for i, n in enumerate(sizes):
            qm, qv, ms, vs, m, v = _host_step(gs[i].cpu().numpy(), *host[i], 3, t, i)
            m.reshape(-1)[n:] = 0
            v.reshape(-1)[n:] = 0
            host[i] = m, v
            assert np.array_equal(scales[0][i].cpu().numpy(), ms[:, 0]) and np.array_equal(scales[1][i].cpu().numpy(), vs[:, 0])
            assert np.array_equal(codes[0][i].cpu().numpy(), qm.reshape(-1)[:n])
            assert np.array_equal(codes[1][i].cpu().numpy(), qv.reshape(-1)[:n])
