"""Weights of 4 bits on the CPU: their layout, their quantisation, and what the entry points refuse without touching a GPU."""
import pytest
import torch

import graphcuda_b200 as gc
from graphcuda_b200 import _lib

L = _lib.lib
M, K, N = 250, 200, 33
D, H, O = 40, 24, 16


def _linear(x=16, ldx=K, w=16, group=64, zeros=0, m=M, k=K, n=N, y=16, ldy=N, ws=16, wsb=None):
    need = L().gc_linear_int4_workspace_bytes(M, K, N)
    return L().gc_linear_int4_bf16(x, ldx, w, group, zeros, m, k, n, y, ldy, ws, need if wsb is None else wsb, None)


def _block(x=16, ldx=D, wi=16, gi=64, zi=0, wo=16, go=128, zo=1, m=M, d=D, h=H, o=O, act=0, y=16, ldy=O, ws=16,
           wsb=None):
    need = L().gc_gated_ffn_int4_workspace_bytes(M, D, H, O)
    return L().gc_gated_ffn_int4_bf16(x, ldx, wi, gi, zi, wo, go, zo, m, d, h, o, act, y, ldy, ws, need if wsb is None else wsb, None)


def test_what_the_product_refuses():
    for bad in (dict(m=-1), dict(k=-1), dict(n=-1), dict(ldx=K - 1), dict(ldy=N - 1), dict(x=None), dict(y=None), dict(w=None),
                dict(group=16), dict(group=256), dict(group=0), dict(w=8), dict(ws=24)):
        assert _linear(**bad) == -1, bad
    assert _linear(m=1 << 30) == -2 and _linear(k=1 << 27, ldx=1 << 27) == -2
    assert _linear(ws=None) == -4 and _linear(wsb=L().gc_linear_int4_workspace_bytes(M, K, N) - 1) == -4
    assert _linear(m=0, x=None, y=None) == 0 and _linear(n=0, y=None) == 0


def test_what_the_block_refuses():
    for bad in (dict(m=-1), dict(d=-1), dict(h=-1), dict(o=-1), dict(ldx=D - 1), dict(ldy=O - 1), dict(x=None), dict(y=None), dict(wi=None),
                dict(wo=None), dict(gi=1), dict(go=1), dict(wi=8), dict(wo=8), dict(act=3), dict(act=-1), dict(ws=24)):
        assert _block(**bad) == -1, bad
    assert _block(m=1 << 30) == -2 and _block(h=1 << 29) == -2
    assert _block(ws=None) == -4 and _block(wsb=L().gc_gated_ffn_int4_workspace_bytes(M, D, H, O) - 1) == -4
    assert _block(m=0, x=None, y=None) == 0 and _block(o=0, y=None) == 0


def test_queries():
    for q in (lambda m: L().gc_linear_int4_workspace_bytes(m, K, N), lambda m: L().gc_gated_ffn_int4_workspace_bytes(m, D, H, O)):
        assert q(0) == q(-1) == q(1 << 30) == 0 and q(1000) >= q(250) > 0
    assert L().gc_linear_int4_workspace_bytes(32, 2000, 3000) < 2000 * 3000  # weights are not unpacked for so few rows


@pytest.mark.parametrize("k,n,group", [(1, 1, 32), (130, 20, 32), (200, 33, 64), (128, 16, 128), (300, 70, 128), (0, 5, 32), (7, 0, 64)])
@pytest.mark.parametrize("zeros", [False, True])
def test_layout_and_back(k, n, group, zeros):
    g = torch.Generator().manual_seed(k)
    codes = torch.randint(0, 16, (k, n), generator=g, dtype=torch.uint8)
    groups = -(-k // group)
    scale = torch.randn(groups, n, generator=g).bfloat16()
    zero = torch.randint(0, 16, (groups, n), generator=g, dtype=torch.uint8) if zeros else None
    w = gc.Int4Weight.from_codes(codes, scale, zero, group=group)
    of = torch.arange(k) // group
    assert torch.equal(w.dequantize(), (codes.float() - (zero.float()[of] if zeros else 8)) * scale.float()[of])
    if not k or not n:
        return
    for kk, nn in ((0, 0), (k - 1, n - 1), (k // 2, n // 3)):  # the layout that the C interface documents
        c = kk % 128
        at = nn % 16 * 64 + (c % 32 // 8 * 4 + c // 32) * 4
        record = w.records[nn // 16, kk // 128]
        word = int.from_bytes(bytes(record[at:at + 4].tolist()), "little")
        e = c % 8
        assert word >> (4 * (e // 2 + e % 2 * 4)) & 15 == int(codes[kk, nn])
        of = nn % 16 * (128 // group) + c // group
        assert record[1024:1024 + 32 * (128 // group)].clone().view(torch.bfloat16)[of] == scale[kk // group, nn]
        assert not zeros or record[1024 + 32 * (128 // group) + of] == zero[kk // group, nn]


def test_refused_codes():
    codes, scale = torch.zeros(64, 8, dtype=torch.uint8), torch.ones(1, 8, dtype=torch.bfloat16)
    for args, kw in (((codes, scale), dict(group=16)), ((codes.int(), scale), dict(group=64)), ((codes[0], scale), dict(group=64)),
                     ((codes, scale.float()), dict(group=64)), ((codes, scale), dict(group=32)), ((codes + 16, scale), dict(group=64)),
                     ((codes, scale, scale), dict(group=64)), ((codes, scale, codes[:1] + 200), dict(group=64)),
                     ((codes, scale, codes[:2]), dict(group=64))):
        with pytest.raises(RuntimeError):
            gc.Int4Weight.from_codes(*args, **kw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
def test_quantisation(dtype, group, zeros):
    """A value is off by half a step, and by what the scale's rounding (2^-8 of it) moves the ends of the range."""
    g = torch.Generator().manual_seed(group)
    w = torch.randn(333, 21, generator=g)
    w[:, 3] += 4
    w[:, 4] = 0
    w[128:256, 5] = 0
    w[:, 6] = w[:, 6].abs()
    w[:, 7] *= 1e30
    w[:, 8] *= 1e-30
    w = w.to(dtype)
    got = gc.quantize_weight_int4(w, group, zeros).dequantize()
    t = torch.zeros(-(-333 // group) * group, 21)
    t[:333] = w.float()
    t = t.view(-1, group, 21)
    step = (t.amax(1).clamp(min=0) - t.amin(1).clamp(max=0)) / 15 if zeros else t.abs().amax(1) / 7.5
    step = step.repeat_interleave(group, 0)[:333] * (1 + 2.0 ** -8)
    reach = 15 if zeros else 7.5  # steps between zero and the far end
    assert bool(((got - w.float()).abs() <= step * (0.5 + reach * 2.0 ** -7) + 1e-45).all())
    assert not got[:, 4].any() and not got[128:256, 5].any()


def test_refused_weights():
    for w, kw in ((torch.zeros(4), {}), (torch.zeros(4, 4, dtype=torch.int32), {}), (torch.zeros(4, 4), dict(group=48)),
                  (torch.full((4, 4), float("nan")), {}), (torch.full((4, 4), float("inf")), {})):
        with pytest.raises(RuntimeError):
            gc.quantize_weight_int4(w, **kw)


def test_cpu_tensors_are_refused():
    w = gc.quantize_weight_int4(torch.randn(8, 16))
    with pytest.raises(RuntimeError, match="CUDA"):
        gc.linear_int4(torch.zeros(2, 8, dtype=torch.bfloat16), w)
    with pytest.raises(RuntimeError, match="CUDA"):
        gc.gated_ffn_int4(torch.zeros(2, 8, dtype=torch.bfloat16), w, gc.quantize_weight_int4(torch.randn(8, 4)))
    with pytest.raises(ValueError):
        gc.gated_ffn_int4(torch.zeros(2, 8, dtype=torch.bfloat16), w, w, activation="tanh")


def test_state_and_moves():
    w = gc.quantize_weight_int4(torch.randn(100, 40), 32, True)
    assert set(w.state_dict()) == {"records"}
    w.half(), w.float()  # of no concern to bytes
    other = gc.quantize_weight_int4(torch.randn(100, 40), 32, True)
    other.load_state_dict(w.state_dict())
    assert torch.equal(other.dequantize(), w.dequantize())
    block = gc.GatedFFN(16, 24, 8)
    assert type(block.for_serving(4)).__name__ == "GatedFFNInt4" and type(block.for_serving()).__name__ == "GatedFFNFp8"
    with pytest.raises(ValueError):
        block.for_serving(2)
