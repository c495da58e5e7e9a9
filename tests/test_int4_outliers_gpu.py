"""Gated blocks with 4-bit weights where a few weights or inputs are far larger than the others.

A hidden value's rounding is of its own size, down to 2^-13 of its row's largest: what a bound over the row, an input that few weights
take up, or a weight that meets zeros would come to has no say in it.  The
error on average is the documented one (see test_int4_gpu): the result's rounding, 2^-8 / sqrt(3) at most, and above 64 rows an
eighth of that each for both weights, the hidden row, and once more for the slope."""
import pytest
import torch

import graphcuda_b200 as gc
from tests.test_int4_gpu import HALF, act64, rms, rows

pytestmark = pytest.mark.gpu
DEV = "cuda"
ALLOWED = HALF / 3 ** 0.5 * 1.09 ** 0.5
D, H, O = 4096, 512, 256


def normal(k, n, seed):
    return torch.randn(k, n, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV) / k ** 0.5


def error(x, w_in, w_out, act):
    G, U = (x.double() @ w_in.dequantize().double()).split(w_out.in_features, 1)
    want = (act64(act, G)[0] * U) @ w_out.dequantize().double()
    return rms(gc.gated_ffn_int4(x, w_in, w_out, activation=act), want)


@pytest.mark.parametrize("m", [64, 65, 300, 1000])
@pytest.mark.parametrize("times", [16, 64, 256, 4096])
@pytest.mark.parametrize("half", ["gate", "up", "both"])
def test_a_column_that_no_output_takes_up(m, times, half):
    """One hidden column is `times` the others, and its row of the second weight is zero."""
    wi, wo = normal(D, 2 * H, 1), normal(H, O, 2)
    if half != "up":
        wi[:, 77] *= times
    if half != "gate":
        wi[:, H + 77] *= times
    wo[77] = 0
    assert error(rows(m, D), gc.quantize_weight_int4(wi, 32), gc.quantize_weight_int4(wo, 32), "silu") <= ALLOWED


@pytest.mark.parametrize("m", [64, 65, 300])
@pytest.mark.parametrize("group,zeros", [(32, False), (64, True), (128, False)])
@pytest.mark.parametrize("weight,value", [(300, 1), (100, 50), (300, 50), (1, 1000)])
def test_one_large_weight_and_one_large_input(m, group, zeros, weight, value):
    wi, wo, x = normal(D, 2 * H, 3), normal(H, O, 4), rows(m, D)
    wi[123, 45] *= weight
    x[:, 999] *= value
    assert error(x, gc.quantize_weight_int4(wi, group, zeros), gc.quantize_weight_int4(wo, group, zeros), "gelu") <= ALLOWED


@pytest.mark.parametrize("m", [65, 700])
def test_columns_over_a_wide_range_that_the_second_weight_evens_out(m):
    """Hidden columns of all sizes, each with as much of a say; a group of the second weight has rows of a few sizes."""
    wi, wo = normal(D, 2 * H, 5), normal(H, O, 6)
    size = 2.0 ** torch.linspace(-5, 5, H, device=DEV)
    wi[:, :H] *= size
    wi[:, H:] *= size
    wo /= wi[:, :H].norm(dim=0)[:, None] * wi[:, H:].norm(dim=0)[:, None]
    for act in ("silu", "relu"):
        assert error(rows(m, D), gc.quantize_weight_int4(wi, 64), gc.quantize_weight_int4(wo, 32), act) <= ALLOWED


@pytest.mark.parametrize("m", [64, 65, 300])
@pytest.mark.parametrize("power", [0, 3, 6, 9, 12])
def test_large_groups_that_meet_zeros(m, power):
    """Weights of inputs, and of hidden columns, that are zero: the others keep their bits beside them."""
    wi, wo, x = normal(512, 2 * 64, 12), normal(64, 32, 13), rows(m, 512)
    wi[:32] *= 300
    x[:, :32] = 0
    wi[:, :32] = 0  # of G: so these hidden columns are zero
    wo *= 2.0 ** power  # (wherever that lies among the steps of outputs' exponents)
    wo[:32] *= 2.0 ** 14
    assert error(x, gc.quantize_weight_int4(wi, 32), gc.quantize_weight_int4(wo, 32), "silu") <= ALLOWED


@pytest.mark.parametrize("m", [64, 65, 300])
@pytest.mark.parametrize("d,zeros", [(64, False), (64, True), (512, True), (4096, False), (4096, True)])
@pytest.mark.parametrize("act", ["silu", "relu"])
def test_inputs_of_all_sizes_that_the_weights_even_out(m, d, zeros, act):
    """Channels of the input differ by some thousands, and so do the weights that take them up: what they come to is far below the
    product of the row's length and the weights'."""
    g = torch.Generator(device=DEV).manual_seed(d)
    size = torch.exp(2 * torch.randn(d, generator=g, device=DEV))
    wi, wo = normal(d, 2 * 256, 14), normal(256, 128, 15)
    wi = wi / size[:, None] * torch.exp(1.5 * torch.randn(2 * 256, generator=g, device=DEV))
    wo = wo * torch.exp(2 * torch.randn(256, generator=g, device=DEV))[:, None]
    x = (rows(m, d).float() * size).bfloat16()
    assert error(x, gc.quantize_weight_int4(wi, 32, zeros), gc.quantize_weight_int4(wo, 32, zeros), act) <= ALLOWED


@pytest.mark.parametrize("power", [10, 16, 20])
@pytest.mark.parametrize("inputs", [32, 2048])
def test_small_groups_whose_inputs_make_up_for_it(power, inputs):
    for shift in (0, 5, 10):  # wherever that lies among the steps of outputs' exponents
        wi, wo, x = normal(D, 2 * 256, 22) * 2.0 ** shift, normal(256, 128, 23), rows(300, D).float()
        wi[:inputs] *= 2.0 ** -power
        x[:, :inputs] *= 2.0 ** power
        assert error(x.bfloat16(), gc.quantize_weight_int4(wi, 32), gc.quantize_weight_int4(wo, 32), "silu") <= ALLOWED


@pytest.mark.parametrize("m", [65, 300])
@pytest.mark.parametrize("times", [300, 4096, 65_536])
def test_large_weights_of_inputs_that_are_zero(m, times):
    wi, wo, x = normal(D, 2 * H, 16), normal(H, O, 17), rows(m, D)
    wi[7] *= times
    x[:, 7] = 0
    assert error(x, gc.quantize_weight_int4(wi, 32), gc.quantize_weight_int4(wo, 32), "silu") <= ALLOWED


@pytest.mark.parametrize("m", [65, 300])
@pytest.mark.parametrize("times", [1000.0, 1e5])
def test_a_large_input_that_no_weight_takes_up(m, times):
    wi, wo, x = normal(D, 2 * H, 18), normal(H, O, 19), rows(m, D)
    x[:, 40] = times
    wi[40] = 0
    assert error(x, gc.quantize_weight_int4(wi, 32), gc.quantize_weight_int4(wo, 32), "gelu") <= ALLOWED


def test_rows_of_all_sizes():
    """Rows that follow the gate and the other weights closely, rows that hardly meet any, and rows of zeros, side by side."""
    wi, wo, x = normal(256, 2 * 96, 20), normal(96, 40, 21), rows(200, 256).float()
    x[1::5] = wi[:, 5] * 1000
    x[2::5] = wi[:, 96 + 5] * 1e-3
    x[3::5, 1:] = 0
    x[4::5] = 0
    q, o, x = gc.quantize_weight_int4(wi, 32), gc.quantize_weight_int4(wo, 32), x.bfloat16()
    for first in range(4):
        got = gc.gated_ffn_int4(x, q, o)[first::5]
        G, U = (x[first::5].double() @ q.dequantize().double()).split(96, 1)
        assert rms(got, (act64("silu", G)[0] * U) @ o.dequantize().double()) <= ALLOWED
    assert not gc.gated_ffn_int4(x, q, o)[4::5].any()


def test_columns_of_zeros_and_a_weight_of_zeros():
    wi, wo = normal(256, 2 * 96, 8), normal(96, 40, 9)
    wi[:, :40] = 0
    wi[:, 96 + 50:] = 0
    wi[:, 41] *= 300
    for w in (wi, torch.zeros_like(wi)):
        q, o = gc.quantize_weight_int4(w, 32), gc.quantize_weight_int4(wo, 32)
        got = gc.gated_ffn_int4(rows(200, 256), q, o)
        if w.any():
            assert error(rows(200, 256), q, o, "silu") <= ALLOWED
        else:
            assert not got.any()


@pytest.mark.parametrize("h", [96, 100, 267])
def test_large_columns_in_every_place(h):
    """First, last, on either side of the halves' border, alone in a group."""
    for at in (0, h - 1, h, 2 * h - 1, h // 2):
        wi, wo = normal(512, 2 * h, 10), normal(h, 64, 11)
        wi[:, at] *= 1000
        wo[at % h] = 0
        assert error(rows(130, 512), gc.quantize_weight_int4(wi, 64), gc.quantize_weight_int4(wo, 64), "relu") <= ALLOWED
