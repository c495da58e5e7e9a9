"""Distillation loss of rows far from zero: softmax does not know a row's offset, so neither loss nor gradient may.

Tolerances are those of test_distill_gpu (the differences that the formula takes are exact beside their size, whatever the offset)."""
import pytest
import torch

import graphcuda_b200 as gc
from tests.test_distill_gpu import check, make

pytestmark = pytest.mark.gpu
DEV = "cuda"

# 8 threads a row; a warp; a CTA, of 128 threads and beside a long list; parts of a row; one pass, in short segments and in long ones; rows
# longer than the ring
FORMS = [(40, 47, 8), (40, 1000, 8), (40, 5001, 8), (150, 9000, 300), (40, 20_000, 8), (160, 9000, 8), (150, 40_001, 8), (148, 101_377, 8)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,C,k", FORMS)
@pytest.mark.parametrize("offset", [1e3, -1e4, 1e5, 1e6])
def test_offsets(M, C, k, offset, dtype):
    logits, top, index = make(M, C, k, seed=C, dtype=dtype)
    check((logits.float() + offset).to(dtype), top, index, temperature=1.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,C,k", FORMS)
@pytest.mark.parametrize("value,temperature", [(-1e4, 1.0), (-1e9, 1.0), (-1e9, 3.0), (1e9, 0.5), (-1e30, 1.0), (None, 7.0)])
def test_rows_of_one_value(M, C, k, value, temperature, dtype):
    """As a mask fills them: uniform."""
    _, top, index = make(M, C, k, seed=C, dtype=dtype)
    logits = torch.full((M, C), torch.finfo(dtype).min if value is None else value, dtype=dtype, device=DEV)
    check(logits, top, index, temperature=temperature)


@pytest.mark.parametrize("M,C,k", FORMS)
def test_low_temperatures(M, C, k):
    """What counts is the maximum over the temperature."""
    check(*make(M, C, k, seed=C), temperature=0.03)


@pytest.mark.parametrize("M,C,k", FORMS)
def test_rows_near_zero_and_far_from_it_together(M, C, k):
    """Every row by itself, and a row whose threads meet small maxima before large ones: it begins at -1e5 and ends at 20."""
    logits, top, index = make(M, C, k, seed=C)
    logits[1::4] += 1e5
    logits[2::4] -= 1e5
    logits[3::4] -= torch.linspace(1e5, -20, C, device=DEV)
    check(logits, top, index, temperature=2.0)


@pytest.mark.parametrize("M,C,k", [(160, 9000, 8), (150, 40_001, 8)])
def test_the_value_is_the_same_with_a_gradient_and_without(M, C, k):
    logits, top, index = make(M, C, k, seed=C)
    for offset in (0.0, 1e6, -1e8):
        z = logits + offset
        with torch.no_grad():
            value = float(gc.distill_loss(z, top, index))
        assert abs(float(gc.distill_loss(z.requires_grad_(), top, index)) - value) <= 1e-5 * abs(value)
