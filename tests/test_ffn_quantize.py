"""quantize_weight_fp8 on the CPU: columns of every magnitude that float32 has."""
import pytest
import torch


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_columns_of_next_to_nothing(dtype):
    """A column whose scale is subnormal, and so coarse that its largest element is more than 448 of them, stays finite."""
    from graphcuda_b200 import quantize_weight_fp8
    w = torch.randn(50, 300, generator=torch.Generator().manual_seed(0), dtype=torch.float64)
    w = (w * torch.exp2(torch.linspace(-149, 100, 300, dtype=torch.float64))).to(dtype)
    w[:, 7] = 0
    w[:, :2] = torch.tensor([700, 1], dtype=torch.float64).mul(2.0 ** -149).to(dtype)
    w8, scale = quantize_weight_fp8(w)
    assert w8.shape == (300, 50) and w8.dtype == torch.float8_e4m3fn and scale.shape == (300,)
    value = w8.double() * scale.double()[:, None]
    assert torch.isfinite(value).all()
    wt = w.double().t()
    # half a step of the code; a scale of subnormal numbers is itself off by half of the smallest, 448 times
    err = (value - wt).abs() - wt.abs() * 2.0 ** -4 * 1.001 - scale.double()[:, None] * 2.0 ** -10 * 1.001 - 448 * 2.0 ** -150
    assert float(err.max()) <= 0


def test_columns_that_are_not_finite():
    from graphcuda_b200 import quantize_weight_fp8
    w = torch.randn(8, 4)
    w[2, 1], w[3, 2] = float("inf"), float("nan")
    w8, scale = quantize_weight_fp8(w)
    value = w8.float() * scale[:, None]
    assert torch.isfinite(value[[0, 3]]).all()
    assert not torch.isfinite(value[1, 2]) and torch.isnan(value[2, 3])
