"""The norm's kernels where a group of threads has several wide rows.

Tolerances are those of test_norm_gpu.py: under 64 roundings of 2^-24 of the summed magnitudes, 8e-6; a 16-bit result
is rounded once more (2^-8), an 8-bit one by half a step (2^-4, or 2^-10 scales below the smallest normal number).  The weight gradient
adds up to 4000 rows in float32: 2e-5 of the summed magnitudes."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
SUM = 8e-6
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8 * 1.01}


def _randn(shape, seed, dtype=F32):
    return torch.randn(shape, generator=torch.Generator("cuda").manual_seed(seed), device="cuda").to(dtype)


def _over(got, ref, tol):
    assert got.shape == ref.shape
    return float(((got.detach().double() - ref).abs() - tol).max())


@pytest.mark.parametrize("types", [(F32, F32, F32), (BF16, BF16, BF16), (BF16, F32, BF16)], ids=str)
@pytest.mark.parametrize("shape", [(2500, 1096), (4001, 2048), (1300, 4096), (2401, 5000), (1201, 8192), (4000, 1029), (1999, 1433),
                                   (1250, 4099), (1500, 1300)], ids=str)
def test_many_wide_rows(cuda, shape, types):
    import graphcuda_b200 as gc
    tx, ts, ty = types
    x, r, w = _randn(shape, 0, tx), 2 * _randn(shape, 1, ts), 1 + 0.2 * _randn(shape[1:], 2)
    dy, ds = _randn(shape, 3, ty), _randn(shape, 4, ts)
    leaves = [t.requires_grad_() for t in (x, w, r)]
    y, h = gc.rms_norm(*leaves, out_dtype=ty)
    grads = torch.autograd.grad((y, h), leaves, (dy, ds))
    x, w, r, dy, ds = (t.detach().double() for t in (x, w, r, dy, ds))
    hh = x + r
    c = 1 / (hh.square().mean(1, keepdim=True) + 1e-6).sqrt()
    hat = hh * c
    ref = hat * w
    assert _over(y, ref, (SUM + HALF[ty]) * ref.abs()) <= 0
    assert _over(h, hh, HALF[ts] * hh.abs()) <= 0
    gw = dy * w
    d = c * (gw - hat * (gw * hat).mean(1, keepdim=True)) + ds
    tol = SUM * (c * (gw.abs() + hat.abs() * (gw * hat).abs().mean(1, keepdim=True)) + ds.abs())
    assert _over(grads[0], d, tol + HALF[tx] * d.abs()) <= 0
    assert _over(grads[2], d, tol + HALF[ts] * d.abs()) <= 0
    assert _over(grads[1], (dy * hat).sum(0), 2e-5 * (dy * hat).abs().sum(0)) <= 0
    with torch.no_grad():
        y8, scale, h8 = gc.rms_norm_fp8(*leaves)
    assert torch.equal(h8, h)
    top = ref.abs().max(1).values / 448
    assert _over(scale, top, SUM * top) <= 0
    assert _over(y8.double() * scale.double()[:, None], ref, ref.abs() * (2.0 ** -4 + 1e-5) + top[:, None] * 2.0 ** -10) <= 0
