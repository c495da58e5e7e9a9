"""Weights without inputs or outputs, in 4 bits."""
import pytest
import torch

import graphcuda_b200 as gc


@pytest.mark.parametrize("k,n", [(64, 0), (0, 5), (0, 0)])
@pytest.mark.parametrize("zeros", [False, True])
def test_quantised(k, n, zeros):
    w = gc.quantize_weight_int4(torch.ones(k, n), 32, zeros)
    assert (w.in_features, w.out_features) == (k, n)
    assert w.dequantize().shape == (k, n)


def test_a_block_without_hidden_columns():
    block = gc.GatedFFN(16, 0, 8).for_serving(bits=4)
    assert block.w_in.out_features == 0 and block.w_out.in_features == 0
