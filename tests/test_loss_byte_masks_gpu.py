"""A row is selected by any byte that is not zero, and counts once."""
import pytest
import torch

import graphcuda_b200 as gc
from tests.test_distill_gpu import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("values", [(0, 1), (0, 255), (0, 2, 7)])
def test_default_scale(values):
    logits, top, index = make(30, 20, 3)
    mask = torch.tensor(values, dtype=torch.uint8, device="cuda")[torch.arange(30, device="cuda") % len(values)]
    labels = index[:, 0]
    for f in (lambda m: gc.distill_loss(logits, top, index, m), lambda m: gc.log_softmax_nll_loss(logits, labels, m)):
        assert torch.equal(f(mask), f(mask != 0))
