"""Served models that were pickled before they had a choice of bits."""
import io

import pytest
import torch

import graphcuda_b200 as gc
from graphcuda_b200.models import ResidualGCN


def before_the_choice(served):
    """The model as its pickle was then: without ``bits``."""
    for m in (served, *served.blocks):
        m.__dict__.pop("bits", None)
    buf = io.BytesIO()
    torch.save(served, buf)
    buf.seek(0)
    return torch.load(buf, weights_only=False)


def test_serve_in_8_bits():
    served = before_the_choice(ResidualGCN(20, 64, 2, 7).for_serving())
    assert served.bits == 8 and served.for_serving() is served and served.for_serving(8) is served
    with pytest.raises(RuntimeError, match="8 bits"):
        served.for_serving(4)


@pytest.mark.gpu
def test_give_the_same_answers():
    torch.manual_seed(0)
    model = ResidualGCN(20, 64, 2, 7).cuda().for_serving()
    adj = gc.normalized_adjacency(torch.randint(0, 100, (2, 500), device="cuda"), 100)
    x = torch.randn(100, 20, device="cuda")
    want = model(x, adj)
    assert torch.equal(before_the_choice(model)(x, adj), want)
