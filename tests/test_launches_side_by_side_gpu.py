"""One kernel launched by two threads at once with unlike amounts of shared memory: neither's call changes what the other's may have."""
import threading

import pytest
import torch

import graphcuda_b200 as gc
from tests.test_distill_gpu import make
from tests.test_int4_gpu import rows, weight

pytestmark = pytest.mark.gpu
DEV = "cuda"


def distill(M, C, k, dtype=torch.float32, grad=1.0):
    logits, top, index = make(M, C, k, distinct=False, dtype=dtype)
    factor = torch.tensor(grad, device=DEV)

    def call():
        x = logits.detach().requires_grad_()
        return torch.autograd.grad(gc.distill_loss(x, top, index, scale=0.1), x, factor)[0]
    return call


def linear(m, k, n):
    x, w = rows(m, k), weight(k, n)
    return lambda: gc.linear_int4(x, w)


def block(m, d, h, o):
    x, wi, wo = rows(m, d), weight(d, 2 * h), weight(h, o, seed=1)
    return lambda: gc.gated_ffn_int4(x, wi, wo)


PAIRS = [
    ("rows of few inputs and many", lambda: linear(1, 128, 16), lambda: linear(1, 2048, 4096)),
    ("two operands of rows", lambda: linear(12, 256, 64), lambda: linear(12, 8192, 512)),
    ("tens of rows", lambda: linear(24, 128, 64), lambda: linear(24, 4096, 256)),
    ("blocks", lambda: block(3, 128, 32, 32), lambda: block(3, 2048, 512, 256)),
    ("blocks of tens of rows", lambda: block(24, 128, 32, 32), lambda: block(24, 2048, 512, 256)),
    ("short lists and long, with the gradient", lambda: distill(40, 1000, 400), lambda: distill(40, 1000, 1000)),
    ("short lists and long, gradient by itself", lambda: distill(40, 1000, 400, grad=2.0), lambda: distill(40, 1000, 1000, grad=2.0)),
    ("rings beside short lists and long", lambda: distill(150, 5000, 4), lambda: distill(150, 5000, 256)),
]


@pytest.mark.parametrize("name,small,large", PAIRS, ids=[p[0] for p in PAIRS])
def test_two_threads(name, small, large):
    calls = (small(), large())
    wants = [f().clone() for f in calls]
    torch.cuda.synchronize()
    errors = []
    start = threading.Barrier(2)

    def work(f, want):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait(30)
                for i in range(1500):
                    got = f()
                    if i % 50 == 0 and not torch.equal(got, want):
                        errors.append("another result")
                        return
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(repr(e))

    threads = [threading.Thread(target=work, args=a) for a in zip(calls, wants)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
