"""The linear layer over the whole range of fp32 values, and its activations value by value."""
import math

import pytest
import torch

gpu = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _built():
    import build
    build.build()
    build.build_entry()


def api():
    import qr_b200
    return qr_b200


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


@gpu
@pytest.mark.parametrize("m", [1, 5, 130])
def test_largest_values(m):
    """Values up to finfo.max, which the nearest bf16 value would take past it, are finite operands.  Few-term
    sums in fp32: the module's 2^-14 of the result."""
    k, n = 40, 24
    top = torch.finfo(F32).max
    g = gen()
    x = torch.randn(m, k, generator=g, device="cuda")
    x[:, 3], x[:, 17], x[0, 20] = -top, top * (1 - 2.0 ** -9), top * (1 - 2.0 ** -8)
    w = torch.randn(n, k, generator=g, device="cuda") * 2.0 ** -8
    dy = torch.randn(m, n, generator=g, device="cuda") * 2.0 ** -8
    close = lambda got, want: (got.double() - want).norm() <= 2.0 ** -14 * want.norm()
    assert close(api().linear(x, w), x.double() @ w.double().T)
    dx, dw, _ = api().linear_backward(dy, x, w)
    assert close(dw, dy.double().T @ x.double()) and close(dx, dy.double() @ w.double())
    dy[0, 5] = -top
    dx, dw, _ = api().linear_backward(dy, x * 2.0 ** -126, w)
    assert close(dx, dy.double() @ w.double())
    assert close(api().linear(w, x), w.double() @ x.double().T)
    x[0, 4] = math.inf                                                # which stays what it is
    y = api().linear(x, w.abs())
    assert (y[0] == math.inf).all() and torch.isfinite(y[1:]).all()
