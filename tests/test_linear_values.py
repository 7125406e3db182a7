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


@gpu
@pytest.mark.parametrize("dtype,m", [(HF, 2 ** 18), (BF, 2 ** 20)])
def test_sums_over_many_rows(dtype, m):
    """dw of many rows, of one sign each, where every SM has a tile of its own and nothing else cuts the sum.  The
    tensor cores' additions truncate, and what that takes off may be half of the output's rounding, eps / 4, in the
    mean; the rounding itself is at most eps / 2 of each value."""
    n, k, g = 2048, 1664, gen(1)
    dy, x = (torch.empty(m, c, dtype=dtype, device="cuda") for c in (n, k))
    for i in range(0, m, 2 ** 16):
        dy[i:i + 2 ** 16] = torch.rand(2 ** 16, n, generator=g, device="cuda") / 16
        x[i:i + 2 ** 16] = torch.rand(2 ** 16, k, generator=g, device="cuda") / 64
    _, dw, db = api().linear_backward(dy, x, torch.empty(n, k, dtype=dtype, device="cuda"), with_dx=False, with_bias=True)
    want = sum(a.double().T @ b.double() for a, b in zip(dy[:, :128].split(2 ** 16), x[:, -128:].split(2 ** 16)))
    eps = torch.finfo(dtype).eps
    off = dw[:128, -128:].double() / want - 1
    assert off.mean().abs() <= eps / 4 and off.abs().max() <= eps / 4 + eps / 2
    assert (db[:128].double() / sum(a.double().sum(0) for a in dy[:, :128].split(2 ** 16)) - 1).abs().max() <= eps / 2 + 2.0 ** -14
