"""How exact the linear layer is in fp32, and its activations value by value.

Products, relative 2-norms, derived:
  * three bf16 planes leave 2^-27 of an operand and the dropped products 2^-25 of a term, of random sign;
  * the tensor cores' addition truncates, 16 products at a time; k is cut at 512, which is 32 additions of
    0.72 * 2^-24 of the running sum in the mean, in the mean over a sum of random terms 2/3 of the whole:
    9.2e-7.  fp32 additions of the parts round to nearest.  BOUND = 2^-20 = 9.5e-7, and twice that where an
    activation's own error (below) and slope (1.13 at most) come to it, or cancellation in its range.
The model below takes the planes apart on the host: with two in place of three the bound does not hold.

Activations, one value each, relative to the parts they are made of.  exp by ex2: 2^-22 and its argument's rounding,
2^-23 times the argument; reciprocals 2^-23; the fit under the normal distribution function 2.2e-7, and its
argument's rounding three times 2^-23.
"""
import math

import pytest
import torch

gpu = pytest.mark.gpu
F32 = torch.float32
BOUND = 2.0 ** -20
ACTS = {"none": lambda x: x, **{n: getattr(torch.nn.functional, n) for n in ("relu", "silu", "gelu")}}


@pytest.fixture(scope="module", autouse=True)
def _built():
    import build
    build.build()
    build.build_entry()


def api():
    import qr_b200
    return qr_b200


def make(m, k, n, device):
    gen = torch.Generator(device=device).manual_seed(8)
    r = lambda *s: torch.randn(*s, generator=gen, device=device)
    return r(m, k), r(n, k) / math.sqrt(k), 0.5 * r(n), r(m, n), r(m, n)


def rel(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


SIZES = [(1, 4096, 600), (4, 1432, 200), (40, 1432, 300), (130, 512, 256), (300, 1432, 512), (300, 4100, 200),
         (1024, 8192, 2048), (2100, 600, 2100)]


@gpu
@pytest.mark.parametrize("size", SIZES)
def test_products_in_fp32(size):
    x, w, b, pre, dy = make(*size, "cuda")
    for act in ACTS:
        y, p = api().linear(x, w, b, activation=act, return_pre=True)
        want = x.double() @ w.double().T + b.double()
        assert rel(p, want) <= BOUND, rel(p, want)
        assert rel(y, ACTS[act](want)) <= (BOUND if act in ("none", "relu") else 2 * BOUND), act
        leaf = pre.double().requires_grad_()
        dp = torch.autograd.grad(ACTS[act](leaf), leaf, dy.double())[0]
        dx, dw, db = api().linear_backward(dy, x, w, activation=act, pre=pre, with_bias=True)
        # a sum that cancels is measured against the root of its squared terms
        for name, got, a, c in (("dx", dx, dp, w.double()), ("dw", dw, dp.T, x.double())):
            room = torch.maximum((a @ c).norm(), (a.square() @ c.square()).sum().sqrt())
            assert (got.double() - a @ c).norm() <= 2 * BOUND * room, (act, name)
        # fp32 sums of 8 rows, 8 of those and then of the blocks of 64, rounded to nearest: at most 16 + m / 512 + 8
        # additions of 2^-24 of what they add up; dp itself is slope's 2^-21 off
        room = (24 + size[0] / 512) * 2.0 ** -24 * dp.abs().sum(0).norm() + 2 * BOUND * dp.norm()
        assert (db.double() - dp.sum(0)).norm() <= room, act


def split(x, count):
    out = []
    for _ in range(count):
        out.append(x.float().bfloat16().double())
        x = x - out[-1]
    return out


@pytest.mark.parametrize("size", [(60, 512, 70), (40, 1432, 40)])
def test_two_planes_are_seen(size):
    x, w = (t.double() for t in make(*size, "cpu")[:2])
    off = {}
    for planes in (2, 3):
        a, c = split(x, planes), split(w, planes)
        off[planes] = rel(sum(a[i] @ c[j].T for i in range(planes) for j in range(planes - i)), x @ w.T)
    assert off[2] > BOUND and off[3] <= BOUND / 16, off


# ---- activations ----
def values():
    big = torch.linspace(-14, 14, 2000, dtype=torch.float64)
    tiny = torch.logspace(-12, -1, 100, dtype=torch.float64)
    return torch.cat([big, tiny, -tiny, torch.tensor([0.0, -0.0, 50.0, -50.0, 90.0, -90.0], dtype=torch.float64)]).float().cuda()


def tail(x):
    """The normal distribution's mass beyond |x|, and how far off its relative value may be."""
    return 0.5 * torch.special.erfc(x.abs() * math.sqrt(0.5)), 2.2e-7 + 2.0 ** -22 + 4 * 2.0 ** -23 + x.square() * 2.0 ** -23


def exp_off(x):
    return 2.0 ** -22 + x.abs() * 2.0 ** -23


def check(x, got, want, room, what):
    """A factor (the sigmoid, the tail, the density) below fp32's smallest normal value, 2^-126, is flushed to zero by
    the approximate exponential and reciprocal; times x, or added to it, that is up to (1 + |x|) 2^-126 of a result:
    silu(-90) = -90 * 8.2e-40 = -7.4e-38 comes out as 0, within 91 * 1.2e-38."""
    off, room = (got.double() - want).abs(), room + (1 + x.abs()) * 2.0 ** -126
    worst = (off / room).argmax()
    assert (off <= room).all(), (what, worst.item(), want[worst].item(), off[worst].item(), room[worst].item())


# rows, k: few rows; operands in exchanged places; tiles; k in parts, which the adding kernel joins
PATHS = [(1, 16), (40, 16), (200, 16), (200, 1100)]


@gpu
@pytest.mark.parametrize("m,k", PATHS)
def test_activations_value_by_value(m, k):
    v = values()
    n = v.numel()
    x, w = torch.zeros(m, k, device="cuda"), torch.ones(n, k, device="cuda")
    d = v.double()
    beyond, off = tail(d)
    phi = torch.where(d < 0, beyond, 1 - beyond)
    s = torch.sigmoid(d)
    half = 2.0 ** -23      # roundings of the last multiplications and additions
    want = {"gelu": (d * phi, (d * beyond * off).abs() + 2 * half * (d * phi).abs()),
            "silu": (d * s, (d * s * ((1 - s) * exp_off(d) + 3 * half)).abs())}
    for act, (y, room) in want.items():
        got, pre = api().linear(x, w, v, activation=act, return_pre=True)
        assert torch.equal(pre, v.expand(m, n))
        assert torch.equal(got, got[:1].expand(m, n))
        check(d, got[0], y, room, act)


@gpu
def test_slopes_value_by_value():
    v = values()
    d = v.double()
    beyond, off = tail(d)
    phi, half = torch.where(d < 0, beyond, 1 - beyond), 2.0 ** -23
    density = torch.exp(-0.5 * d.square()) / math.sqrt(2 * math.pi)
    s = torch.sigmoid(d)
    ds = (1 - s) * exp_off(d) + 2 * half
    want = {"gelu": (phi + d * density, beyond * off + 2 * half * phi + (d * density).abs() *
                     (exp_off(0.5 * d.square()) + d.square() * half + 3 * half)),
            # s (1 + x (1 - s)): s twice, and 1 - s, which cancels
            "silu": (s * (1 + d * (1 - s)), s * (ds * (1 + (d * (1 - s)).abs() + (d * s).abs()) + 3 * half * (1 + d.abs())))}
    w = torch.ones(v.numel(), 8, device="cuda")
    for act, (slope, room) in want.items():
        _, _, db = api().linear_backward(torch.ones(1, v.numel(), device="cuda"), torch.zeros(1, 8, device="cuda"), w,
                                         activation=act, pre=v[None], with_dx=False, with_dw=False, with_bias=True)
        check(d, db, slope, room, act)
