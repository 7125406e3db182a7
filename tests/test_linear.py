"""The linear layer (qr_b200.linear, linear_backward) against 64-bit torch, and the layer it forms
with the gated delta rule.

Tolerances, relative 2-norms of a whole output, derived:
  * a result rounded to type t is off by at most finfo(t).eps / 2 of each value;
  * sums of the 16-bit types: exact products added 16 at a time by the tensor cores, which truncate:
    k / 16 additions of at most 2^-23 of the running sum, k <= 8192 here: 2^-14;
  * fp32: three bf16 planes (2^-27 an operand), the small products apart, and k / 16 additions with
    k <= 4096 to the large sum before fp32 addition takes over: 256 * 2^-23 = 2^-15; activations at
    most double a relative error (their slope stays below 1.13, cancellation against the residual
    the same);
  * backward, 16-bit types: dp is rounded once more, another eps / 2 of each term (check_sum).
"""
import math

import pytest
import torch

from oracle import delta_oracle as D

gpu = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
ACTS = {"none": lambda x: x, **{n: getattr(torch.nn.functional, n) for n in ("relu", "silu", "gelu")}}


@pytest.fixture(scope="module", autouse=True)
def _built():
    import build
    build.build()
    build.build_entry()


def api():
    import qr_b200
    return qr_b200


def tol(dtype, roundings=1):
    return 2.0 ** -14 if dtype == F32 else roundings * torch.finfo(dtype).eps / 2 + 2.0 ** -14


def rel(x, ref):
    x, ref = x.double(), ref.double()
    n, d = ref.norm().item(), (x - ref).norm().item()
    return d / n if n else d


def make(m, k, n, dtype, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    return ((r(m, k)).to(dtype), (r(n, k) / math.sqrt(k)).to(dtype), (0.5 * r(n)).to(dtype), r(m, n).to(dtype),
            r(m, n).to(dtype))


def check_sum(got, a, b, dtype, what):
    """got = a b, where a was rounded to the type first.  That changes each term a_ij b_jk by at most eps / 2 of
    itself, with independent signs: the sum by (eps / 2) sqrt(sum_j a_ij^2 b_jk^2 / 3) in the mean square, and
    twice the root without the 3 is 3.5 standard deviations for a single output; of whole outputs it is about
    twice their norm, unless the terms cancel (one output of 300 terms may be a twentieth of its root).  fp32
    operands are not rounded; their sums' 2^-14 takes eps / 2's place."""
    ref = a @ b
    term = tol(dtype, 0) if dtype == F32 else torch.finfo(dtype).eps / 2
    off = (got.double() - ref).norm().item()
    room = tol(dtype) * ref.norm().item() + 2 * term * (a.square() @ b.square()).sum().sqrt().item()
    assert off <= room, (*what, off, room)


def reference(x, w, b, act, res):
    p = torch.nn.functional.linear(x.double(), w.double(), None if b is None else b.double())
    y = ACTS[act](p)
    return p, y if res is None else y + res.double()


SIZES = [(1, 1, 1), (1, 64, 128), (1, 2048, 1111), (3, 65, 257), (16, 512, 512), (64, 100, 40), (65, 130, 66),
         (128, 8192, 64), (129, 64, 128), (130, 1001, 250), (255, 256, 256), (300, 72, 1032), (512, 352, 176), (300, 1, 1), (257, 3, 2), (140, 5, 300),
         (1000, 4100, 72), (2049, 128, 136)]


@gpu
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("size", SIZES)
def test_forward(size, dtype):
    x, w, b, res, _ = make(*size, dtype)
    for act in ACTS:
        for bias, r in ((b, res), (None, None)):
            y, pre = api().linear(x, w, bias, activation=act, residual=r, return_pre=True)
            rp, ry = reference(x, w, bias, act, r)
            assert y.dtype == dtype and rel(y, ry) <= tol(dtype), (act, rel(y, ry))
            assert rel(pre, rp) <= tol(dtype), (act, rel(pre, rp))
            assert torch.equal(y, api().linear(x, w, bias, activation=act, residual=r))


@gpu
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("size", SIZES)
def test_backward(size, dtype):
    x, w, b, pre, dy = make(*size, dtype)
    for act in ACTS:
        p = pre.double().requires_grad_()
        dp = torch.autograd.grad(ACTS[act](p), p, dy.double())[0]
        dx, dw, db = api().linear_backward(dy, x, w, activation=act, pre=pre, with_bias=True)
        check_sum(dx, dp, w.double(), dtype, (act, "dx"))
        check_sum(dw, dp.T, x.double(), dtype, (act, "dw"))
        # sums over m of terms of both signs: m additions of 2^-24 of their absolute sum
        room = tol(dtype) + 2.0 ** -24 * size[0] * dp.abs().sum(0).norm() / dp.sum(0).norm().clamp_min(1e-30)
        assert rel(db, dp.sum(0)) <= room, (act, "dbias")
        again = api().linear_backward(dy, x, w, activation=act, pre=pre, with_bias=True)
        assert all(torch.equal(a, c) for a, c in zip((dx, dw, db), again))
        only = api().linear_backward(dy, x, w, activation=act, pre=pre, with_dx=False)
        assert only[0] is None and only[2] is None and torch.equal(only[1], dw)
        only = api().linear_backward(dy, x, w, activation=act, pre=pre, with_dw=False, with_bias=True)
        assert only[1] is None and torch.equal(only[0], dx) and torch.equal(only[2], db)


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("m", [1, 40, 200])
def test_strides(m, dtype):
    x, w, b, res, dy = make(m, 96, 80, dtype)
    want = api().linear(x, w, b, activation="silu", residual=res)
    wd = api().linear_backward(dy, x, w, with_bias=True)
    for pad, off in ((8, 8), (3, 1), (1, 0)):
        def view(t):
            big = torch.full((t.shape[0], t.shape[1] + pad + off), float("nan"), dtype=dtype, device="cuda")
            big[:, off:off + t.shape[1]] = t
            return big[:, off:off + t.shape[1]]
        y = api().linear(view(x), view(w), b, activation="silu", residual=view(res))
        assert torch.equal(y, want)
        out = view(torch.zeros_like(res))
        assert api().linear(view(x), view(w), b, activation="silu", residual=view(res), out=out).data_ptr() == out.data_ptr()
        assert torch.equal(out, want)
        assert all(torch.equal(p, q) for p, q in zip(api().linear_backward(view(dy), view(x), view(w), with_bias=True), wd))
    tr = lambda t: t.t().contiguous().t()
    assert torch.equal(api().linear(tr(x), tr(w), b, activation="silu", residual=tr(res)), want)
    assert torch.equal(api().linear(x[:1].expand(m, -1), w), api().linear(x[:1].repeat(m, 1), w))
    inplace = res.clone()
    assert torch.equal(api().linear(x, w, b, activation="silu", residual=inplace, out=inplace), want)
    deep = x.reshape(m, 1, 96).expand(m, 2, 96)
    got = api().linear(deep, w, b)
    assert got.shape == (m, 2, 80) and torch.equal(got[:, 0], got[:, 1])


@gpu
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("size", [(300, 72, 1001), (129, 8, 257), (1023, 200, 13), (513, 64, 70)])
def test_rows_with_room_behind(size, dtype):
    """Rows that begin on 16 bytes and end inside a unit of them: what lies behind stays as it was."""
    m, k, n = size
    x, w, b, res, _ = make(m, k, n, dtype)
    ld = (n + 15) // 8 * 8
    big = [torch.full((m, ld), 7.0, dtype=dtype, device="cuda") for _ in range(2)]
    big[0][:, :n] = res
    for act in ("none", "gelu"):
        out = api().linear(x, w, b, activation=act, residual=big[0][:, :n], out=big[1][:, :n])
        assert rel(out, reference(x, w, b, act, res)[1]) <= tol(dtype)
        assert (big[1][:, n:] == 7).all()
        assert torch.equal(out, api().linear(x, w, b, activation=act, residual=res))


@gpu
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("m", [1, 40, 200])
def test_activations_at_their_ends(m, dtype):
    b = torch.tensor([math.inf, -math.inf, math.nan, 0.0, -0.0, 6e4, -6e4, 30.0, -30.0, 1e-4], device="cuda").to(dtype)
    x, w = torch.zeros(m, 16, dtype=dtype, device="cuda"), torch.ones(10, 16, dtype=dtype, device="cuda")
    for act in ACTS:
        y, want = api().linear(x, w, b, activation=act), ACTS[act](b.double())
        for i in (0, 2, 3, 4, 5, 6, 7, 8, 9):     # -inf: the limit or, as inf * 0, NaN
            got = y[:, i].double()
            assert got.isnan().all() if want[i].isnan() else torch.allclose(got, want[i], rtol=1e-2, atol=1e-6), (act, i)
        assert (y[:, 1].isnan() | (y[:, 1] == ACTS[act](b.double())[1].nan_to_num(0.0, 0.0, -math.inf))).all(), act


@gpu
def test_rows_are_independent():
    """Rows of the result come from their rows of x alone, whatever the others hold."""
    for m in (5, 300):
        x, w, b, res, _ = make(m, 200, 144, BF)
        want = api().linear(x, w, b, activation="gelu", residual=res)
        x[3], res[3] = float("nan"), math.inf
        got = api().linear(x, w, b, activation="gelu", residual=res)
        keep = [i for i in range(m) if i != 3]
        assert torch.equal(got[keep], want[keep]) and got[3].isnan().all()
        assert api().linear(x, w, b, activation="relu")[3].isnan().all()
    x = torch.tensor([[math.inf, 1.0], [1.0, 2.0]], device="cuda")
    y = api().linear(x, torch.ones(3, 2, device="cuda"))
    assert torch.equal(y, torch.tensor([[math.inf] * 3, [3.0] * 3], device="cuda"))


@gpu
def test_autograd():
    for dtype in (BF, F32):
        x, w, b, res, dy = make(70, 64, 48, dtype)
        leaves = [t.clone().requires_grad_() for t in (x, w, b, res)]
        y = api().linear(*leaves[:3], activation="gelu", residual=leaves[3])
        got = torch.autograd.grad(y, leaves, dy)
        y2, pre = api().linear(x, w, b, activation="gelu", residual=res, return_pre=True)
        want = (*api().linear_backward(dy, x, w, activation="gelu", pre=pre, with_bias=True), dy)
        assert torch.equal(y, y2) and all(torch.equal(p, q) for p, q in zip(got, want))
        leaf = w.clone().requires_grad_()
        assert torch.equal(torch.autograd.grad(api().linear(x, leaf), leaf, dy)[0], api().linear_backward(dy, x, w)[1])
    with pytest.raises(ValueError, match="out and return_pre"):
        api().linear(*leaves[:2], return_pre=True)


@gpu
def test_gradients_against_differences():
    x, w, b, res, dy = make(9, 7, 5, F32)
    for act in ("silu", "gelu"):
        _, pre = api().linear(x, w, b, activation=act, return_pre=True)
        grads = api().linear_backward(dy, x, w, activation=act, pre=pre, with_bias=True)
        value = lambda *a: (reference(*a, act, None)[1] * dy.double()).sum()
        full = [x.double(), w.double(), b.double()]
        for i, gr in enumerate(grads):
            step = torch.randn_like(full[i])
            up, down = list(full), list(full)
            up[i], down[i] = full[i] + 1e-5 * step, full[i] - 1e-5 * step
            want = (value(*up) - value(*down)) / 2e-5
            # differences: 1e-10 of third derivatives; gradient: 2^-14 of its norm times the step's
            assert abs(want - (gr.double() * step).sum()) <= 2.0 ** -14 * gr.double().norm() * step.norm() + 1e-7


@gpu
def test_streams_and_graphs():
    x, w, b, res, dy = make(200, 300, 130, BF)
    run = lambda: (api().linear(x, w, b, activation="silu", residual=res),
                   *api().linear_backward(dy, x, w, activation="silu", pre=res, with_bias=True),
                   api().linear(x[:1], w, b))
    want = [t.clone() for t in run()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    side.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    graphs, res_ = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res_.append(run())
        graphs.append(g)
    for _ in range(2):
        for g, r in zip(graphs, res_):
            for t in r:
                t.fill_(9)
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, c) for a, c in zip(r, want))
    from qr_b200 import _lib
    assert _lib.lib().qrb_device_error() == 0


@gpu
def test_far_strides():
    """Rows past 2^31 elements."""
    m, k, n = 200, 64, 96
    x, w, b, res, dy = make(m, k, n, BF)
    ld = 2 ** 31 // (m - 8) // 8 * 8
    big = torch.empty(ld * m, dtype=BF, device="cuda")
    xv = big.as_strided((m, k), (ld, 1))
    xv.copy_(x)
    out = big.as_strided((m, n), (ld, 1), 512)
    assert torch.equal(api().linear(xv, w, b, out=out), api().linear(x, w, b))
    assert all(torch.equal(p, q) for p, q in zip(api().linear_backward(dy, xv, w)[:2], api().linear_backward(dy, x, w)[:2]))
    assert torch.equal(api().linear(xv[-3:], w), api().linear(x[-3:], w))


@gpu
def test_empty():
    x, w, b, _, _ = make(4, 16, 8, BF)
    assert api().linear(x[:0], w, b).shape == (0, 8)
    dx, dw, db = api().linear_backward(torch.empty(0, 8, dtype=BF, device="cuda"), x[:0], w, with_bias=True)
    assert dx.shape == (0, 16) and (dw == 0).all() and (db == 0).all()


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape", [(2, 100, 1, 2), (1, 65, 2, 2)])
def test_layer(shape, dtype):
    """The operators together: projections, the gated delta rule, an output projection onto the residual
    stream; its value and every gradient, then the same layer token by token."""
    B, T, hk, hv = shape
    d, width = 64, 96
    gen = torch.Generator(device="cuda").manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    x = r(B, T, width).to(dtype)
    sizes = (hk * d, hk * d, hv * d)
    w = [(0.5 * r(n, width) / math.sqrt(width)).to(dtype) for n in (sum(sizes), 2 * hv)]
    bias, wo = (0.1 * r(sum(sizes))).to(dtype), (r(width, hv * d) / math.sqrt(hv * d)).to(dtype)
    dy = r(B, T, width).to(dtype)

    def gates(z):
        z = z if z.dtype == torch.float64 else z.float()
        return -torch.nn.functional.softplus(z[..., :hv]), torch.sigmoid(z[..., hv:])

    def layer(x, w0, w1, bias, wo, state=None):
        q, k, v = api().linear(x, w0, bias, activation="silu").split(sizes, -1)
        g, beta = gates(api().linear(x, w1))
        heads = lambda t, h: t.unflatten(-1, (h, d))
        if state is not None:
            o = api().gated_delta_step(heads(q, hk), heads(k, hk), heads(v, hv), g, beta, state, scale=0.1)
        else:
            o, _ = api().gated_delta_rule(heads(q, hk), heads(k, hk), heads(v, hv), g, beta, scale=0.1)
        return api().linear(o.flatten(-2), wo, residual=x)

    def layer64(x, w0, w1, bias, wo):
        q, k, v = torch.nn.functional.silu(x @ w0.T + bias).split(sizes, -1)
        g, beta = gates(x @ w1.T)
        heads = lambda t, h: t.unflatten(-1, (h, d)).repeat_interleave(hv // h, -2)
        q, k, v = heads(q, hk), heads(k, hk), heads(v, hv)
        S, outs = torch.zeros(B, hv, d, d, dtype=torch.float64, device="cuda"), []
        for t in range(T):
            S = g[:, t].exp()[..., None, None] * S
            u = beta[:, t][..., None] * (v[:, t] - torch.einsum("bhkv,bhk->bhv", S, k[:, t]))
            S = S + torch.einsum("bhk,bhv->bhkv", k[:, t], u)
            outs.append(0.1 * torch.einsum("bhkv,bhk->bhv", S, q[:, t]))
        return torch.stack(outs, 1).flatten(-2) @ wo.T + x

    args = [t.clone().requires_grad_() for t in (x, *w, bias, wo)]
    wide = [t.detach().double().requires_grad_() for t in args]
    y, y64 = layer(*args), layer64(*wide)
    # roundings on the way to y: q k v, o, y, each eps / 2 of its values, the first through the recurrence
    # (doubled: a state holds products of two rounded vectors); fp32: 2^-14 for each of the five operators
    room = {BF: 8 * torch.finfo(BF).eps / 2, F32: 5 * 2.0 ** -14}[dtype]
    assert rel(y, y64) <= room
    got, want = torch.autograd.grad(y, args, dy), torch.autograd.grad(y64, wide, dy.double())
    for name, a, c in zip("x w0 w1 bias wo".split(), got, want):
        assert rel(a, c) <= 3 * room, (name, rel(a, c))     # as many roundings again on the way back, twice met
    with torch.no_grad():
        state = torch.zeros(B, hv, d, d, device="cuda")
        steps = torch.stack([layer(x[:, t], *w, bias, wo, state) for t in range(T)], 1)
    assert rel(steps, y64) <= room


# ---- refusals, before anything touches a device ----
@pytest.mark.parametrize("change,error,match", [
    (dict(x=torch.zeros(4, 6, dtype=torch.float64)), TypeError, "x must be float32, bfloat16 or float16"),
    (dict(w=torch.zeros(5, 7)), ValueError, "w must have shape"),
    (dict(w=torch.zeros(5)), ValueError, "w must have shape"),
    (dict(w=torch.zeros(5, 6).half()), TypeError, "w must be"),
    (dict(x=torch.zeros(4, 0), w=torch.zeros(5, 0)), ValueError, "at least 1"),
    (dict(bias=torch.zeros(6)), ValueError, "bias must have shape"),
    (dict(bias=torch.zeros(5).half()), TypeError, "bias must be"),
    (dict(residual=torch.zeros(5)), ValueError, "residual must have shape"),
    (dict(activation="tanh"), ValueError, "activation must be"),
    (dict(out=torch.zeros(4, 6)), ValueError, "out must have shape"),
    (dict(out=torch.zeros(5, 4).t()), ValueError, "out must be contiguous"),
    (dict(), ValueError, "no CPU path"),
])
def test_refusals(change, error, match):
    a = dict(x=torch.zeros(4, 6), w=torch.zeros(5, 6))
    a.update(change)
    with pytest.raises(error, match=match):
        api().linear(**a)


@pytest.mark.parametrize("change,error,match", [
    (dict(dy=torch.zeros(4, 6)), ValueError, "dy must have shape"),
    (dict(dy=torch.zeros(4, 5).half()), TypeError, "dy must be"),
    (dict(activation="gelu"), ValueError, "needs pre"),
    (dict(activation="gelu", pre=torch.zeros(4, 4)), ValueError, "pre must have shape"),
    (dict(), ValueError, "no CPU path"),
])
def test_backward_refusals(change, error, match):
    a = dict(dy=torch.zeros(4, 5), x=torch.zeros(4, 6), w=torch.zeros(5, 6))
    a.update(change)
    with pytest.raises(error, match=match):
        api().linear_backward(**a)


def test_c_abi_refusals():
    import ctypes

    from qr_b200 import _lib
    lib = _lib.lib()
    for fn in (lib.qrb_linear_forward, lib.qrb_linear_backward):
        assert fn(None, None, 0, None) == _lib.QRB_ERR_INVALID_ARG
    raw = ctypes.create_string_buffer(512)
    assert lib.qrb_linear_forward(ctypes.addressof(raw), None, 0, None) == _lib.QRB_ERR_INVALID_ARG
    assert "k and n >= 1" in _lib.last_error()[1]
    assert lib.qrb_linear_workspace_size(ctypes.addressof(raw)) == 0
