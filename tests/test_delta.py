"""The gated delta rule (qr_b200.gated_delta_rule, its backward pass and its single-token step)
against the token-by-token recurrence in 64 bits (oracle/delta_oracle.py).

Tolerances, all relative 2-norms of a whole output (derived, not fitted):
  * a result rounded to type t is off by at most finfo(t).eps / 2 of each value;
  * fp32 operands are split into bf16 pieces: two pieces (16-bit types, forward) leave 2^-18 of each
    operand and the dropped product as much, 3 * 2^-18 a product.  A state goes through three dependent
    products a chunk (with S, with X, with K^T) and the triangular factor X, whose row sums stay below 8
    for the keys used here: 3 * 3 * 2^-18 * 8 < 2^-11 in the worst case and, the errors being of random
    sign over the 64 or more terms of each sum, an eighth of it: 2^-14 is asked;
  * three pieces (fp32 and every backward recurrence) leave 2^-27; fp32 sums of up to 128 + 64 terms,
    three dependent products and X's sums: 192 * 2^-24 * 3 / 2 < 2^-15 at worst, 2^-15 is asked;
  * dg is a difference of sums over a chunk: its error is measured against those sums
    (sqrt(64) times the norms of o.do and v.dv, and <S, dS>), not against dg.
"""
import math

import pytest
import torch

from oracle import delta_oracle as D

gpu = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
STATE_TOL = {BF: 2.0 ** -14, HF: 2.0 ** -14, F32: 2.0 ** -15}
BACK_TOL = 2.0 ** -15


@pytest.fixture(scope="module", autouse=True)
def _built():
    import build
    build.build()
    build.build_entry()


def api():
    import qr_b200
    return qr_b200


def tol(dtype, internal):
    return (torch.finfo(dtype).eps / 2 if dtype != F32 else 0.0) + internal


def rel(x, ref):
    x, ref = x.double().cpu(), ref.double().cpu()
    n = ref.norm().item()
    d = (x - ref).norm().item()
    return d / n if n else d


def make(batch, time, hk, hv, dk, dv, dtype, seed=0, device="cuda"):
    gen = torch.Generator(device=device).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device=device)
    unit = lambda x: (x / x.norm(dim=-1, keepdim=True).clamp_min(1e-6)).to(dtype)
    q, k = (unit(torch.nn.functional.silu(r(batch, time, hk, dk) + 0.2)) for _ in range(2))
    v = r(batch, time, hv, dv).to(dtype)
    g = -torch.nn.functional.softplus(r(batch, time, hv) - 1)
    beta = torch.sigmoid(r(batch, time, hv))
    return q, k, v, g, beta


def states(n, hv, dk, dv, seed=1):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return 0.3 * torch.randn(n, hv, dk, dv, generator=gen, device="cuda")


def check_forward(x, init, offsets, o, s, scale=None):
    q, k, v, g, beta = x
    dtype = q.dtype
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    S0 = torch.zeros_like(s) if init is None else init
    for i in range(s.shape[0]):
        part = [t[i] if offsets is None else t[0, offsets[i]:offsets[i + 1]] for t in (*x, o)]
        ro, rs, _ = D.forward(*part[:5], scale, S0[i])
        if ro.numel():
            assert rel(part[5], ro) <= tol(dtype, STATE_TOL[dtype]), (i, rel(part[5], ro))
        assert rel(s[i], rs) <= STATE_TOL[dtype], (i, rel(s[i], rs))


def check_backward(grads, do, dS, x, init, offsets, scale=None):
    q, k, v, g, beta = x
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    n = g.shape[0] if offsets is None else len(offsets) - 1
    shape = (n, v.shape[2], q.shape[-1], v.shape[-1])
    S0 = torch.zeros(shape, device="cuda") if init is None else init
    dE = torch.zeros(shape, device="cuda") if dS is None else dS
    for i in range(n):
        cut = lambda t: t[i] if offsets is None else t[0, offsets[i]:offsets[i + 1]]
        args = [cut(t) for t in x]
        ref = D.backward(cut(do), dE[i], *args, scale, S0[i])
        o, S_end, _ = D.forward(*args, scale, S0[i])
        for name, got, want in zip(("dq", "dk", "dv"), grads[:3], ref[:3]):
            if want.numel():
                # dk is the sum of four products that may cancel to a quarter of their norm
                assert rel(cut(got), want) <= tol(q.dtype, 4 * STATE_TOL[q.dtype]), (i, name, rel(cut(got), want))
        if ref[4].numel():
            assert rel(cut(grads[4]), ref[4]) <= 4 * STATE_TOL[q.dtype], (i, "dbeta")
            terms = 8 * ((o * cut(do).double()).norm() + (args[2].double() * ref[2]).norm())
            terms = terms + (S_end * dE[i].double()).norm() * math.sqrt(args[0].shape[0]) + ref[3].norm()
            off = (cut(grads[3]).double() - ref[3]).norm()
            assert off <= BACK_TOL * terms, (i, "dg", (off / terms).item())
        if init is not None:
            assert rel(grads[5][i], ref[5]) <= BACK_TOL, (i, "dinitial_state")


SIZES = [  # batch, time, hk, hv, dk, dv
    (1, 1, 1, 1, 128, 128), (2, 2, 1, 2, 64, 64), (1, 63, 2, 2, 128, 128), (2, 64, 2, 4, 128, 64), (1, 65, 1, 3, 64, 128),
    (3, 130, 1, 1, 128, 256), (1, 257, 2, 2, 96, 80), (1, 100, 1, 2, 1, 1), (2, 70, 3, 3, 33, 31), (1, 190, 1, 1, 127, 33)]


@gpu
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("size", SIZES)
def test_forward(size, dtype):
    x = make(*size, dtype)
    b, t, hk, hv, dk, dv = size
    init = states(b, hv, dk, dv)
    o, s = api().gated_delta_rule(*x, initial_state=init)
    assert o.dtype == dtype and s.dtype == F32
    check_forward(x, init, None, o, s)
    o, s = api().gated_delta_rule(*x, scale=0.3)
    check_forward(x, None, None, o, s, 0.3)


@gpu
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("size", SIZES)
def test_backward(size, dtype):
    x = make(*size, dtype)
    b, t, hk, hv, dk, dv = size
    init, dS = states(b, hv, dk, dv), states(b, hv, dk, dv, 2)
    do = make(*size, dtype, seed=5)[2]
    grads = api().gated_delta_rule_backward(do, *x, initial_state=init, dfinal_state=dS)
    check_backward(grads, do, dS, x, init, None)
    again = api().gated_delta_rule_backward(do, *x, initial_state=init, dfinal_state=dS)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    grads = api().gated_delta_rule_backward(do, *x, scale=0.3)
    assert grads[5] is None
    check_backward(grads, do, None, x, None, None, 0.3)


LENS = [[64, 1, 0, 130, 63], [0, 0, 5], [200], [1] * 40, [0]]


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("pad", [0, 3, 200])
@pytest.mark.parametrize("lens", LENS)
def test_packed(lens, pad, dtype):
    offs = [0]
    for n in lens:
        offs.append(offs[-1] + n)
    total = offs[-1] + pad
    x = make(1, total, 2, 4, 64, 96, dtype)
    do = make(1, total, 2, 4, 64, 96, dtype, seed=5)[2]
    for t in (*x, do):
        t[:, offs[-1]:] = float("nan")          # nothing behind the last sequence is read
    init, dS = states(len(lens), 4, 64, 96), states(len(lens), 4, 64, 96, 2)
    for kind in (torch.int32, torch.int64):
        so = torch.tensor(offs, dtype=kind, device="cuda")
        o, s = api().gated_delta_rule(*x, initial_state=init, seq_offsets=so)
        check_forward(x, init, offs, o, s)
        assert (o[:, offs[-1]:] == 0).all()
    grads = api().gated_delta_rule_backward(do, *x, initial_state=init, seq_offsets=so, dfinal_state=dS)
    check_backward(grads, do, dS, x, init, offs)
    assert all((t[:, offs[-1]:] == 0).all() for t in grads[:5])
    out = (torch.full_like(x[2], 7.0), torch.empty_like(init))
    o, s = api().gated_delta_rule(*x, initial_state=init, seq_offsets=so, out=out)
    assert o.data_ptr() == out[0].data_ptr() and s.data_ptr() == out[1].data_ptr()
    assert (o[:, offs[-1]:] == 7).all()
    check_forward(x, init, offs, o, s)


@gpu
def test_wrong_offsets_stay_inside():
    """Offsets that leave the tensors or decrease give some result, and touch nothing outside."""
    x = make(1, 100, 1, 1, 64, 64, BF)
    guard = torch.full((300, 64), 5.0, dtype=BF, device="cuda")
    o = guard[100:200].view(1, 100, 1, 64)
    for offs in ([-50, 40, 1000], [90, 20, 95, 3, 100], [0, 2 ** 31 - 1], [200, 300], [0, 100, 0, 100, 0, 100]):
        so = torch.tensor(offs, dtype=torch.int32, device="cuda")
        s = torch.empty(len(offs) - 1, 1, 64, 64, device="cuda")
        api().gated_delta_rule(*x, seq_offsets=so, out=(o, s))
        torch.cuda.synchronize()
        assert (guard[:100] == 5).all() and (guard[200:] == 5).all()
    assert torch.isfinite(api().gated_delta_rule(*x)[0]).all()


@gpu
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_strided_views(dtype):
    """q, k, v as slices of one projection's rows, at an odd offset, and transposed batches."""
    b, t, hk, hv, dk, dv = 2, 75, 2, 4, 64, 48
    x = make(b, t, hk, hv, dk, dv, dtype)
    width = hk * dk * 2 + hv * dv
    for off in (0, 1):
        row = torch.zeros(b, t, width + 8, dtype=dtype, device="cuda")
        q = row[..., off:off + hk * dk].unflatten(-1, (hk, dk))
        k = row[..., off + hk * dk:off + 2 * hk * dk].unflatten(-1, (hk, dk))
        v = row[..., off + 2 * hk * dk:off + width].unflatten(-1, (hv, dv))
        gates = torch.zeros(b, t, hv, 2, device="cuda")
        views = (q, k, v, gates[..., 0], gates[..., 1])
        for dst, src in zip(views, x):
            dst.copy_(src)
        o, s = api().gated_delta_rule(*views)
        want = api().gated_delta_rule(*x)
        assert torch.equal(o, want[0]) and torch.equal(s, want[1])
        do = torch.randn_like(v.contiguous().float()).to(dtype)
        for a, c in zip(api().gated_delta_rule_backward(do.transpose(2, 3).contiguous().transpose(2, 3), *views),
                        api().gated_delta_rule_backward(do, *x)):
            assert a is None and c is None or torch.equal(a, c)
    tr = [t_.transpose(0, 1).contiguous().transpose(0, 1) for t_ in x]
    assert torch.equal(api().gated_delta_rule(*tr)[0], api().gated_delta_rule(*x)[0])


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_gates_at_their_ends(dtype):
    """g = -inf empties the state, beta = 0 writes nothing, beta = 2 with unit keys reflects, g > 0 grows."""
    x = make(1, 200, 1, 2, 64, 64, dtype)
    q, k, v, g, beta = x
    g[:, 70], g[:, 71], g[:, 130] = -math.inf, -1e30, 0.3
    beta[:, 10:20], beta[:, 90:100], beta[:, 100] = 0.0, 2.0, -1.0
    init, dS = states(1, 2, 64, 64), states(1, 2, 64, 64, 2)
    o, s = api().gated_delta_rule(*x, initial_state=init)
    check_forward(x, init, None, o, s)
    do = make(1, 200, 1, 2, 64, 64, dtype, seed=5)[2]
    grads = api().gated_delta_rule_backward(do, *x, initial_state=init, dfinal_state=dS)
    g64 = g.clone()
    g64[:, 70], g64[:, 71] = -200.0, -200.0     # exp is 0 in 64 bits' products too, and inf * 0 is not formed
    check_backward(grads, do, dS, (q, k, v, g64, beta), init, None)


@gpu
def test_nan_stays_in_its_sequence_and_behind_its_chunk():
    x = make(2, 200, 1, 1, 64, 64, BF)
    want, _ = api().gated_delta_rule(*x)
    x[2][0, 130, 0, 3] = float("nan")
    o, s = api().gated_delta_rule(*x)
    assert torch.equal(o[1], want[1]) and torch.equal(o[0, :128], want[0, :128])
    assert o[0, 131:, 0, 3].isnan().all() and s[0, 0, :, 3].isnan().all() and torch.isfinite(s[1]).all()
    x = make(1, 64, 1, 1, 64, 64, BF)
    x[1][0, 10, 0, 0] = math.inf
    assert not torch.isfinite(api().gated_delta_rule(*x)[0][0, 11:]).any()


@gpu
def test_gradients_against_differences():
    b, t, hk, hv, dk, dv = 1, 70, 1, 2, 16, 16
    x = make(b, t, hk, hv, dk, dv, F32)
    init = states(b, hv, dk, dv)
    do, dS = torch.randn(b, t, hv, dv, device="cuda"), torch.randn(b, hv, dk, dv, device="cuda")
    grads = api().gated_delta_rule_backward(do, *x, initial_state=init, dfinal_state=dS)

    def value(*a):
        o, S, _ = D.forward(*[y[0] for y in a[:5]], dk ** -0.5, a[5][0])
        return (o * do[0].double()).sum() + (S * dS[0].double()).sum()

    full = [y.double() for y in (*x, init)]
    for i, gr in enumerate(grads):
        step = torch.randn_like(full[i])
        h = 1e-5
        a, c = list(full), list(full)
        a[i], c[i] = full[i] + h * step, full[i] - h * step
        want = (value(*a) - value(*c)) / (2 * h)
        got = (gr.double() * step).sum()
        # the differences are good to h^2 and 1e-16 / h, the gradient to 2^-15 of its norm
        assert abs(got - want) <= 2.0 ** -15 * gr.double().norm() * step.norm() / math.sqrt(step.numel()) * 8 + 1e-6


@gpu
def test_autograd():
    x = make(1, 100, 2, 4, 64, 64, BF)
    init = states(1, 4, 64, 64)
    leaves = [t.clone().requires_grad_() for t in (*x, init)]
    o, s = api().gated_delta_rule(*leaves[:5], initial_state=leaves[5])
    do, dS = torch.randn_like(o), torch.randn_like(s)
    got = torch.autograd.grad((o, s), leaves, (do, dS))
    want = api().gated_delta_rule_backward(do, *x, initial_state=init, dfinal_state=dS)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    o, s = api().gated_delta_rule(*leaves[:5])
    got = torch.autograd.grad(s, leaves[:5], dS)
    want = api().gated_delta_rule_backward(torch.zeros_like(do), *x, dfinal_state=dS)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(ValueError, match="out"):
        api().gated_delta_rule(*leaves[:5], out=(o, s))
    with pytest.raises(RuntimeError, match="no gradient"):
        api().gated_delta_step(*[t[:, 0] for t in leaves[:5]], init)


@gpu
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("size", [(1, 1, 1, 128, 128), (5, 2, 6, 64, 100), (3, 1, 1, 33, 31), (2, 1, 2, 1, 1), (4, 2, 2, 128, 256)])
def test_step(size, dtype):
    b, hk, hv, dk, dv = size
    x = [t[:, 0] for t in make(b, 1, hk, hv, dk, dv, dtype)]
    x[3][0, 0] = -math.inf
    state = states(b, hv, dk, dv)
    before = state.clone()
    kept = torch.empty_like(state)
    o = api().gated_delta_step(*x, state, state_out=kept)
    assert torch.equal(state, before)
    o2 = api().gated_delta_step(*x, state)
    assert torch.equal(state, kept) and torch.equal(o, o2)
    for i in range(b):
        ro, rs, _ = D.forward(*[t[i][None] for t in x], dk ** -0.5, before[i])
        # fp32 sums of up to 128 terms: 128 * 2^-24 / 2 and a few roundings
        assert rel(o[i], ro[0]) <= tol(dtype, 2.0 ** -17)
        assert rel(state[i], rs) <= 2.0 ** -17


@gpu
def test_step_slots():
    b, hk, hv, dk, dv = 8, 1, 2, 64, 64
    x = [t[:, 0] for t in make(b, 1, hk, hv, dk, dv, BF)]
    pool = torch.randn(10, 3, hv, dk, dv, device="cuda")[:, 1]      # strided slots
    before = pool.clone()
    slots = torch.tensor([7, -1, 3, 7, 12, 0, -5, 9], dtype=torch.int32, device="cuda")
    o = api().gated_delta_step(*x, pool, slots=slots)
    assert (o[[1, 6]] == 0).all()                                   # padding
    assert o[[3, 4]].isnan().all()                                  # held already, outside
    live = [0, 2, 5, 7]
    want = before[slots[live].long()].clone()
    ow = api().gated_delta_step(*[t[live] for t in x], want)
    assert torch.equal(o[live], ow) and torch.equal(pool[slots[live].long()], want)
    rest = [1, 2, 4, 5, 6, 8]
    assert torch.equal(pool[rest], before[rest])


@gpu
def test_step_far_into_a_pool():
    """Slots whose offset passes 2^31 elements."""
    hv, dk, dv = 16, 128, 128
    n = 2 ** 31 // (hv * dk * dv) + 4
    pool = torch.empty(n, hv, dk, dv, device="cuda")
    pool[-1] = states(1, hv, dk, dv)[0]
    x = [t[:, 0] for t in make(1, 1, hv, hv, dk, dv, BF)]
    want = pool[-1:].clone()
    ow = api().gated_delta_step(*x, want)
    o = api().gated_delta_step(*x, pool, slots=torch.tensor([n - 1], dtype=torch.int32, device="cuda"))
    assert torch.equal(o, ow) and torch.equal(pool[-1], want[0])


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_prompt_then_tokens(dtype):
    """A prompt through the chunked form, then tokens through the step, is one sequence."""
    x = make(2, 100, 2, 4, 128, 128, dtype)
    whole_o, whole_s = api().gated_delta_rule(*x)
    o, s = api().gated_delta_rule(*[t[:, :90] for t in x])
    outs = [o] + [api().gated_delta_step(*[t[:, i] for t in x], s)[:, None] for i in range(90, 100)]
    assert rel(torch.cat(outs, 1), whole_o) <= 2 * tol(dtype, STATE_TOL[dtype])
    assert rel(s, whole_s) <= 2 * STATE_TOL[dtype]


@gpu
def test_streams_and_graphs():
    x = make(2, 150, 1, 2, 64, 64, BF)
    do = torch.randn_like(x[2])
    state = states(2, 2, 64, 64)
    want = api().gated_delta_rule(*x), api().gated_delta_rule_backward(do, *x)
    tok = [t[:, 0].contiguous() for t in x]
    kept = torch.empty_like(state)
    wo = api().gated_delta_step(*tok, state, state_out=kept)
    wk = kept.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = api().gated_delta_rule(*x)
    side.synchronize()
    assert torch.equal(got[0], want[0][0])
    graphs, res = [], []
    for _ in range(2):                       # two graphs that do not share a workspace
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res.append((api().gated_delta_rule(*x), api().gated_delta_rule_backward(do, *x),
                        api().gated_delta_step(*tok, state, state_out=kept)))
        graphs.append(gr)
    for _ in range(2):
        for gr, (f, bw, o) in zip(graphs, res):
            for t in (*f, *bw[:5], o, kept):
                t.fill_(3)
            gr.replay()
            torch.cuda.synchronize()
            assert torch.equal(f[0], want[0][0]) and torch.equal(f[1], want[0][1])
            assert all(torch.equal(a, b) for a, b in zip(bw[:5], want[1][:5]))
            assert torch.equal(o, wo) and torch.equal(kept, wk)


@gpu
def test_two_streams_at_once():
    """Calls that overlap on the device do not meet: each has its own workspace, and blocks that want the
    same tensor memory wait for it."""
    calls = [make(1, 700, 2, 8, 128, 128, BF, seed=i) for i in range(4)]
    want = [(*api().gated_delta_rule(*x), *api().gated_delta_rule_backward(x[2], *x)[:5]) for x in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for s, x in zip(streams, calls):
            with torch.cuda.stream(s):
                got.append((*api().gated_delta_rule(*x), *api().gated_delta_rule_backward(x[2], *x)[:5]))
    torch.cuda.synchronize()
    for i, res in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(res, want[i % 4])), i
    from qr_b200 import _lib
    assert _lib.lib().qrb_device_error() == 0


FIRST_CALL = """
import sys
sys.path.insert(0, {pkg!r})
import torch, qr_b200
r = lambda *s: torch.randn(*s, device="cuda")
q, k, v = (r(1, 100, 2, 64).bfloat16() for _ in range(3))
g, b = -r(1, 100, 2).abs(), r(1, 100, 2).sigmoid()
state, x, w = r(2, 2, 64, 64), r(200, 72).bfloat16(), r(96, 72).bfloat16()
dy = r(200, 96).bfloat16()
k = torch.nn.functional.normalize(k.float(), dim=-1).bfloat16()
torch.cuda.synchronize()
def run():
    return [*qr_b200.gated_delta_rule(q, k, v, g, b), *qr_b200.gated_delta_rule_backward(v, q, k, v, g, b)[:5],
            qr_b200.gated_delta_step(q[0, :2], k[0, :2], v[0, :2], g[0, :2], b[0, :2], state, state_out=state.clone()),
            qr_b200.linear(x, w), *qr_b200.linear_backward(dy, x, w)[:2], qr_b200.linear(x[:1], w)]
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = run()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, c) for a, c in zip(out, run()))
print("same")
"""


@gpu
def test_first_call_of_a_process_may_be_captured():
    import subprocess
    import sys

    from conftest import PKG
    r = subprocess.run([sys.executable, "-c", FIRST_CALL.format(pkg=str(PKG))], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]


@gpu
def test_final_state_over_initial_state():
    x = make(2, 90, 1, 2, 64, 96, BF)
    init = states(2, 2, 64, 96)
    want = api().gated_delta_rule(*x, initial_state=init)
    o = torch.empty_like(x[2])
    api().gated_delta_rule(*x, initial_state=init, out=(o, init))
    assert torch.equal(o, want[0]) and torch.equal(init, want[1])


@gpu
def test_far_strides():
    """Batch strides past 2^31 elements."""
    far = 2 ** 31 + 64
    x = make(2, 70, 1, 1, 64, 64, BF)
    want = api().gated_delta_rule(*x)
    wb = api().gated_delta_rule_backward(x[2], *x)
    big = torch.empty(far + 70 * 192 + 64, dtype=BF, device="cuda")
    views = []
    for i in range(3):
        v = big.as_strided((2, 70, 1, 64), (far, 192, 64, 1), 64 * i)
        v.copy_(x[i])
        views.append(v)
    got = api().gated_delta_rule(*views, *x[3:])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert all(torch.equal(a, b) for a, b in zip(api().gated_delta_rule_backward(views[2], *views, *x[3:])[:5], wb[:5]))


@gpu
def test_long_sequence_in_parts():
    """100,001 tokens in one call and in two with the state carried over: chunks lie differently, so values
    agree to the kernels' accuracy, not bit for bit."""
    x = make(1, 100001, 1, 1, 64, 64, BF)
    o, s = api().gated_delta_rule(*x)
    cut = 33333
    o1, s1 = api().gated_delta_rule(*[t[:, :cut] for t in x])
    o2, s2 = api().gated_delta_rule(*[t[:, cut:] for t in x], initial_state=s1)
    assert rel(torch.cat([o1, o2], 1), o) <= 2 * tol(BF, STATE_TOL[BF]) and rel(s2, s) <= 2 * STATE_TOL[BF]


# Few heads and long sequences, which run as segments side by side: two segments, many, a last one of one
# token, several sequences, two blocks of value columns, odd sizes, two segments on two thirds of the SMs.
LONG = [(1, 600, 1, 1, 64, 64), (1, 4097, 1, 2, 128, 128), (2, 1473, 1, 1, 33, 200), (3, 1025, 2, 4, 64, 31),
        (1, 3001, 1, 1, 128, 256), (1, 9999, 2, 2, 16, 16), (2, 1050, 16, 32, 32, 40),
        (2, 1300, 8, 16, 128, 20)]


@gpu
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("size", LONG)
def test_long(size, dtype):
    b, t, hk, hv, dk, dv = size
    x = make(*size, dtype)
    do = make(b, t, hk, hv, dk, dv, dtype, seed=5)[2]
    init, dS = states(b, hv, dk, dv), states(b, hv, dk, dv, 2)
    o, s = api().gated_delta_rule(*x, initial_state=init)
    check_forward(x, init, None, o, s)
    grads = api().gated_delta_rule_backward(do, *x, initial_state=init, dfinal_state=dS)
    check_backward(grads, do, dS, x, init, None)
    over = init.clone()
    api().gated_delta_rule(*x, initial_state=over, out=(torch.empty_like(o), over))
    assert torch.equal(over, s)
    again = api().gated_delta_rule_backward(do, *x, initial_state=init, dfinal_state=dS)
    assert all(torch.equal(a, c) for a, c in zip(grads, again))
    check_forward(x, None, None, *api().gated_delta_rule(*x))
    check_backward(api().gated_delta_rule_backward(do, *x), do, None, x, None, None)


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lens", [[0, 2500, 3, 1100, 0, 64, 700], [1, 1, 4000], [1500, 1500], [5000], [0, 0, 1216, 0]])
def test_long_packed(lens, dtype):
    test_packed(lens, 70, dtype)


@gpu
def test_long_decay_and_values_that_are_not_finite():
    """A closed gate empties the state between segments; a NaN stays behind its chunk, in its sequence."""
    x = make(2, 2000, 1, 1, 64, 64, BF)
    x[3][0, 500:1500:37] = -math.inf
    x[3][1, 700] = -1e30
    init = states(2, 1, 64, 64)
    o, s = api().gated_delta_rule(*x, initial_state=init)
    check_forward([t.clamp_min(-200) if i == 3 else t for i, t in enumerate(x)], init, None, o, s)
    x[2][0, 1300, 0, 3] = float("nan")
    p, r = api().gated_delta_rule(*x, initial_state=init)
    assert torch.equal(p[1], o[1]) and torch.equal(r[1], s[1]) and torch.equal(p[0, :1280], o[0, :1280])
    assert p[0, 1300:1301, 0, 3].isnan().all()


@gpu
@pytest.mark.parametrize("offs", [None, [0, 2500, 2500, 2503, 4097]])
def test_long_captured(offs):
    """Both passes in one graph, replayed with other values, beside the same calls on another stream."""
    x = make(1, 4097, 2, 2, 96, 64, BF)
    so = None if offs is None else torch.tensor(offs, device="cuda")
    n = 1 if offs is None else len(offs) - 1
    init, dS = states(n, 2, 96, 64), states(n, 2, 96, 64, 2)

    def both(x, init):
        return (*api().gated_delta_rule(*x, initial_state=init, seq_offsets=so),
                *api().gated_delta_rule_backward(x[2], *x, initial_state=init, seq_offsets=so, dfinal_state=dS))
    both(x, init)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        got = both(x, init)
    y, init2 = make(1, 4097, 2, 2, 96, 64, BF, seed=9), states(n, 2, 96, 64, 7)
    want = both(y, init2)
    for a, b in zip((*x, init), (*y, init2)):
        a.copy_(b)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        beside = both(y, init2)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(torch.equal(a, b) for a, b in zip(beside, want))


@gpu
def test_wrong_offsets_of_long_sequences_stay_inside():
    x = make(1, 2000, 1, 1, 64, 64, BF)
    guard = torch.full((6000, 64), 5.0, dtype=BF, device="cuda")
    o = guard[2000:4000].view(1, 2000, 1, 64)
    for offs in ([-50, 900, 100000], [1900, 20, 1950, 3, 2000], [0, 2 ** 31 - 1], [0, 2000, 0, 2000, 0, 2000], [5000, 6000]):
        so = torch.tensor(offs, dtype=torch.int32, device="cuda")
        s = torch.empty(len(offs) - 1, 1, 64, 64, device="cuda")
        api().gated_delta_rule(*x, seq_offsets=so, out=(o, s))
        api().gated_delta_rule_backward(x[2], *x, seq_offsets=so)
        torch.cuda.synchronize()
        assert (guard[:2000] == 5).all() and (guard[4000:] == 5).all()


@gpu
def test_many_short_sequences():
    n = 3000
    lens = [(i * 7) % 4 for i in range(n)]
    offs = [0]
    for m in lens:
        offs.append(offs[-1] + m)
    x = make(1, offs[-1], 1, 1, 16, 16, F32)
    o, s = api().gated_delta_rule(*x, seq_offsets=torch.tensor(offs, device="cuda"))
    for i in (0, 1, 2, 3, 1500, 2998, 2999):
        ro, rs, _ = D.forward(*[t[0, offs[i]:offs[i + 1]] for t in x], 0.25, torch.zeros(1, 16, 16, device="cuda"))
        assert rel(o[0, offs[i]:offs[i + 1]], ro) <= STATE_TOL[F32] and rel(s[i], rs) <= STATE_TOL[F32]


@gpu
def test_gradients_are_refused_under_capture():
    x = [t.requires_grad_() for t in make(1, 10, 1, 1, 64, 64, BF)]
    gr = torch.cuda.CUDAGraph()
    a = torch.zeros(1, device="cuda")
    with torch.cuda.graph(gr):
        a += 1
        with pytest.raises(RuntimeError, match="gated_delta_rule_backward"):
            api().gated_delta_rule(*x)
        with torch.no_grad():
            o, _ = api().gated_delta_rule(*x)
    gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(o, api().gated_delta_rule(*x)[0])


@gpu
def test_empty_calls():
    x = make(0, 5, 1, 2, 64, 64, BF)
    o, s = api().gated_delta_rule(*x)
    assert o.shape == (0, 5, 2, 64) and s.shape == (0, 2, 64, 64)
    x = make(2, 0, 1, 2, 64, 64, BF)
    init = states(2, 2, 64, 64)
    o, s = api().gated_delta_rule(*x, initial_state=init)
    assert o.shape == (2, 0, 2, 64) and torch.equal(s, init)
    assert (api().gated_delta_rule(*x)[1] == 0).all()
    dS = states(2, 2, 64, 64, 3)
    grads = api().gated_delta_rule_backward(x[2], *x, initial_state=init, dfinal_state=dS)
    assert torch.equal(grads[5], dS) and grads[0].shape == x[0].shape
    assert api().gated_delta_step(*[t[:0, 0] for t in make(1, 1, 1, 2, 64, 64, BF)], init).shape == (0, 2, 64)


# ---- refusals, before anything touches a device ----
def cpu_args(**change):
    a = dict(q=torch.zeros(2, 3, 1, 8), k=torch.zeros(2, 3, 1, 8), v=torch.zeros(2, 3, 2, 4), g=torch.zeros(2, 3, 2),
             beta=torch.zeros(2, 3, 2))
    a.update(change)
    return a


@pytest.mark.parametrize("change,error,match", [
    (dict(q=torch.zeros(2, 3, 1, 8, dtype=torch.float64)), TypeError, "q must be float32, bfloat16 or float16"),
    (dict(q=torch.zeros(2, 3, 8)), ValueError, "q must have shape"),
    (dict(v=torch.zeros(2, 3, 8)), ValueError, "v must have shape"),
    (dict(k=torch.zeros(2, 3, 1, 9)), ValueError, "k must have shape"),
    (dict(k=torch.zeros(2, 3, 1, 8).half()), TypeError, "k must be"),
    (dict(v=torch.zeros(2, 4, 2, 4)), ValueError, "v must have shape"),
    (dict(g=torch.zeros(2, 3, 2).half()), TypeError, "g must be"),
    (dict(g=torch.zeros(2, 3, 1)), ValueError, "g must have shape"),
    (dict(beta=torch.zeros(2, 3)), ValueError, "beta must have shape"),
    (dict(q=torch.zeros(2, 3, 2, 8), k=torch.zeros(2, 3, 2, 8), v=torch.zeros(2, 3, 3, 4), g=torch.zeros(2, 3, 3),
          beta=torch.zeros(2, 3, 3)), ValueError, "multiple of q's heads"),
    (dict(q=torch.zeros(2, 3, 1, 129), k=torch.zeros(2, 3, 1, 129)), ValueError, "1 to 128 columns"),
    (dict(v=torch.zeros(2, 3, 2, 257)), ValueError, "1 to 256 columns"),
    (dict(initial_state=torch.zeros(2, 2, 4, 8)), ValueError, "initial_state must have shape"),
    (dict(initial_state=torch.zeros(2, 2, 8, 4).half()), TypeError, "initial_state must be"),
    (dict(seq_offsets=torch.zeros(3, dtype=torch.int32)), ValueError, "batch 1"),
    (dict(seq_offsets=torch.zeros(3)), TypeError, "seq_offsets must be int32"),
    (dict(seq_offsets=torch.zeros(1, dtype=torch.int32)), ValueError, "seq_offsets must have shape"),
    (dict(), ValueError, "no CPU path"),
])
def test_refusals(change, error, match):
    a = cpu_args(**change)
    args = [a.pop(n) for n in ("q", "k", "v", "g", "beta")]
    with pytest.raises(error, match=match):
        api().gated_delta_rule(*args, **a)
    with pytest.raises(error, match=match):
        api().gated_delta_rule_backward(args[2], *args, **a)


def test_backward_refusals():
    a = cpu_args()
    with pytest.raises(ValueError, match="do must have shape"):
        api().gated_delta_rule_backward(torch.zeros(2, 3, 2, 5), **a)
    with pytest.raises(TypeError, match="do must be"):
        api().gated_delta_rule_backward(torch.zeros(2, 3, 2, 4).half(), **a)


@pytest.mark.parametrize("change,error,match", [
    (dict(q=torch.zeros(2, 3, 1, 8)), ValueError, "q must have shape"),
    (dict(k=torch.zeros(3, 1, 8)), ValueError, "k must have shape"),
    (dict(state=torch.zeros(1, 2, 8, 4)), ValueError, "a slot for each"),
    (dict(state=torch.zeros(2, 2, 8, 5)), ValueError, "state must have shape"),
    (dict(state=torch.zeros(2, 2, 4, 8).transpose(2, 3)), ValueError, "dense"),
    (dict(state=torch.zeros(1, 2, 8, 4).expand(2, 2, 8, 4)), ValueError, "overlap"),
    (dict(state=torch.zeros(2, 2, 8, 4).half()), TypeError, "state must be"),
    (dict(slots=torch.zeros(2, dtype=torch.int64)), TypeError, "slots must be"),
    (dict(slots=torch.zeros(3, dtype=torch.int32)), ValueError, "slots must have shape"),
    (dict(state_out=torch.zeros(3, 2, 8, 4)), ValueError, "state_out must have shape"),
    (dict(), ValueError, "no CPU path"),
])
def test_step_refusals(change, error, match):
    a = dict(q=torch.zeros(2, 1, 8), k=torch.zeros(2, 1, 8), v=torch.zeros(2, 2, 4), g=torch.zeros(2, 2),
             beta=torch.zeros(2, 2), state=torch.zeros(2, 2, 8, 4))
    a.update(change)
    with pytest.raises(error, match=match):
        api().gated_delta_step(**a)


def test_c_abi_refusals():
    """qrb_delta_*: wrong arguments are statuses with a message, found before the device is touched."""
    import ctypes

    from qr_b200 import _lib
    lib = _lib.lib()
    assert lib.qrb_delta_workspace_size(None, 0) == 0
    for fn in (lib.qrb_delta_forward, lib.qrb_delta_backward):
        assert fn(None, None, 0, None) == _lib.QRB_ERR_INVALID_ARG
    assert lib.qrb_delta_step(None, None) == _lib.QRB_ERR_INVALID_ARG
    assert _lib.last_error()[1] == "args is null"
    raw = ctypes.create_string_buffer(512)            # dtype 0, all sizes 0
    assert lib.qrb_delta_forward(ctypes.addressof(raw), None, 0, None) == _lib.QRB_ERR_INVALID_ARG
    assert "hv must be" in _lib.last_error()[1]


def test_header_and_binding_agree():
    import re

    from conftest import ROOT
    from qr_b200 import _lib
    names = re.findall(r"QRB_API\s+[\w\s\*]+?\b(qrb_\w+)\s*\(", (ROOT / "include" / "qrb200_nn.h").read_text())
    assert names
    for n in names:
        assert hasattr(_lib.lib(), n) and n in _lib.SIGNATURES, n
