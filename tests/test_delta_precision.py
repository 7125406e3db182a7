"""How exact the gated delta rule's fp32 results are: final states, dbeta, dinitial_state and dg of every type, and
all results of fp32 calls.  Relative 2-norms of a whole result, derived:

  * Three bf16 pieces leave 2^-27 of an operand, and what the pieces cost altogether is below 1e-8 (the host model
    below takes every operand apart as the kernels do, with sums in 64 bits).  What is left is the tensor cores'
    addition, which truncates: 16 products at a time, so 8 additions for a sum of 128 terms and 4 for one of 64,
    each by 0.72 * 2^-24 of the running sum in the mean, which in the mean over a sum is 2/3 of the whole.
  * A chunk's state passes through K S0 (8), X F (4) and K^T W (4), its gradient through K dS' (8), P^T dO and X^T F
    (4 each) and Q^T and K^T (8 together): at most 24 additions, 24 * 0.72 * 2/3 * 2^-24 = 7e-7, which the factor
    I + X beta may double: BOUND = 2^-19 = 1.9e-6.  Later chunks see what the decay and the rule itself leave of it.
  * dg is a difference of sums of o do and v dV over up to 64 tokens and 8 (sqrt 64) times their norms is `terms`:
    o and dV are 12 * 0.72 * 2/3 * 2^-24 = 3.4e-7 off, and the tokens that are summed are 32 in the mean, which
    leaves 1 / sqrt 2 of the 8: 2.4e-7, and half of this again for <S, dS>: DG_BOUND = 2^-21 = 4.8e-7.

With one piece fewer anywhere the model is beyond these bounds, which it shows here too.
"""
import math

import pytest
import torch

import test_delta as T
from oracle import delta_oracle as D

gpu = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
BOUND, DG_BOUND = 2.0 ** -19, 2.0 ** -21
NAMES = ("dq", "dk", "dv", "dg", "dbeta", "dinitial_state")


@pytest.fixture(scope="module", autouse=True)
def _built():
    import build
    build.build()
    build.build_entry()


def make(batch, time, hk, hv, dk, dv, dtype, device):
    x = list(T.make(batch, time, hk, hv, dk, dv, dtype, seed=4, device=device))
    x[3] = x[3] * torch.linspace(0.05, 2.0, hv, device=device)          # heads that forget slowly and quickly
    gen = torch.Generator(device=device).manual_seed(6)
    r = lambda *s: torch.randn(*s, generator=gen, device=device)
    init, dS = 0.3 * r(batch, hv, dk, dv), 0.3 * r(batch, hv, dk, dv)
    return x, r(batch, time, hv, dv).to(dtype), init, dS


def reference(x, do, init, dS):
    """Results of one sequence in 64 bits, and what dg's error is measured against."""
    scale = x[0].shape[-1] ** -0.5
    o, S, _ = D.forward(*x, scale, init)
    grads = dict(zip(NAMES, D.backward(do, dS, *x, scale, init)))
    terms = 8 * ((o * do.double()).norm() + (x[2].double() * grads["dv"]).norm())
    terms = terms + (S * dS.double()).norm() * math.sqrt(x[0].shape[0])
    return dict(o=o, final_state=S, **grads), terms


def errors(got, want, terms):
    off = {n: (got[n].double() - want[n]).norm() for n in want}
    return {n: (off[n] / (terms if n == "dg" else want[n].norm())).item() for n in want}


def bound(name):
    return DG_BOUND if name == "dg" else BOUND


# ---- the kernels ----
SIZES = [(1, 300, 2, 2, 128, 128), (2, 130, 1, 2, 64, 64), (1, 257, 2, 4, 96, 80), (2, 64, 2, 2, 33, 200),
         (1, 1000, 1, 2, 128, 128), (1, 3000, 2, 2, 64, 96)]


@gpu
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("size", SIZES)
def test_results_in_fp32(size, dtype):
    x, do, init, dS = make(*size, dtype, "cuda")
    o, S = T.api().gated_delta_rule(*x, initial_state=init)
    grads = T.api().gated_delta_rule_backward(do, *x, initial_state=init, dfinal_state=dS)
    got = dict(o=o, final_state=S, **dict(zip(NAMES, grads)))
    for i in range(size[0]):
        want, terms = reference([t[i] for t in x], do[i], init[i], dS[i])
        for name, off in errors({n: t[i] for n, t in got.items()}, want, terms).items():
            if got[name].dtype == F32:
                assert off <= bound(name), (i, name, off)


# ---- a model of the pieces, on the host ----
def pieces(x, count):
    out = []
    for _ in range(count):
        out.append(x.float().bfloat16().double())
        x = x - out[-1]
    return out


def product(a, b, count):
    return sum(x @ y for i, x in enumerate(a) for j, y in enumerate(b) if i + j < count)


def model(q, k, v, g, beta, S, do, dS, inputs, chain, state, back):
    """One head of the chunked form, sums in 64 bits; pieces of q, k and dO, of X, F and W, of S0, P and u, and in the
    backward recurrence."""
    C, scale = 64, q.shape[-1] ** -0.5
    q, k, v, g, beta, S, do, dS = (t.double() for t in (q, k, v, g, beta, S, do, dS))
    t = lambda p: [m.T for m in p]
    chunks, got = [], {n: torch.zeros_like(m) for n, m in zip(("o", "dq", "dk", "dv", "dg", "dbeta"), (v, q, k, v, g, g))}
    for at in range(0, q.shape[0], C):
        sl = slice(at, min(at + C, q.shape[0]))
        n, G, b = sl.stop - at, g[sl].cumsum(0), beta[sl][:, None]
        decay = torch.where(torch.ones(n, n).tril() > 0, (G[:, None] - G).exp(), torch.zeros((), dtype=torch.float64))
        K, Q = pieces(k[sl], inputs), pieces(q[sl], inputs)
        M, P = product(K, t(K), 3) * decay.tril(-1), scale * product(Q, t(K), 3) * decay
        X = torch.linalg.solve_triangular(torch.eye(n, dtype=torch.float64) + M * b.T, -M, upper=False, unitriangular=True)
        gamma, tail, S0 = G.exp()[:, None], (G[-1] - G).exp()[:, None], pieces(S, state)
        e0 = v[sl] - gamma * product(K, S0, state)
        e = e0 + product(pieces(X, chain), pieces(b * e0, chain), chain)
        got["o"][sl] = scale * gamma * product(Q, S0, state) + product(pieces(P, state), pieces(b * e, state), state)
        before, S = S, gamma[-1] * S + product(t(K), pieces(tail * b * e, chain), chain)
        chunks.append((sl, K, Q, decay, P, X, gamma, tail, b, before, e, S))
    got["final_state"] = S
    for sl, K, Q, decay, P, X, gamma, tail, b, S0, e, S1 in reversed(chunks):
        d, u = pieces(do[sl], inputs), b * e
        du = product(t(pieces(P, back)), d, back) + tail * product(K, pieces(dS, back), back)
        du = du + product(t(pieces(X, back)), pieces(b * du, back), back)
        y = b * du
        sums = (got["o"][sl] * do[sl]).sum(1) - (v[sl] * y).sum(1)
        got["dg"][sl] = sums.flip(0).cumsum(0).flip(0) + (S1 * dS).sum()
        got["dbeta"][sl], got["dv"][sl] = (e * du).sum(1), y
        both = lambda m: pieces(m, back)
        Z = both(scale * decay * product(d, t(both(u)), back))
        N = -decay.tril(-1) * product(both(y), t(both(u)), back)
        got["dq"][sl] = scale * gamma * product(d, t(both(S0)), back) + product(Z, K, back)
        got["dk"][sl] = (tail * product(both(u), t(both(dS)), back) - gamma * product(both(y), t(both(S0)), back)
                         + product(t(Z), Q, back) + product(both(N + N.T), K, back))
        dS = (gamma[-1] * dS + product(t(Q), both(scale * gamma * do[sl]), back) - product(t(K), both(gamma * y), back))
    return dict(got, dinitial_state=dS)


# the piece counts of a call (inputs, chain, state, back), and which results show that one of them is missing
THREE = {BF: (1, 3, 3, 3), F32: (3, 3, 3, 3)}
FEWER = [(BF, (1, 2, 3, 3), ["final_state"]), (BF, (1, 3, 2, 3), ["dg"]),
         (BF, (1, 3, 3, 2), ["dbeta", "dg", "dinitial_state"]),
         (F32, (2, 3, 3, 3), ["final_state", "dq", "dv", "dbeta", "dinitial_state"]), (F32, (3, 2, 3, 3), ["final_state"]),
         (F32, (3, 3, 2, 3), ["o", "dg"]), (F32, (3, 3, 3, 2), ["dq", "dk", "dv", "dg", "dbeta", "dinitial_state"])]


def model_errors(size, dtype, counts):
    x, do, init, dS = make(*size, dtype, "cpu")
    x, do, init, dS = [t[0] for t in x], do[0], init[0], dS[0]
    want, terms = reference(x, do, init, dS)
    heads = [model(*[t[:, h] for t in x], init[h], do[:, h], dS[h], *counts) for h in range(size[3])]
    got = {n: torch.stack([h[n] for h in heads], 0 if "state" in n else 1) for n in want}
    return errors(got, want, terms)


MODEL_SIZES = [(1, 300, 2, 2, 128, 128), (1, 130, 2, 2, 64, 64)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("size", MODEL_SIZES)
def test_three_pieces_leave_room(size, dtype):
    for name, off in model_errors(size, dtype, THREE[dtype]).items():
        assert off <= bound(name) / 64, (name, off)


@pytest.mark.parametrize("dtype,counts,seen", FEWER)
@pytest.mark.parametrize("size", MODEL_SIZES)
def test_a_piece_fewer_is_seen(size, dtype, counts, seen):
    off = model_errors(size, dtype, counts)
    for name in seen:
        assert off[name] > bound(name), (name, off[name])
