"""Workloads of the library's sequence and projection operators, each in two forms.

The operators are the gated delta rule (a product of scaled Householder-like transforms applied
to a per-head state matrix) over whole sequences, its backward pass and its single-token step,
and the linear layer ``act(x w^T + b) + r`` with its backward pass.  ``run`` computes a case with
elementary torch operations in 32 bits while ``own`` is false, and through ``qr_b200`` when it is
true.  ``exact`` computes the same from the operators' definitions in 64 bits: token by token for
the delta rule.

Delta rule, per head, with S_0 given (S is dk x dv, g the logarithm of the decay):
    S~_t = exp(g_t) S_{t-1},  u_t = beta_t (v_t - S~_t^T k_t),  S_t = S~_t + k_t u_t^T,
    o_t = scale S_t^T q_t.
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False

_PKG = str(Path(__file__).resolve().parent.parent / "linalg-gpu-comp_b200")
_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
CHUNK = 64


def _api():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import qr_b200
    return qr_b200


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def _delta(name, kind, dtype, seqs, tokens, hk, hv, dk, dv, packed=False, pad=0):
    c = {"kind": kind, "dtype": dtype, "seqs": seqs, "tokens": tokens, "hk": hk, "hv": hv, "dk": dk, "dv": dv,
         "packed": packed, "pad": pad}
    return {"name": name, **c} if name else c


def _step(name, dtype, batch, slots, padded, hk, hv, dk, dv):
    c = {"kind": "step", "dtype": dtype, "batch": batch, "slots": slots, "padded": padded, "hk": hk, "hv": hv,
         "dk": dk, "dv": dv}
    return {"name": name, **c} if name else c


def _lin(name, kind, dtype, m, k, n, act, bias, residual):
    c = {"kind": kind, "dtype": dtype, "m": m, "k": k, "n": n, "act": act, "bias": bias, "residual": residual}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one sequence answering, token by token: latency only
        _step("step_one", "bf16", 1, 0, 0, 16, 16, 128, 128),
        # a serving batch over a pool of states, two q/k heads' worth of v heads each, some rows padding
        _step("step_pool", "bf16", 256, 300, 6, 8, 16, 128, 128),
        # a short prompt of one user
        _delta("prompt", "forward", "bf16", 1, 512, 8, 16, 128, 128),
        # prompts of very different lengths packed into one call, rows of padding behind them
        _delta("packed", "forward", "bf16", 24, 16384, 16, 32, 128, 128, packed=True, pad=37),
        # fp32 with head sizes and a length that no tile divides
        _delta("odd_fp32", "forward", "fp32", 3, 3 * 777, 5, 5, 96, 80),
        # a training batch's backward pass
        _delta("train", "backward", "bf16", 4, 8192, 16, 16, 128, 128),
        # packed training samples, small heads, shared q/k heads
        _delta("train_packed", "backward", "fp16", 7, 3001, 3, 6, 64, 64, packed=True),
        # the projection of one token
        _lin("linear_token", "linear", "bf16", 1, 2048, 8192, "silu", True, False),
        # the projection of a prompt or a training batch
        _lin("linear_batch", "linear", "bf16", 4096, 2048, 8192, "gelu", True, False),
        # sizes that no tile divides and rows that are not 16-byte aligned, joined to a residual stream
        _lin("linear_odd", "linear", "fp16", 777, 1001, 1111, "none", True, True),
        # a training batch's backward pass through activation, weight and bias
        _lin("linear_train", "linear_backward", "bf16", 8192, 2048, 2048, "silu", True, False),
        _lin("linear_train_odd", "linear_backward", "fp16", 1500, 500, 1100, "gelu", True, False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["step", "forward", "forward", "backward", "backward", "linear", "linear", "linear_backward"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "step":
        batch = _log(rng, 1, 256)
        hk = rng.choice([1, 2, 4, 8])
        return _step(None, dtype, batch, rng.choice([0, batch + _log(rng, 1, 40)]), rng.choice([0, batch // 8]),
                     hk, hk * rng.choice([1, 2]), rng.choice([64, 96, 128]), rng.choice([64, 100, 128]))
    if kind in ("forward", "backward"):
        hk = rng.choice([1, 2, 3, 4, 8])
        hv = hk * rng.choice([1, 2, 4] if hk < 8 else [1, 2])
        dk, dv = rng.choice([(64, 64), (128, 128), (128, 128), (96, 80), (40, 128)])
        top = 12000 if kind == "forward" else 6000
        if rng.random() < 0.5:
            seqs = _log(rng, 1, 30)
            return _delta(None, kind, dtype, seqs, max(seqs, _log(rng, 100, top)), hk, hv, dk, dv, True,
                          rng.choice([0, 5, 130]))
        seqs = _log(rng, 1, 8)
        return _delta(None, kind, dtype, seqs, seqs * _log(rng, 1, top // seqs), hk, hv, dk, dv)
    m = _log(rng, 1, 4096)
    k, n = _log(rng, 32, 2048), _log(rng, 32, 4096 if kind == "linear" else 2048)
    if rng.random() < 0.5:
        k, n = -(-k // 8) * 8, -(-n // 8) * 8
    return _lin(None, kind, dtype, m, k, n, rng.choice(["none", "relu", "silu", "gelu"]), rng.random() < 0.7,
                kind == "linear" and rng.random() < 0.4)


def _lengths(case):
    """Sequence lengths of a case: equal, or (packed) spread widely with an empty and a one-token sequence."""
    n, total = case["seqs"], case["tokens"]
    if not case["packed"]:
        return [total // n] * n
    rng = random.Random(total * 1009 + n)
    w = [rng.random() ** 3 + 0.01 for _ in range(n)]
    if n >= 3:
        w[n // 2] = 0.0
    if n >= 2:
        w[1] = 0.0
    scale = total / sum(w)
    lens = [int(x * scale) for x in w]
    if n >= 2:
        lens[1] = 1
    lens[0] += total - sum(lens)
    return lens


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _unit(shape, dk, gen, dtype):
    """Keys and queries as a model has them: SiLU outputs (mostly of one sign, so correlated), normalised."""
    x = torch.nn.functional.silu(torch.randn(*shape, dk, generator=gen, device="cuda") + 0.2)
    return (x / x.square().sum(-1, keepdim=True).add(1e-12).sqrt()).to(dtype)


def _gates(shape, heads, gen):
    rate = torch.exp(torch.empty(heads, device="cuda").uniform_(-3.0, 0.7, generator=gen))
    g = -rate * torch.nn.functional.softplus(torch.randn(*shape, heads, generator=gen, device="cuda") - 1.0)
    beta = torch.sigmoid(torch.randn(*shape, heads, generator=gen, device="cuda"))
    return g, beta


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(1000003 * seed + 17)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    dt = _DT[case["dtype"]]
    st = {"case": case}
    if case["kind"] in ("linear", "linear_backward"):
        m, k, n = case["m"], case["k"], case["n"]
        st["x"], st["w"] = rnd(m, k).to(dt), (rnd(n, k) / math.sqrt(k)).to(dt)
        st["bias"] = (0.5 * rnd(n)).to(dt) if case["bias"] else None
        st["residual"] = rnd(m, n).to(dt) if case["residual"] else None
        if case["kind"] == "linear_backward":
            st["dy"] = rnd(m, n).to(dt)
            # what the forward pass kept: the activation's argument
            st["pre"] = rnd(m, n).to(dt) if case["act"] != "none" else None
        return st
    hk, hv, dk, dv = case["hk"], case["hv"], case["dk"], case["dv"]
    if case["kind"] == "step":
        b = case["batch"]
        st["q"], st["k"] = _unit((b, hk), dk, gen, dt), _unit((b, hk), dk, gen, dt)
        st["v"] = rnd(b, hv, dv).to(dt)
        st["g"], st["beta"] = _gates((b,), hv, gen)
        rows = case["slots"] or b
        st["state"] = 0.3 * rnd(rows, hv, dk, dv)
        st["state_out"] = torch.zeros_like(st["state"])
        st["slots"] = None
        if case["slots"]:
            slots = torch.randperm(rows, generator=gen, device="cuda")[:b].to(torch.int32)
            if case["padded"]:
                slots[-case["padded"]:] = -1
            st["slots"] = slots
        return st
    lens = _lengths(case)
    shape = (1, case["tokens"] + case["pad"]) if case["packed"] else (case["seqs"], lens[0])
    st["q"], st["k"] = _unit((*shape, hk), dk, gen, dt), _unit((*shape, hk), dk, gen, dt)
    st["v"] = rnd(*shape, hv, dv).to(dt)
    st["g"], st["beta"] = _gates(shape, hv, gen)
    st["initial_state"] = 0.3 * rnd(case["seqs"], hv, dk, dv)
    st["seq_offsets"], st["lens"] = None, lens
    if case["packed"]:
        offs = [0]
        for n in lens:
            offs.append(offs[-1] + n)
        st["seq_offsets"] = torch.tensor(offs, dtype=torch.int32, device="cuda")
    if case["kind"] == "backward":
        st["do"] = rnd(*shape, hv, dv).to(dt)
        st["dfinal_state"] = 0.3 * rnd(case["seqs"], hv, dk, dv)
    return st


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(state):
    kind = state["case"]["kind"]
    if own:
        return _own(kind, state)
    return {"step": _plain_step, "forward": _plain_forward, "backward": _plain_backward, "linear": _plain_linear,
            "linear_backward": _plain_linear_backward}[kind](state)


def _own(kind, st):
    api = _api()
    if kind == "step":
        o = api.gated_delta_step(st["q"], st["k"], st["v"], st["g"], st["beta"], st["state"], slots=st["slots"],
                                 state_out=st["state_out"])
        return {"o": o, "state": st["state_out"]}
    if kind == "forward":
        o, s = api.gated_delta_rule(st["q"], st["k"], st["v"], st["g"], st["beta"], initial_state=st["initial_state"],
                                    seq_offsets=st["seq_offsets"])
        return {"o": o, "final_state": s}
    if kind == "backward":
        names = ("dq", "dk", "dv", "dg", "dbeta", "dinitial_state")
        return dict(zip(names, api.gated_delta_rule_backward(
            st["do"], st["q"], st["k"], st["v"], st["g"], st["beta"], initial_state=st["initial_state"],
            seq_offsets=st["seq_offsets"], dfinal_state=st["dfinal_state"])))
    c = st["case"]
    if kind == "linear":
        return api.linear(st["x"], st["w"], st["bias"], activation=c["act"], residual=st["residual"])
    dx, dw, db = api.linear_backward(st["dy"], st["x"], st["w"], activation=c["act"], pre=st["pre"],
                                     with_bias=c["bias"])
    return {"dx": dx, "dw": dw, "dbias": db} if c["bias"] else {"dx": dx, "dw": dw}


# ---- plain forms ---------------------------------------------------------------------------
def _rows(st, x):
    """(batch, time, heads, ...) or packed (1, tokens, heads, ...) -> (seqs, heads, chunks, CHUNK, ...), zero behind
    each sequence, in 32 bits."""
    lens = st["lens"]
    top = max(1, -(-max(lens) // CHUNK)) * CHUNK
    out = x.new_zeros((len(lens), top, *x.shape[2:]), dtype=torch.float32)
    if st["seq_offsets"] is None:
        out[:, :lens[0]] = x
    else:
        at = 0
        for i, n in enumerate(lens):
            out[i, :n] = x[0, at:at + n]
            at += n
    out = out.transpose(1, 2)
    return out.reshape(out.shape[0], out.shape[1], top // CHUNK, CHUNK, *out.shape[3:])


def _unrows(st, y, like):
    """The inverse of _rows, rounded to like's type; rows of padding are zero."""
    y = y.reshape(y.shape[0], y.shape[1], -1, *y.shape[4:]).transpose(1, 2)
    lens = st["lens"]
    if st["seq_offsets"] is None:
        return y[:, :lens[0]].to(like.dtype).contiguous()
    out = like.new_zeros((1, like.shape[1], *y.shape[2:]))
    at = 0
    for i, n in enumerate(lens):
        out[0, at:at + n] = y[i, :n].to(like.dtype)
        at += n
    return out


def _chunks(st):
    """What both passes need of every chunk: e = E0 + X (beta E0) solves the chunk's triangular system."""
    c = st["case"]
    group = c["hv"] // c["hk"]
    q = _rows(st, st["q"]).repeat_interleave(group, 1)
    k = _rows(st, st["k"]).repeat_interleave(group, 1)
    v, g, beta = _rows(st, st["v"]), _rows(st, st["g"]), _rows(st, st["beta"])
    G = g.double().cumsum(-1)
    low = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=g.device).tril()
    D = torch.where(low, (G[..., :, None] - G[..., None, :]), -math.inf).exp().float()
    gamma, tail = G.exp().float(), (G[..., -1:] - G).exp().float()
    M = (k @ k.transpose(-1, -2)) * D.tril(-1)
    X = -M
    for i in range(1, CHUNK):
        X[..., i, :] = -M[..., i, :] - ((M[..., i, :i] * beta[..., :i])[..., None, :] @ X[..., :i, :])[..., 0, :]
    P = (q @ k.transpose(-1, -2)) * D / math.sqrt(c["dk"])
    return q, k, v, beta, D, gamma, tail, X, P


def _plain_forward(st, keep=False):
    c = st["case"]
    scale = 1 / math.sqrt(c["dk"])
    q, k, v, beta, D, gamma, tail, X, P = ch = _chunks(st)
    S = st["initial_state"].float()
    o, starts, es = torch.empty_like(v), [], []
    for i in range(v.shape[2]):
        starts.append(S)
        E0 = v[:, :, i] - gamma[:, :, i, :, None] * (k[:, :, i] @ S)
        e = E0 + X[:, :, i] @ (beta[:, :, i, :, None] * E0)
        u = beta[:, :, i, :, None] * e
        if keep:
            es.append(e)
        else:
            o[:, :, i] = scale * gamma[:, :, i, :, None] * (q[:, :, i] @ S) + P[:, :, i] @ u
        S = gamma[:, :, i, -1, None, None] * S + k[:, :, i].transpose(-1, -2) @ (tail[:, :, i, :, None] * u)
    if keep:
        return ch, torch.stack(starts, 2), torch.stack(es, 2), S
    return {"o": _unrows(st, o, st["v"]), "final_state": S}


def _plain_backward(st):
    c = st["case"]
    scale = 1 / math.sqrt(c["dk"])
    (q, k, v, beta, D, gamma, tail, X, P), S0, e, S_end = _plain_forward(st, keep=True)
    do = _rows(st, st["do"])
    dS = st["dfinal_state"].float()
    T = lambda x: x.transpose(-1, -2)
    bt, ga, ta = beta[..., None], gamma[..., None], tail[..., None]
    ends, ys, dus = [None] * v.shape[2], [None] * v.shape[2], [None] * v.shape[2]
    for i in range(v.shape[2] - 1, -1, -1):
        ends[i] = dS
        du = T(P[:, :, i]) @ do[:, :, i] + ta[:, :, i] * (k[:, :, i] @ dS)
        du = du + T(X[:, :, i]) @ (bt[:, :, i] * du)
        dus[i], ys[i] = du, bt[:, :, i] * du
        dS = (gamma[:, :, i, -1, None, None] * dS + T(scale * ga[:, :, i] * q[:, :, i]) @ do[:, :, i]
              - T(ga[:, :, i] * k[:, :, i]) @ ys[i])
    dE, y, du = torch.stack(ends, 2), torch.stack(ys, 2), torch.stack(dus, 2)
    u = bt * e
    Z = scale * D * (do @ T(u))
    N = -(D.tril(-1)) * (y @ T(u))
    dq = scale * ga * (do @ T(S0)) + Z @ k
    dk = -ga * (y @ T(S0)) + ta * (u @ T(dE)) + T(Z) @ q + (N + T(N)) @ k
    dbeta = (e * du).sum(-1)
    last = torch.cat([S0[:, :, 1:], S_end[:, :, None]], 2)
    dots = (q * dq).sum(-1) - (v * y).sum(-1)
    dots[..., -1] += (last * dE).sum((-1, -2))
    dg = dots.flip(-1).cumsum(-1).flip(-1)
    shared = lambda x: x.reshape(x.shape[0], c["hk"], -1, *x.shape[2:]).sum(2)
    return {"dq": _unrows(st, shared(dq), st["q"]), "dk": _unrows(st, shared(dk), st["k"]),
            "dv": _unrows(st, y, st["v"]), "dg": _unrows(st, dg, st["g"]), "dbeta": _unrows(st, dbeta, st["beta"]),
            "dinitial_state": dS}


def _plain_step(st):
    c = st["case"]
    group = c["hv"] // c["hk"]
    q, k = (st[x].float().repeat_interleave(group, 1) for x in ("q", "k"))
    v, slots, out = st["v"].float(), st["slots"], st["state_out"]
    live = torch.ones(v.shape[0], dtype=torch.bool, device="cuda") if slots is None else slots >= 0
    at = torch.arange(v.shape[0], device="cuda") if slots is None else slots.clamp(min=0).long()
    s = st["state"][at] * st["g"].exp()[..., None, None]
    u = st["beta"][..., None] * (v - (k[..., None] * s).sum(-2))
    s = s + k[..., None] * u[..., None, :]
    o = (q[..., None] * s).sum(-2) / math.sqrt(c["dk"])
    if slots is None:
        out.copy_(s)
    else:
        out[at[live]] = s[live]
    return {"o": torch.where(live[:, None, None], o, 0.0).to(st["v"].dtype), "state": out}


def _act(x, name):
    if name == "relu":
        return torch.where(x > 0, x, torch.zeros_like(x))
    if name == "silu":
        return x / (1 + (-x).exp())
    if name == "gelu":
        return 0.5 * x * (1 + torch.erf(x * math.sqrt(0.5)))
    return x


def _dact(x, name):
    if name == "relu":
        return (x > 0).to(x.dtype)
    if name == "silu":
        s = 1 / (1 + (-x).exp())
        return s * (1 + x * (1 - s))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(x * math.sqrt(0.5))) + x * (-0.5 * x * x).exp() / math.sqrt(2 * math.pi)
    return torch.ones_like(x)


def _plain_linear(st):
    y = st["x"].float() @ st["w"].float().T
    if st["bias"] is not None:
        y = y + st["bias"].float()
    y = _act(y, st["case"]["act"])
    if st["residual"] is not None:
        y = y + st["residual"].float()
    return y.to(st["x"].dtype)


def _plain_linear_backward(st):
    dp = st["dy"].float()
    if st["pre"] is not None:
        dp = dp * _dact(st["pre"].float(), st["case"]["act"])
    dt = st["x"].dtype
    out = {"dx": (dp @ st["w"].float()).to(dt), "dw": (dp.T @ st["x"].float()).to(dt)}
    if st["case"]["bias"]:
        out["dbias"] = dp.double().sum(0).to(dt)
    return out


# ---------------------------------------------------------------------------------------------
# least work
# ---------------------------------------------------------------------------------------------
def work(case):
    b = _SIZE[case["dtype"]]
    if case["kind"] in ("linear", "linear_backward"):
        m, k, n = case["m"], case["k"], case["n"]
        extra = n if case["bias"] else 0
        if case["kind"] == "linear":
            return {"bytes": b * (m * k + n * k + m * n * (2 if case["residual"] else 1) + extra), "flops": 2 * m * k * n}
        grads = m * n * (2 if case["act"] != "none" else 1) + 2 * (m * k + n * k) + extra
        return {"bytes": b * grads, "flops": 4 * m * k * n}
    hk, hv, dk, dv = case["hk"], case["hv"], case["dk"], case["dv"]
    if case["kind"] == "step":
        live = case["batch"] - (case["padded"] if case["slots"] else 0)
        token = b * (2 * hk * dk + 2 * hv * dv) + 8 * hv
        return {"bytes": case["batch"] * token + live * 8 * hv * dk * dv, "flops": live * hv * 7 * dk * dv}
    t = case["tokens"]
    states = case["seqs"] * hv * dk * dv * 4
    # per token and head the recurrence itself: decay, S^T k, the rank-one update and S^T q
    if case["kind"] == "forward":
        rows = t + case["pad"]
        return {"bytes": t * (b * (2 * hk * dk + hv * dv) + 8 * hv) + rows * b * hv * dv + 2 * states,
                "flops": t * hv * 7 * dk * dv}
    rows = t + case["pad"]
    token = b * (2 * hk * dk + 2 * hv * dv) + 8 * hv
    grads = b * (2 * hk * dk + hv * dv) + 8 * hv
    return {"bytes": t * token + rows * grads + 3 * states, "flops": t * hv * 20 * dk * dv}


# ---------------------------------------------------------------------------------------------
# 64 bits, from the definitions
# ---------------------------------------------------------------------------------------------
def _tokens(st, x, heads):
    """x as (time, seqs, heads, ...) in 64 bits and the (time, seqs) mask of real tokens."""
    lens, rep = st["lens"], heads // x.shape[2]
    top = max(lens)
    y = torch.zeros((top, len(lens), *x.shape[2:]), dtype=torch.float64, device="cuda")
    live = torch.zeros((top, len(lens)), dtype=torch.bool, device="cuda")
    at = 0
    for i, n in enumerate(lens):
        y[:n, i] = (x[i, :n] if st["seq_offsets"] is None else x[0, at:at + n]).double()
        live[:n, i] = True
        at += n
    return y.repeat_interleave(rep, 2), live


def _back(st, y, like):
    out = torch.zeros((*like.shape[:2], *y.shape[2:]), dtype=torch.float64, device="cuda")
    at = 0
    for i, n in enumerate(st["lens"]):
        if st["seq_offsets"] is None:
            out[i, :n] = y[:n, i]
        else:
            out[0, at:at + n] = y[:n, i]
        at += n
    return out


def _advance(S, g, k, v, beta):
    """One token: (decayed state, prediction error, new state)."""
    Sd = g.exp()[..., None, None] * S
    err = v - torch.einsum("nhkv,nhk->nhv", Sd, k)
    return Sd, err, Sd + torch.einsum("nhk,nhv->nhkv", k, beta[..., None] * err)


def exact(case, seed):
    st = prepare(case, seed)
    wide = lambda name: None if st[name] is None else st[name].double()
    act = {"none": lambda x: x, **{a: getattr(torch.nn.functional, a) for a in ("relu", "silu", "gelu")}}.get(case.get("act"))
    if case["kind"] == "linear":
        y = act(torch.nn.functional.linear(wide("x"), wide("w"), wide("bias")))
        return y if st["residual"] is None else y + wide("residual")
    if case["kind"] == "linear_backward":
        dp = wide("dy")
        if st["pre"] is not None:
            with torch.enable_grad():
                p = wide("pre").requires_grad_()
                dp = torch.autograd.grad(act(p), p, dp)[0]
        out = {"dx": dp @ st["w"].double(), "dw": dp.T @ st["x"].double()}
        if case["bias"]:
            out["dbias"] = dp.sum(0)
        return out
    hv, scale = case["hv"], case["dk"] ** -0.5
    if case["kind"] == "step":
        rep = hv // case["hk"]
        q, k = (st[x].double().repeat_interleave(rep, 1) for x in ("q", "k"))
        out = st["state_out"].double()
        o = torch.zeros(st["v"].shape, dtype=torch.float64, device="cuda")
        where = list(range(case["batch"])) if st["slots"] is None else st["slots"].tolist()
        rows = [i for i, s in enumerate(where) if s >= 0]
        at = torch.tensor([where[i] for i in rows], device="cuda")
        rows = torch.tensor(rows, device="cuda")
        _, _, S = _advance(st["state"][at].double(), st["g"][rows].double(), k[rows], st["v"][rows].double(),
                           st["beta"][rows].double())
        o[rows] = scale * torch.einsum("nhkv,nhk->nhv", S, q[rows])
        out[at] = S
        return {"o": o, "state": out}
    q, live = _tokens(st, st["q"], hv)
    k, v, g, beta = (_tokens(st, st[x], hv)[0] for x in ("k", "v", "g", "beta"))
    S = st["initial_state"].double()
    if case["kind"] == "forward":
        o = torch.zeros_like(v)
        for t in range(v.shape[0]):
            S = _advance(S, g[t], k[t], v[t], beta[t])[2]   # padding has k = 0, beta = 0 and g = 0
            o[t] = scale * torch.einsum("nhkv,nhk->nhv", S, q[t])
        return {"o": _back(st, o, st["v"]), "final_state": S}
    do = _tokens(st, st["do"], hv)[0]
    top, step = v.shape[0], 64
    marks = []
    for t in range(top):
        if t % step == 0:
            marks.append(S)
        S = _advance(S, g[t], k[t], v[t], beta[t])[2]
    dS = st["dfinal_state"].double()
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    dg, db = torch.zeros_like(g), torch.zeros_like(beta)
    for m in range(len(marks) - 1, -1, -1):
        t0, t1 = m * step, min(top, (m + 1) * step)
        S, kept = marks[m], []
        for t in range(t0, t1):
            kept.append(_advance(S, g[t], k[t], v[t], beta[t]))
            S = kept[-1][2]
        for t in range(t1 - 1, t0 - 1, -1):
            Sd, err, S = kept.pop()
            dq[t] = scale * torch.einsum("nhkv,nhv->nhk", S, do[t])
            dS = dS + scale * torch.einsum("nhk,nhv->nhkv", q[t], do[t])
            du = torch.einsum("nhkv,nhk->nhv", dS, k[t])
            derr = beta[t][..., None] * du
            dk[t] = torch.einsum("nhkv,nhv->nhk", dS, beta[t][..., None] * err) - torch.einsum("nhkv,nhv->nhk", Sd, derr)
            dv[t], db[t] = derr, (err * du).sum(-1)
            dS = dS - torch.einsum("nhk,nhv->nhkv", k[t], derr)
            dg[t] = (Sd * dS).sum((-1, -2))
            dS = g[t].exp()[..., None, None] * dS
    shared = lambda x: x.reshape(*x.shape[:2], case["hk"], -1, x.shape[-1]).sum(3)
    return {"dq": _back(st, shared(dq), st["q"]), "dk": _back(st, shared(dk), st["k"]), "dv": _back(st, dv, st["v"]),
            "dg": _back(st, dg, st["g"]), "dbeta": _back(st, db, st["beta"]), "dinitial_state": dS}
