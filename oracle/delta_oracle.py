"""The gated delta rule token by token in 64 bits, forward and backward: the oracle of the kernels'
tests.  One sequence and head at a time would be the definition; here they are vectorised and the
tokens are not.

    S~_t = exp(g_t) S_{t-1},  u_t = beta_t (v_t - S~_t^T k_t),  S_t = S~_t + k_t u_t^T,
    o_t = scale S_t^T q_t
"""
from __future__ import annotations

import torch


def _heads(x, hv):
    return x.double().repeat_interleave(hv // x.shape[-2], -2)


def forward(q, k, v, g, beta, scale, S):
    """(time, heads, ...) inputs of one sequence, S (heads, dk, dv): (o, final S, per-token records)."""
    hv = v.shape[1]
    q, k, v, g, beta, S = _heads(q, hv), _heads(k, hv), v.double(), g.double(), beta.double(), S.double()
    o, kept = torch.zeros_like(v), []
    for t in range(v.shape[0]):
        Sd = g[t].exp()[:, None, None] * S
        err = v[t] - torch.einsum("hkv,hk->hv", Sd, k[t])
        S = Sd + torch.einsum("hk,hv->hkv", k[t], beta[t][:, None] * err)
        o[t] = scale * torch.einsum("hkv,hk->hv", S, q[t])
        kept.append((Sd, err, S))
    return o, S, kept


def backward(do, dS, q, k, v, g, beta, scale, S):
    """Gradients (dq, dk, dv, dg, dbeta, dS0) of <o, do> + <final S, dS>, and dg's scale: the norms of
    the sums dg is the difference of."""
    hv, hk = v.shape[1], q.shape[1]
    o, S_end, kept = forward(q, k, v, g, beta, scale, S)
    q, k, v, g, beta, do, dS = _heads(q, hv), _heads(k, hv), v.double(), g.double(), beta.double(), do.double(), dS.double()
    dq, dk, dv, dg, db = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), torch.zeros_like(g), torch.zeros_like(g)
    for t in range(v.shape[0] - 1, -1, -1):
        Sd, err, S = kept[t]
        dq[t] = scale * torch.einsum("hkv,hv->hk", S, do[t])
        dS = dS + scale * torch.einsum("hk,hv->hkv", q[t], do[t])
        du = torch.einsum("hkv,hk->hv", dS, k[t])
        dv[t] = beta[t][:, None] * du
        db[t] = (err * du).sum(-1)
        dk[t] = torch.einsum("hkv,hv->hk", dS, beta[t][:, None] * err) - torch.einsum("hkv,hv->hk", Sd, dv[t])
        dS = dS - torch.einsum("hk,hv->hkv", k[t], dv[t])
        dg[t] = (Sd * dS).sum((-1, -2))
        dS = g[t].exp()[:, None, None] * dS
    fold = lambda x: x.reshape(x.shape[0], hk, hv // hk, x.shape[-1]).sum(2)
    return fold(dq), fold(dk), dv, dg, db, dS
