"""qr_b200 -- B200-native batched Householder QR (sm_100a CUDA behind a C ABI).

Public API mirrors the reference's submission interface:

* ``custom_kernel(data) -> (H, tau)``   (torch.geqrf compact form)
* ``form_q(H, tau) -> Q``               (torch.linalg.householder_product)
* ``qr(A) -> (H, tau, Q)``              (both, one library call)
* ``geqrf`` / ``orgqr``                 (aliases with explicit names)

Sequence operators that share QR's compact-WY products:

* ``gated_delta_rule(q, k, v, g, beta) -> (o, final_state)``, ``gated_delta_rule_backward`` and
  ``gated_delta_step`` (one token per row)
* ``linear(x, w, bias, activation=..., residual=...) -> y`` and ``linear_backward``

The ops (and with them ``libqrb200.so``) load on first attribute access, so that
``qr_b200.inputs`` -- the seeded input generators -- can be imported by code that
must not map the library (the CPU reference arm of ``bench.py``).
"""
from __future__ import annotations

import importlib

_OPS = ("custom_kernel", "form_q", "geqrf", "orgqr", "qr", "qr_host")
_DELTA = ("gated_delta_rule", "gated_delta_rule_backward", "gated_delta_step")
_LINEAR = ("linear", "linear_backward")
_LIB = ("QRBError", "lib")

__all__ = [*_OPS, *_DELTA, *_LINEAR, *_LIB]


_WHERE = {**dict.fromkeys(_OPS, ".ops"), **dict.fromkeys(_DELTA, ".delta"), **dict.fromkeys(_LINEAR, "._linear"),
          **dict.fromkeys(_LIB, "._lib")}


def __getattr__(name: str):
    if name not in _WHERE:
        raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
    value = getattr(importlib.import_module(_WHERE[name], __name__), name)
    globals()[name] = value   # the next access finds it without coming here (3 us a call)
    return value
