"""Packed sequences of the gated delta rule over types and head sizes, against the oracle: tests/test_delta.py has the
lengths and the tolerances."""
import pytest
import torch

import test_delta as T

gpu = pytest.mark.gpu
BF, HF, F32 = T.BF, T.HF, T.F32


@pytest.fixture(scope="module", autouse=True)
def _built():
    import build
    build.build()
    build.build_entry()


HEADS = [(2, 4, 64, 64), (1, 3, 128, 128), (2, 2, 96, 80), (1, 2, 33, 200), (3, 3, 64, 256)]   # hk, hv, dk, dv


def check(lens, pad, heads, dtype):
    hk, hv, dk, dv = heads
    offs = [0]
    for n in lens:
        offs.append(offs[-1] + n)
    total, end = offs[-1] + pad, offs[-1]
    x = T.make(1, total, hk, hv, dk, dv, dtype)
    do = T.make(1, total, hk, hv, dk, dv, dtype, seed=5)[2]
    for t in (*x, do):
        t[:, end:] = float("nan")                               # nothing behind the last sequence is read
    init, dS = T.states(len(lens), hv, dk, dv), T.states(len(lens), hv, dk, dv, 2)
    so = torch.tensor(offs, dtype=torch.int32, device="cuda")
    o, s = T.api().gated_delta_rule(*x, initial_state=init, seq_offsets=so)
    T.check_forward(x, init, offs, o, s)
    assert (o[:, end:] == 0).all()
    grads = T.api().gated_delta_rule_backward(do, *x, initial_state=init, seq_offsets=so, dfinal_state=dS)
    T.check_backward(grads, do, dS, x, init, offs)
    assert all((t[:, end:] == 0).all() for t in grads[:5])
    alone = T.api().gated_delta_rule_backward(do, *x, seq_offsets=so)
    assert alone[5] is None
    T.check_backward(alone, do, None, x, None, offs)


@gpu
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("lens", [[64, 1, 0, 130, 63], [0, 0, 5, 128], [200]])
def test_packed(lens, heads, dtype):
    check(lens, 3, heads, dtype)


@gpu
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("lens", [[0, 1500, 3, 700, 0, 64, 1]])      # cut into segments side by side
def test_long_packed(lens, heads, dtype):
    check(lens, 70, heads, dtype)


@gpu
@pytest.mark.parametrize("lens", T.LENS)
def test_packed_fp16(lens):
    T.test_packed(lens, 200, HF)
