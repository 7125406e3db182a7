"""What a call may write into: outputs over tensors that the kernels still read are refused (found on the host,
so on CPU tensors here), and those that only lie between or beside them are taken."""
import random

import pytest
import torch

gpu = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _built():
    import build
    build.build()
    build.build_entry()


def api():
    import qr_b200
    return qr_b200


TAKEN = "no CPU path"      # what a call of CPU tensors that passes every other check ends with


def linear_case(**change):
    a = dict(x=torch.zeros(8, 16), w=torch.zeros(16, 16), bias=torch.zeros(16), residual=torch.zeros(8, 16))
    a.update(change)
    return a


def test_linear_out_over_an_input():
    a = linear_case()
    buf = torch.zeros(8 * 16 * 4)
    for out in (a["x"], a["x"].view(-1).view(8, 16), a["w"][:8], a["w"][8:]):
        with pytest.raises(ValueError, match="must not overlap x, w or bias"):
            api().linear(**a, out=out)
    x, shifted = buf[:128].view(8, 16), buf[127:255].view(8, 16)
    with pytest.raises(ValueError, match="must not overlap x, w or bias"):
        api().linear(**linear_case(x=x), out=shifted)
    with pytest.raises(ValueError, match=TAKEN):
        api().linear(**linear_case(x=x), out=buf[128:256].view(8, 16))
    wide = torch.zeros(8, 40)
    with pytest.raises(ValueError, match=TAKEN):                 # column slices of one buffer
        api().linear(**linear_case(x=wide[:, 2:18]), out=wide[:, 18:34])
    with pytest.raises(ValueError, match=TAKEN):
        api().linear(**linear_case(x=wide[:, 18:34], bias=wide[3, :2].repeat(8)), out=wide[:, 2:18])
    with pytest.raises(ValueError, match="must not overlap x, w or bias"):
        api().linear(**linear_case(x=wide[:, 2:18]), out=wide[:, 17:33])
    with pytest.raises(ValueError, match="must not overlap x, w or bias"):
        api().linear(**linear_case(bias=wide[7, 4:20]), out=wide[:, :16])


def test_linear_out_and_residual():
    wide = torch.zeros(9, 40)
    with pytest.raises(ValueError, match=TAKEN):
        api().linear(**linear_case(residual=wide[:8, :16]), out=wide[:8, :16])
    same = torch.zeros(8, 16)
    with pytest.raises(ValueError, match=TAKEN):
        api().linear(**linear_case(residual=same), out=same)
    with pytest.raises(ValueError, match=TAKEN):
        api().linear(**linear_case(residual=wide[:8, :16]), out=wide[:8, 16:32])
    for residual in (wide[1:, :16], wide[:8, 1:17], wide.view(-1)[:128].view(8, 16), wide[0, :16].expand(8, 16)):
        with pytest.raises(ValueError, match="residual itself"):
            api().linear(**linear_case(residual=residual), out=wide[:8, :16])


def test_random_views_of_one_buffer():
    """The host's answer against the sets of elements themselves."""
    rng = random.Random(5)
    yes = no = 0
    for _ in range(3000):
        n, rows, cols = 600, rng.randint(1, 9), 4
        buf = torch.arange(n, dtype=torch.float32)

        def rows_of(count):
            ld = rng.choice([cols, cols, cols + 1, 10, 13, 20, 31])
            at = rng.randrange(n - (count - 1) * ld - cols)
            return buf.as_strided((count, cols), (ld, 1), at)
        out, other = rows_of(rows), rows_of(rng.randint(1, 9) if rng.random() < 0.5 else rows)
        if rng.random() < 0.3:                                    # as a matrix of other strides, or with repeats
            other = other.t().contiguous().t() if rng.random() < 0.1 else other[:, :1].expand(-1, cols)
        meets = bool(set(out.flatten().tolist()) & set(other.flatten().tolist())) and other.data_ptr() >= buf.data_ptr() \
            and other.data_ptr() < buf.data_ptr() + 4 * n
        w = torch.zeros(cols, cols)
        a = dict(x=torch.zeros(rows, cols), w=w, out=out)
        if other.shape[0] == cols and rng.random() < 0.5:
            a["w"] = other
        elif other.shape[0] == rows:
            a["x"] = other
        else:
            continue
        yes, no = yes + meets, no + (not meets)
        with pytest.raises(ValueError, match="must not overlap" if meets else TAKEN):
            api().linear(**a)
    assert yes > 100 and no > 100


def rule_case(**change):
    a = dict(q=torch.zeros(1, 8, 1, 4), k=torch.zeros(1, 8, 1, 4), v=torch.zeros(1, 8, 2, 6), g=torch.zeros(1, 8, 2),
             beta=torch.zeros(1, 8, 2), initial_state=torch.zeros(2, 2, 4, 6),
             seq_offsets=torch.tensor([0, 3, 8], dtype=torch.int32))
    a.update(change)
    return a


def test_rule_out():
    buf = torch.zeros(1000)
    o, state = buf[:96].view(1, 8, 2, 6), buf[200:296].view(2, 2, 4, 6)

    def refused(match, out, **change):
        with pytest.raises(ValueError, match=match):
            api().gated_delta_rule(**rule_case(**change), out=out)

    refused(TAKEN, (o, state))
    refused(TAKEN, (o, state), initial_state=state)
    refused(TAKEN, (o, state), initial_state=buf[296:392].view(2, 2, 4, 6))
    refused(r"out\[1\] may be initial_state itself", (o, state), initial_state=buf[206:302].view(2, 2, 4, 6))
    refused(r"out\[0\] must not overlap", (o, state), initial_state=buf[95:191].view(2, 2, 4, 6))
    refused(r"out\[0\] must not overlap", (o, buf[95:191].view(2, 2, 4, 6)))
    ints = torch.zeros(100, dtype=torch.int32)
    f = ints.view(torch.float32)
    refused(r"out\[0\] must not overlap", (f[:96].view(1, 8, 2, 6), state), seq_offsets=ints[95:98])
    refused(r"out\[1\] must not overlap seq_offsets", (o, f[:96].view(2, 2, 4, 6)), seq_offsets=ints[93:96])
    refused(TAKEN, (o, f[:96].view(2, 2, 4, 6)), seq_offsets=ints[96:99])
    refused("share memory", (torch.zeros(1, 8, 1, 6).expand(1, 8, 2, 6), state))
    refused("share memory", (buf.as_strided((1, 8, 2, 6), (96, 6, 3, 1)), state))
    refused(TAKEN, (buf.as_strided((1, 8, 2, 6), (0, 6, 48, 1)), state))          # heads apart, tokens together
    refused(TAKEN, (buf.as_strided((1, 8, 2, 6), (0, 20, 9, 1)), buf[500:596].view(2, 2, 4, 6)))
