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
