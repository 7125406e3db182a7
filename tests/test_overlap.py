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


def step_case(**change):
    a = dict(q=torch.zeros(2, 1, 4), k=torch.zeros(2, 1, 4), v=torch.zeros(2, 2, 6), g=torch.zeros(2, 2),
             beta=torch.zeros(2, 2), state=torch.zeros(3, 2, 4, 6))
    a.update(change)
    return a


def test_step_state_out_and_out():
    def refused(match, **change):
        with pytest.raises(ValueError, match=match):
            api().gated_delta_step(**step_case(**change))

    buf = torch.zeros(3000)
    pool = buf[:144].view(3, 2, 4, 6)
    refused(TAKEN, state=pool, state_out=pool)
    refused(TAKEN, state=pool, state_out=buf[:144].view(3, 2, 4, 6))
    refused(TAKEN, state=pool, state_out=buf[144:288].view(3, 2, 4, 6))
    refused("state itself", state=pool, state_out=buf[48:192].view(3, 2, 4, 6))       # one slot further
    refused("state itself", state=pool, state_out=buf[1:145].view(3, 2, 4, 6))
    both = buf[:288].view(3, 2, 2, 4, 6)                                              # two pools, slot by slot
    refused(TAKEN, state=both[:, 0], state_out=both[:, 1])
    refused("state itself", state=both[:, 0], state_out=buf[47:47 + 288].view(3, 2, 2, 4, 6)[:, 0])
    for name, shape in dict(q=(2, 1, 4), k=(2, 1, 4), v=(2, 2, 6), g=(2, 2), beta=(2, 2)).items():
        n = torch.Size(shape).numel()
        refused("state_out must not overlap", state=pool, **{name: buf[140:140 + n].view(shape)})
        refused("state_out must not overlap", state_out=pool, **{name: buf[140:140 + n].view(shape)})
        refused(TAKEN, state=pool, **{name: buf[144:144 + n].view(shape)})
        out = buf[500:524].view(2, 2, 6)
        refused("out must not overlap", out=out, **{name: buf[523:523 + n].view(shape)})
        refused(TAKEN, out=out, **{name: buf[524:524 + n].view(shape)})
    refused("out must not overlap", out=buf[140:164].view(2, 2, 6), state=pool)
    refused("out must not overlap", out=buf[140:164].view(2, 2, 6), state_out=pool)
    refused(TAKEN, out=out, v=out)
    ints = torch.zeros(24, dtype=torch.int32)
    refused("out must not overlap", out=ints.view(torch.float32).view(2, 2, 6), slots=ints[22:])


@gpu
def test_step_out_over_v():
    gen = torch.Generator(device="cuda").manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    for dtype in (torch.bfloat16, torch.float32):
        q, k, v = r(5, 2, 64).to(dtype), r(5, 2, 64).to(dtype), r(5, 4, 100).to(dtype)
        g, beta, state = -r(5, 4).abs(), r(5, 4).sigmoid(), r(5, 4, 64, 100)
        kept = torch.empty_like(state)
        want = api().gated_delta_step(q, k, v, g, beta, state, state_out=kept)
        assert api().gated_delta_step(q, k, v, g, beta, state, out=v).data_ptr() == v.data_ptr()
        assert torch.equal(v, want) and torch.equal(state, kept)


@gpu
def test_outputs_beside_inputs():
    """Results in slices of the buffers that the inputs lie in."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    wide = torch.randn(300, 200, generator=gen, device="cuda").bfloat16()
    w = torch.randn(64, 96, generator=gen, device="cuda").bfloat16()
    want, x = api().linear(wide[:, :96].contiguous(), w), wide[:, :96].clone()
    assert torch.equal(api().linear(wide[:, :96], w, out=wide[:, 96:160]), want) and torch.equal(wide[:, :96], x)
    pools = torch.randn(4, 2, 2, 32, 32, generator=gen, device="cuda")
    tok = [torch.randn(4, 2, 32, generator=gen, device="cuda") for _ in range(3)]
    g, beta = torch.full((4, 2), -0.5, device="cuda"), torch.full((4, 2), 0.5, device="cuda")
    old = pools[:, 0].clone()
    dense = old.clone()
    want = api().gated_delta_step(*tok, g, beta, dense)
    assert torch.equal(api().gated_delta_step(*tok, g, beta, pools[:, 0], state_out=pools[:, 1]), want)
    assert torch.equal(pools[:, 1], dense) and torch.equal(pools[:, 0], old)
