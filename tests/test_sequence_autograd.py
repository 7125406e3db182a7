"""What the sequence operators tell autograd: tensors they write, and derivatives they do not have."""
import pytest
import torch

gpu = pytest.mark.gpu
MODIFIED = "modified by an inplace operation"


@pytest.fixture(scope="module", autouse=True)
def _built():
    import build
    build.build()
    build.build_entry()


def api():
    import qr_b200
    return qr_b200


def rule_args(device="cuda", time=20):
    r = lambda *s: torch.randn(*s, device=device)
    k = torch.nn.functional.normalize(r(2, time, 1, 32), dim=-1)
    return r(2, time, 1, 32), k, r(2, time, 2, 48), -r(2, time, 2).abs(), r(2, time, 2).sigmoid(), r(2, 2, 32, 48)


def token(x):
    return [t[:, 0].contiguous() for t in x]


WRITES = {
    "step": lambda x, pool: api().gated_delta_step(*token(x), pool),
    "step into another pool": lambda x, pool: api().gated_delta_step(*token(x), torch.zeros_like(pool), state_out=pool),
    "final state": lambda x, pool: api().gated_delta_rule(*x, out=(torch.empty_like(x[2]), pool)),
    "final state over the initial one": lambda x, pool: api().gated_delta_rule(
        *x, initial_state=pool, out=(torch.empty_like(x[2]), pool)),
    "step on a view": lambda x, pool: api().gated_delta_step(*[t[:1] for t in token(x)], pool[1:]),
}


@gpu
@pytest.mark.parametrize("write", WRITES)
def test_a_state_written_before_the_backward_pass_is_noticed(write):
    *x, pool = rule_args()
    leaf = x[2].clone().requires_grad_()
    o, _ = api().gated_delta_rule(x[0], x[1], leaf, *x[3:], initial_state=pool)
    version = pool._version
    with torch.no_grad():
        WRITES[write](x, pool)
    assert pool._version > version
    with pytest.raises(RuntimeError, match=MODIFIED):
        o.sum().backward()


@gpu
def test_outputs_written_before_the_backward_pass_are_noticed():
    *x, pool = rule_args()
    leaf = x[0].clone().requires_grad_()
    o, _ = api().gated_delta_rule(leaf, *x[1:])
    with torch.no_grad():
        api().gated_delta_rule(*(t.clone() for t in x), out=(x[2], torch.empty_like(pool)))
    with pytest.raises(RuntimeError, match=MODIFIED):
        o.sum().backward()
    o, _ = api().gated_delta_rule(leaf, *x[1:])
    with torch.no_grad():
        api().gated_delta_step(*(t.clone() for t in token(x)), pool, out=x[2].view(40, 2, 48)[:2])
    with pytest.raises(RuntimeError, match=MODIFIED):
        o.sum().backward()
    a, w, z = torch.randn(6, 16, device="cuda"), torch.randn(8, 16, device="cuda").requires_grad_(), torch.randn(6, 8, device="cuda")
    y = api().linear(a, w)
    with torch.no_grad():
        api().linear(z, torch.randn(16, 8, device="cuda"), out=a)
    with pytest.raises(RuntimeError, match=MODIFIED):
        y.sum().backward()


@gpu
def test_inputs_keep_their_versions():
    *x, pool = rule_args()
    other = torch.empty_like(pool)
    a, w = torch.randn(6, 16, device="cuda"), torch.randn(8, 16, device="cuda")
    read = [*x, pool, a, w]
    before = [t._version for t in read]
    api().gated_delta_rule(*x, initial_state=pool, out=(torch.empty_like(x[2]), other))
    api().gated_delta_rule_backward(x[2], *x, initial_state=pool)
    api().gated_delta_step(*token(x), pool, state_out=other)
    api().linear(a, w)
    api().linear_backward(torch.randn(6, 8, device="cuda"), a, w)
    assert [t._version for t in read] == before
    leaf = x[2].clone().requires_grad_()
    api().gated_delta_rule(x[0], x[1], leaf, *x[3:], initial_state=pool)[0].sum().backward()
    assert torch.isfinite(leaf.grad).all()


@gpu
def test_states_of_inference_mode_are_written():
    with torch.inference_mode():
        *x, pool = rule_args()
        want = pool.clone()
        api().gated_delta_step(*token(x), want)
    with torch.no_grad():
        api().gated_delta_step(*token(x), pool)
    assert torch.equal(pool, want)


# ---- forward mode: no derivative, so no result either ----
def calls(device):
    *x, pool = rule_args(device)
    a, w, b, r = (torch.randn(*s, device=device) for s in ((6, 16), (8, 16), (8,), (6, 8)))
    rule = dict(zip(("q", "k", "v", "g", "beta"), x))
    return {
        "gated_delta_rule": dict(rule, initial_state=pool),
        "gated_delta_rule_backward": dict(rule, do=torch.randn_like(x[2]), initial_state=pool,
                                          dfinal_state=torch.randn_like(pool)),
        "gated_delta_step": dict(zip(rule, token(x)), state=pool, state_out=torch.zeros_like(pool)),
        "linear": dict(x=a, w=w, bias=b, residual=r),
        "linear_backward": dict(dy=r, x=a, w=w, activation="silu", pre=r.clone()),
    }


def refuse_each_tangent(device, grad):
    import torch.autograd.forward_ad as ad
    for name, args in calls(device).items():
        for which in [n for n, t in args.items() if isinstance(t, torch.Tensor)]:
            with ad.dual_level(), torch.set_grad_enabled(grad):
                primal = args[which].clone().requires_grad_(grad)
                dual = ad.make_dual(primal, torch.ones_like(primal))
                # with gradients too, torch's own refusal of the recorded function
                match = "forward" if not grad else None
                with pytest.raises(RuntimeError if grad else NotImplementedError, match=match):
                    getattr(api(), name)(**dict(args, **{which: dual}))


def test_tangents_are_refused():
    refuse_each_tangent("cpu", False)


@gpu
def test_tangents_are_refused_on_the_device():
    refuse_each_tangent("cuda", False)
    refuse_each_tangent("cuda", True)
    for name, args in calls("cuda").items():
        which = "x" if "linear" in name else "q"
        with pytest.raises(RuntimeError):
            torch.func.jvp(lambda t: getattr(api(), name)(**dict(args, **{which: t})), (args[which],),
                           (torch.ones_like(args[which]),))


def test_outputs_that_require_gradients_are_refused():
    *x, pool = rule_args("cpu")
    o, s = torch.empty_like(x[2]), torch.empty_like(pool)
    leaf = lambda t: t.clone().requires_grad_()
    for out in ((leaf(o), s), (o, leaf(s)), (leaf(o) * 2, s)):
        with pytest.raises(ValueError, match="requires gradients"):
            api().gated_delta_rule(*x, out=out)
    for change in (dict(state_out=leaf(pool)), dict(out=leaf(o[:, 0])), dict(state_out=leaf(pool) * 2)):
        with pytest.raises(RuntimeError, match="no gradient"):
            api().gated_delta_step(*token(x), pool, **change)
    a, w = torch.zeros(6, 16), torch.zeros(8, 16)
    with pytest.raises(ValueError, match="requires gradients"):
        api().linear(a, w, out=leaf(torch.zeros(6, 8)))
    with torch.no_grad(), pytest.raises(ValueError, match="no CPU path"):
        api().linear(a, w, out=leaf(torch.zeros(6, 8)))
