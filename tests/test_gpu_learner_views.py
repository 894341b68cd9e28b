"""GPU: ways of calling the learner operators that torch records beside the values -- tangents, traces, lazy negation."""
import pytest
import torch
import torch.autograd.forward_ad as fw

from test_gpu_learner_ops import ops

pytestmark = pytest.mark.gpu


def inputs():
    g = torch.Generator().manual_seed(0)
    x = {k: torch.randn(s, generator=g).cuda() for k, s in {"gate": (6, 3, 4), "update": (6, 3, 4), "state": (3, 4), "rew": (6, 3), "values": (7, 3), "logits": (6, 3, 5), "ref_logits": (6, 3, 5),
                                                            "old": (6, 3), "adv": (6, 3), "ref_logprobs": (6, 3)}.items()}
    x["first"] = torch.zeros((7, 3), dtype=torch.uint8, device="cuda")
    x["begins"] = x["first"][:-1]
    x["actions"] = torch.zeros((6, 3), dtype=torch.int32, device="cuda")
    return x


CALLS = {
    "recurrence": (lambda x: ops().gated_recurrence(x["gate"], x["update"], x["begins"], x["state"])[0], ["gate", "update", "state"]),
    "advantages": (lambda x: ops().advantages(x["rew"], x["values"], x["first"], gamma=0.9, lam=0.9)[0], ["rew", "values"]),
    "logprobs": (lambda x: ops().action_logprobs(x["logits"], x["actions"])[0], ["logits"]),
    "loss": (lambda x: ops().policy_loss(x["logits"], x["actions"], x["old"], x["adv"], ref_logits=x["ref_logits"], kl_coef=0.1).loss, ["logits", "old", "adv", "ref_logits"]),
    "loss, estimator": (lambda x: ops().policy_loss(x["logits"], x["actions"], x["old"], x["adv"], ref_logprobs=x["ref_logprobs"], kl_coef=0.1).loss, ["ref_logprobs"]),
}
EACH = [(call, name) for call, (_, names) in CALLS.items() for name in names]


@pytest.mark.parametrize("call,name", EACH)
@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode_is_refused_and_not_dropped(call, name, requires_grad):
    x = inputs()
    if requires_grad and name in ("gate", "update", "state", "logits"):
        x[name].requires_grad_()
    with fw.dual_level():
        x[name] = fw.make_dual(x[name], torch.ones_like(x[name]))
        with pytest.raises(ValueError, match="forward-mode"):
            CALLS[call][0](x)
        with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
            CALLS[call][0](x)
    CALLS[call][0](inputs())


def test_a_state_out_with_a_tangent_is_refused():
    x = inputs()
    with torch.no_grad(), fw.dual_level():
        out = fw.make_dual(torch.zeros((3, 4), device="cuda"), torch.ones((3, 4), device="cuda"))
        with pytest.raises(ValueError, match="forward-mode"):
            ops().gated_recurrence(x["gate"], x["update"], state_out=out)


@pytest.mark.parametrize("call", CALLS)
def test_tracing_is_refused_and_does_not_record_empty_outputs(call):
    x = inputs()
    name = CALLS[call][1][0]
    with pytest.raises(ValueError, match="traced"):
        torch.jit.trace(lambda v: CALLS[call][0]({**x, name: v}), x[name], check_trace=False)
    CALLS[call][0](x)


@pytest.mark.parametrize("call", CALLS)
def test_symbolic_tracing_is_refused(call):
    """make_fx records what torch dispatches: the outputs' allocations, and nothing that writes them"""
    from torch.fx.experimental.proxy_tensor import make_fx

    x = inputs()
    name = CALLS[call][1][0]
    for mode in ("real", "fake"):
        with pytest.raises(ValueError, match="traced"):
            make_fx(lambda v: CALLS[call][0]({**x, name: v}), tracing_mode=mode)(x[name])
    CALLS[call][0](x)


def lazily_negated(x):
    """the same values behind a view that torch negates when it reads it"""
    y = torch.complex(torch.zeros_like(x), -x).conj().imag
    assert y.is_neg() and torch.equal(y.resolve_neg(), x)
    return y


@pytest.mark.parametrize("call,name", EACH)
def test_lazily_negated_inputs_are_refused(call, name):
    x = inputs()
    x[name] = lazily_negated(x[name])
    with pytest.raises(ValueError, match="resolve_neg"):
        CALLS[call][0](x)
    x[name] = x[name].resolve_neg()
    assert torch.equal(CALLS[call][0](x), CALLS[call][0](inputs()))


def test_a_lazily_negated_state_out_is_refused():
    x = inputs()
    with torch.no_grad(), pytest.raises(ValueError, match="resolve_neg"):
        ops().gated_recurrence(x["gate"], x["update"], state_out=lazily_negated(x["state"]))


def test_lazily_negated_gradients_are_taken_as_their_values():
    x = inputs()
    g = torch.Generator().manual_seed(1)
    for k in ("gate", "update", "state", "logits"):
        x[k].requires_grad_()
    runs = [(lambda: ops().gated_recurrence(x["gate"], x["update"], None, x["state"]), ["gate", "update", "state"]), (lambda: ops().action_logprobs(x["logits"], x["actions"]), ["logits"]),
            (lambda: ops().policy_loss(x["logits"], x["actions"], x["old"], x["adv"])[:1], ["logits"])]
    for run, names in runs:
        leaves = [x[k] for k in names]
        out = run()
        d = [torch.randn(v.shape, generator=g).cuda() for v in out]
        want = torch.autograd.grad(out, leaves, d)
        got = torch.autograd.grad(run(), leaves, [lazily_negated(v) for v in d])
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_a_state_out_that_may_not_be_written_is_left_as_it_was():
    x = inputs()
    with torch.inference_mode():
        out = torch.full((3, 4), 7.0, device="cuda")
    with torch.no_grad(), pytest.raises(RuntimeError, match="InferenceMode"):
        ops().gated_recurrence(x["gate"], x["update"], state_out=out)
    assert (out == 7).all()
    with torch.inference_mode():
        assert ops().gated_recurrence(x["gate"], x["update"], state_out=out)[1] is not None and (out != 7).all()
