"""GPU: the learner operators' saved tensors under torch.autograd.graph.saved_tensors_hooks, which may hand other memory back than was saved."""
import pytest
import torch

from test_gpu_learner_ops import DTYPES, gen, ops, rand

pytestmark = pytest.mark.gpu


def other_strides(x):
    """the same values, two elements apart or with the first two dimensions swapped in memory"""
    if x.dim() >= 2 and x.shape[0] > 1 and x.shape[1] > 1:
        return x.transpose(0, 1).contiguous().transpose(0, 1)
    return torch.stack([x, x], -1)[..., 0] if x.dim() else x.clone()


def recurrence(T, N, D, dtype, layout):
    g = gen(T)
    dt = DTYPES[dtype]

    def put(x):
        return x.transpose(0, 1).contiguous().cuda().transpose(0, 1) if layout else x.cuda()

    gate, update = (put(torch.rand((T, N, D), generator=g).to(dt)).requires_grad_() for _ in range(2))
    state, first = rand((N, D), g).cuda().requires_grad_(), (torch.rand((T, N), generator=g) < 0.1).cuda()
    d_h, d_last = rand((T, N, D), g, dt).cuda(), rand((N, D), g).cuda()
    return [gate, update, state], lambda: ops().gated_recurrence(gate, update, first, state), [d_h, d_last], first


def logprobs(B, A, dtype, layout):
    g = gen(A)
    wide = rand((2, B + layout, A), g, DTYPES[dtype], 2.0).cuda()
    logits = wide[:, :B].requires_grad_()
    actions = torch.randint(0, A, (2, B), generator=g).cuda()
    return [logits], lambda: ops().action_logprobs(logits, actions), [rand((2, B), g).cuda() for _ in range(2)], None


def loss(B, A, dtype, layout, ref, scale):
    g = gen(A)
    logits = rand((2, B + layout, A), g, DTYPES[dtype], 2.0).cuda()[:, :B].requires_grad_()
    actions = torch.randint(0, A, (2, B), generator=g).cuda()
    old, adv = rand((2, B), g, scale=0.1, shift=-2.0).cuda(), rand((2, B), g).cuda()
    valid = (torch.rand((2, B), generator=g) < 0.8).cuda()
    kw = {} if ref is None else {"kl_coef": 0.3, "ref_logprobs": rand((2, B), g, scale=0.1, shift=-2.0).cuda()} if ref == "logprobs" else {
        "kl_coef": 0.3, "ref_logits": rand((2, B, A), g, DTYPES[dtype], 2.0).cuda()}
    return [logits], lambda: (ops().policy_loss(logits, actions, old, adv, valid=valid, entropy_coef=0.02, **kw).loss,), [torch.tensor(scale).cuda()], None


CASES = [(recurrence, (3, 5, 6, "f32", 0)), (recurrence, (4, 7, 33, "bf16", 1)), (recurrence, (200, 5, 6, "f32", 0)), (recurrence, (1000, 3, 70, "f16", 1)), (recurrence, (40, 600, 64, "bf16", 0)),
         (logprobs, (9, 15, "f32", 0)), (logprobs, (9, 15, "bf16", 2)), (logprobs, (5, 300, "f32", 0)), (logprobs, (5, 9000, "f32", 1)), (logprobs, (5, 9000, "bf16", 0)),
         (loss, (9, 15, "f32", 0, None, 2.0)), (loss, (9, 15, "f32", 1, "logits", 2.0)), (loss, (9, 200, "bf16", 0, "logprobs", 2.0)), (loss, (9, 9000, "f32", 1, "logits", 0.5)),
         (loss, (300, 15, "f32", 0, "logits", 1.0))]


@pytest.mark.parametrize("make,args", CASES)
def test_saved_tensors_may_come_back_with_other_strides(make, args):
    leaves, call, d, _ = make(*args)
    out = call()
    want = torch.autograd.grad(out, leaves, d, retain_graph=True)
    again = torch.autograd.grad(out, leaves, d)
    with torch.autograd.graph.saved_tensors_hooks(lambda x: x, other_strides):
        out = call()
    got = torch.autograd.grad(out, leaves, d, retain_graph=True)
    more = torch.autograd.grad(out, leaves, d)  # without the gradient that the forward call has written
    for w, a, x, y in zip(want, again, got, more):
        assert torch.equal(w, x) and torch.equal(a, y)


@pytest.mark.parametrize("make,args", [CASES[0], CASES[2], CASES[5], CASES[9], CASES[11], CASES[12]])
@pytest.mark.parametrize("change", ["device", "type", "shape"])
def test_saved_tensors_that_come_back_as_something_else_are_refused(make, args, change):
    """each of them in turn: on the host, in another type, with a row less; nothing is enqueued for them"""
    leaves, call, d, _ = make(*args)
    count = []
    with torch.autograd.graph.saved_tensors_hooks(lambda x: count.append(1) or x, lambda x: x):
        call()
    assert len(count) >= 4
    change = {"device": lambda x: x.cpu(), "type": lambda x: x.double(), "shape": lambda x: x[:-1].clone()}[change]
    for k in range(len(count)):
        packed = []

        def pack(x):
            packed.append(x)
            return len(packed) - 1

        with torch.autograd.graph.saved_tensors_hooks(pack, lambda i: change(packed[i]) if i == k else packed[i]):
            out = call()
        with pytest.raises(RuntimeError, match="saved tensor"):
            torch.autograd.grad(out, leaves, d)
