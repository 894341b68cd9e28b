"""
GPU: rows of logits over the whole range of their type -- finite masks of any size, rows of one value, diverged logits -- against 64 bits.

Tolerances are those of test_gpu_learner_ops (running error bounds in 64 bits).  They hold at any size of the logits, because a logit enters only as
its difference to the row's largest one: that subtraction is rounded once, relative to the difference.
"""
import pytest
import torch

from test_gpu_learner_ops import DTYPES, U, Rows64, check, gen, ops, pick, policy_64, put_rows, rounding

pytestmark = pytest.mark.gpu

LOW = torch.finfo(torch.float32).min
FILLS = [s * v for v in (1e3, 1e6, 1e8, 1e9, 1.5e9, 3e9, 1e10, 1e12, 1e20, 1e30, 1e37, 9e37, 2e38, 3.3e38) for s in (1.0, -1.0)] + [LOW]
HALVES = [(1.5e38, 9e37), (2e38, 1e19), (-2e38, -0.9e38), (-1e10, -1e20), (-1e30, LOW), (1e20, 2e38), (1e10, 0.0), (-1e10, 0.0), (5e8, 4.9e8), (1.7e7, 1.7e7 - 2), (3e9, LOW), (0.0, LOW)]
# columns and how often the rows are repeated: a lane per row; groups inside a wave; of two waves (2700 of 16 bits, 1400 of 32); of four (where there
# are 512 rows); a block per row in one batch, several, and more than its LDS keeps
WIDTHS = [(2, 1), (15, 1), (16, 1), (31, 1), (40, 1), (200, 1), (1000, 1), (1400, 1), (2700, 1), (9000, 1), (9000, 20), (50021, 1)]


def gradient_64(w, actions, d_logp, d_entropy):
    """of sum(d_logp * logp + d_entropy * entropy), and how far 32 bits may be off"""
    onehot = torch.zeros_like(w.p).scatter_(1, actions.long()[:, None], 1.0)
    gl, ge = d_logp.double()[:, None], d_entropy.double()[:, None]
    both = torch.where(w.p > 0, w.finite_logp + w.H[:, None], torch.zeros_like(w.p))
    want = gl * (onehot - w.p) - ge * w.p * both
    tol = gl.abs() * w.p * w.rel_p + ge.abs() * w.p * (both.abs() * w.rel_p + w.T_logp + w.T_H[:, None]) + 8 * U * (gl.abs() * (onehot + w.p) + ge.abs() * w.p * both.abs())
    return want, tol


def compare(x, actions, seed, ref=None, layout="plain"):
    """the three calls on rows x [B, A] (on the GPU, at any size) against their definitions in 64 bits"""
    B, A = x.shape
    g = gen(seed)
    w = Rows64(x)
    t = put_rows(x.detach(), layout).requires_grad_()
    logp, entropy = ops().action_logprobs(t, actions)
    check(logp, pick(w.logp, actions).cpu(), pick(w.T_logp, actions).cpu(), "log-probabilities")
    check(entropy, w.H.cpu(), w.T_H.cpu(), "entropy")
    d_logp, d_entropy = (torch.randn((B,), generator=g).cuda() for _ in range(2))
    (d,) = torch.autograd.grad([logp, entropy], [t], [d_logp, d_entropy])
    want, tol = gradient_64(w, actions, d_logp, d_entropy)
    check(d, want.cpu(), (tol + rounding(want, x.dtype)).cpu(), "gradient of the log-probabilities")
    step, adv = (0.05 * torch.rand((B,), generator=g).cuda() + 0.01), torch.randn((B,), generator=g).cuda()
    old = (pick(w.logp, actions) - step).float()
    kl_coef = 0.0 if ref is None else 0.3
    want = [v.cpu() for v in policy_64(x, actions, old, adv, 0.2, 0.2, kl_coef, 0.02, None, ref)]
    out = ops().policy_loss(t, actions, old, adv, kl_coef=kl_coef, ref_logits=ref, entropy_coef=0.02)
    check(out.loss, want[0], want[1], "loss")
    check(out.stats, want[2], want[3], "stats")
    (d,) = torch.autograd.grad(out.loss, t)
    check(d, want[4], want[5] + rounding(want[4], x.dtype), "gradient of the loss")


def rows_of(values, A, dtype, repeat):
    values = [v for v in values if abs(v) <= torch.finfo(DTYPES[dtype]).max] if dtype == "f16" else values
    return torch.tensor(values, dtype=torch.float64).clamp(torch.finfo(DTYPES[dtype]).min, torch.finfo(DTYPES[dtype]).max).to(DTYPES[dtype])[:, None].repeat(repeat, A).cuda()


def watched_inputs(B, A, dtype, seed):
    g = gen(seed)
    x = (2 * torch.randn((B, A), generator=g)).to(DTYPES[dtype])
    actions = torch.randint(0, A, (B,), generator=g)
    old = (pick(Rows64(x).logp, actions) - 0.05 * torch.rand((B,), generator=g) - 0.01).float()
    return g, x, actions, old, torch.randn((B,), generator=g)


@pytest.mark.parametrize("A,repeat", WIDTHS)
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_rows_of_one_value(A, repeat, dtype):
    """wholly masked, or diverged all alike: a uniform distribution, whatever the value; beside an ordinary reference, and as one"""
    x = rows_of(FILLS, A, dtype, repeat)
    g = gen(A)
    actions = torch.randint(0, A, (x.shape[0],), generator=g).cuda()
    compare(x, actions, 1, None)
    other = (2 * torch.randn(x.shape, generator=g)).to(x.dtype).cuda()
    compare(x, actions, 2, other)
    compare(other, actions, 3, x)


@pytest.mark.parametrize("A,repeat", WIDTHS)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_of_two_values(A, repeat, dtype):
    """two values in a row, one in its first half and one in the second, or in one column alone: whole lanes, waves and batches see only one of them"""
    rows = []
    for a, b in HALVES:
        for row in (torch.full((A,), a, dtype=torch.float64), torch.full((A,), b, dtype=torch.float64)):
            row[A // 2:] = b
            rows.append(row.clone())
            rows.append(row.flip(0))
        alone = torch.full((A,), b, dtype=torch.float64)
        alone[A - 1] = a
        rows.append(alone)
    x = torch.stack(rows).clamp(torch.finfo(DTYPES[dtype]).min, torch.finfo(DTYPES[dtype]).max).to(DTYPES[dtype]).repeat(1 if repeat == 1 else 9, 1).cuda()
    actions = x.argmax(1)
    compare(x, actions, 4, None)
    compare(x, actions, 5, x.flip(0) * 0 + x)


@pytest.mark.parametrize("A,repeat", WIDTHS[1:])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_rows_with_finite_masks(A, repeat, dtype):
    """columns masked with one finite value, or with several: those of whole lanes, waves and batches among them, in the logits, the reference or both"""
    g = gen(A + 1)
    dt = DTYPES[dtype]
    masks = [-1e4, -65504.0] if dtype == "f16" else [-1e9, -1e10, -1e12, -1e20, -1e30, -3e38, torch.finfo(dt).min]
    B = (len(masks) + 2) * (1 if repeat == 1 else 58)
    x, ref = ((2 * torch.randn((B, A), generator=g)).to(dt) for _ in range(2))
    masked = torch.rand((B, A), generator=g) < 0.3
    masked[:, A // 8:A // 2] = True
    masked[1::3, A // 2:A - 3] = True
    masked[:, A - 1] = False
    several = torch.tensor(masks)[torch.randint(0, len(masks), (B, A), generator=g)]
    value = torch.tensor((masks + [0.0, 0.0]) * (B // (len(masks) + 2)))[:, None].expand(B, A)
    value = torch.where(value == 0, several, value).to(dt)
    both, mine = torch.where(masked, value, x), torch.where(masked, torch.tensor(masks[0], dtype=dt), x)
    masked_ref = torch.where(masked, value, ref)
    actions = torch.full((B,), A - 1).cuda()
    compare(both.cuda(), actions, 6, None)
    compare(both.cuda(), actions, 7, masked_ref.cuda())
    compare(mine.cuda(), actions, 8, ref.cuda())
    # a reference that excludes with a finite number what the policy may do: KL is about as large as that number, and a number
    far = torch.where(masked, torch.where(value.float() < -1e30, torch.tensor(-1e30), value.float()).to(dt), ref)
    compare(x.cuda(), actions, 9, far.cuda())


@pytest.mark.parametrize("A,repeat", WIDTHS + [(32001, 1)])
@pytest.mark.parametrize("dtype,shift", [("f32", 500.0), ("f32", -5000.0), ("f32", 1e5), ("bf16", 500.0), ("bf16", -30.0), ("f16", -500.0)])
def test_shifted_rows_keep_their_precision(A, repeat, dtype, shift):
    """the gradients of every width carry the rounding of differences, not of the logits themselves"""
    g = gen(A + 4)
    x = (2 * torch.randn((10 * repeat, A), generator=g) + shift).to(DTYPES[dtype])
    actions = torch.randint(0, A, (x.shape[0],), generator=g)
    compare(x.cuda(), actions.cuda(), 10, (x.float() + 0.3 * torch.randn(x.shape, generator=g)).to(x.dtype).cuda())


@pytest.mark.parametrize("A,repeat", WIDTHS[1:])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_nan_in_the_reference_is_not_lost(A, repeat, dtype):
    """among columns so far below the reference's largest that their exponentials are zero, and with the policy's share there zero too"""
    B = 4 * (1 if repeat == 1 else 130)
    g, x, actions, old, adv = watched_inputs(B, A, dtype, A + 6)
    ref = x.clone()
    ref[1::4, :A // 2] = -300.0
    ref[1::4, 0] = float("nan")
    x[2::4, :A // 2] = ref[2::4, :A // 2] = -300.0
    ref[2::4, 0] = float("nan")
    actions[2::4] = A - 1
    old[2::4] = (pick(Rows64(x).logp, actions) - 0.05).float()[2::4]
    t = x.cuda().requires_grad_()
    out = ops().policy_loss(t, actions.cuda(), old.cuda(), adv.cuda(), kl_coef=0.3, ref_logits=ref.cuda())
    (d,) = torch.autograd.grad(out.loss, t)
    assert out.loss.isnan() and out.stats[1].isnan() and not out.stats[[0, 2, 3]].isnan().any()
    for r in range(B):
        held = d[r, A // 2:]  # where the policy has no share its gradient is zero, whatever it is multiplied with
        assert held.isnan().all() if r % 4 in (1, 2) else d[r].isfinite().all(), r


def edges(size):
    """columns around which another number of lanes and chunks, or another kernel, takes a row: of 16-byte chunks of `size` values"""
    few = [4 * size * 2, 4 * size * 3, 4 * size * 5, 8 * size * 3, 16 * size * 5, 64 * size * 3, 256 * size, 64 * size * 5, 64 * size * 8]
    many = [128 * size * 5, 256 * size * 5]
    return [(4, a + d) for a in few for d in (-1, 0, 1)] + [(513, a + d) for a in many for d in (0, 1)]


@pytest.mark.parametrize("B,A,dtype", [(B, A, "bf16") for B, A in edges(8)] + [(B, A, "f32") for B, A in edges(4)])
def test_widths_at_which_another_kernel_begins(B, A, dtype):
    g = gen(A + 5)
    x = (2 * torch.randn((B, A), generator=g)).to(DTYPES[dtype]).cuda()
    actions = torch.randint(0, A, (B,), generator=g).cuda()
    ref = (x.float() + 0.3 * torch.randn((B, A), generator=g).cuda()).to(x.dtype)
    compare(x, actions, 11, None, "pitch")
    compare(x, actions, 12, ref)


@pytest.mark.parametrize("A,repeat", WIDTHS)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_reference_without_weight_does_not_reach_the_gradient(A, repeat, dtype):
    """kl_coef = 0, the KL only watched: reference columns of -inf, of the lowest value and NaN, and rows of nothing else, change the statistics alone"""
    B = 6 * (1 if repeat == 1 else 87)
    g, x, actions, old, adv = watched_inputs(B, A, dtype, A + 2)
    ref = (x.float() + 0.3 * torch.randn((B, A), generator=g)).to(x.dtype)
    ref[1::6, A // 2:] = float("-inf")
    ref[2::6, ::2] = torch.finfo(x.dtype).min
    ref[3::6] = float("-inf")
    ref[4::6, A - 1] = float("nan")
    ref[5::6, 0] = float("inf")
    want = [v.cpu() for v in policy_64(x.cuda(), actions.cuda(), old.cuda(), adv.cuda(), 0.2, 0.2, 0.0, 0.02)]
    t = x.cuda().requires_grad_()
    out = ops().policy_loss(t, actions.cuda(), old.cuda(), adv.cuda(), kl_coef=0.0, ref_logits=ref.cuda(), entropy_coef=0.02)
    assert out.stats[1].isnan()
    check(out.loss, want[0], want[1], "loss")
    check(out.stats[[0, 2, 3]], want[2][[0, 2, 3]], want[3][[0, 2, 3]], "stats")
    (d,) = torch.autograd.grad(out.loss, t, retain_graph=True)
    check(d, want[4], want[5] + rounding(want[4], x.dtype), "gradient")
    (d,) = torch.autograd.grad(out.loss * 4, t)
    check(d, want[4] * 4, want[5] * 4 + rounding(want[4] * 4, x.dtype), "gradient of 4 times the loss")


@pytest.mark.parametrize("A,repeat", WIDTHS)
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_an_estimator_without_weight_does_not_reach_the_gradient(A, repeat, dtype):
    """as above with the reference's log-probabilities: of actions that the policy has all but excluded (the estimator's exponential is infinite), or has"""
    B = 5 * (1 if repeat == 1 else 104)
    g, x, actions, old, adv = watched_inputs(B, A, dtype, A + 3)
    x[0::5] = 0
    x[0::5, A - 1] = -120.0
    x[1::5, A - 1] = float("-inf")
    actions[0::5] = actions[1::5] = A - 1
    old[0::5] = old[1::5] = -1.0
    ref = old + 0.2
    ref[0::5] = ref[1::5] = 0.0
    ref[2::5] = float("-inf")
    ref[3::5] = float("nan")

    def loss(t, **kw):
        return ops().policy_loss(t, actions.cuda(), old.cuda(), adv.cuda(), entropy_coef=0.02, **kw)

    t = x.cuda().requires_grad_()
    want, out = loss(t), loss(t, kl_coef=0.0, ref_logprobs=ref.cuda())
    (d,), (e,) = torch.autograd.grad(want.loss, t), torch.autograd.grad(out.loss, t)
    assert torch.equal(out.loss, want.loss) and torch.equal(out.stats[[0, 2, 3]], want.stats[[0, 2, 3]]) and out.stats[1].isnan()
    assert d.isfinite().all() and torch.equal(d, e)
