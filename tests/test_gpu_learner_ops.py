"""
GPU: the learner operators (procgen_amd/learner_ops.py) against plain 64-bit implementations, element by element.

Tolerances are running error bounds, computed in 64 bits beside the expected values.  U is half a step of 32-bit arithmetic.  A recurrence rounds
once per step and joins pieces of a chain in a few more roundings, each relative to at most S[t] = |gate| S[t-1] + |update| (no cancellation), and
hands errors on through its gates: E[t] = |gate| E[t-1] + 8 U S[t].  A row of logits with x = l - max: exp(x) is off by (2 |x| + 3) U relative (the
product with log2 e, two ulps of the hardware's exp), a sum of n columns by one rounding per term added to one lane's partial sum at the most,
n / 64, and 32 for the joins and the row's own scalar operations.  An output of type t is off by half a step of t more, eps / 2 relative, and by half
a step of its smallest subnormal.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -126}  # a flushed 32-bit subnormal; a step of fp16's subnormals


def ops():
    from procgen_amd import learner_ops

    return learner_ops


def rounding(expected, dtype):
    return expected.abs() * (torch.finfo(dtype).eps / 2) + TINY[dtype]


def check(got, expected, tol, what):
    got = got.detach().double().cpu()
    assert got.shape == expected.shape, what
    same = (got == expected) | (got.isnan() & expected.isnan())
    bad = ~same & ~((got - expected).abs() <= tol)
    if bad.any():
        i = tuple(int(k) for k in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {i}: got {got[i].item()!r}, expected {expected[i].item()!r}, allowed {tol[i].item() if tol.dim() else tol.item()!r}")


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rand(shape, g, dtype=torch.float32, scale=1.0, shift=0.0):
    return (torch.randn(shape, generator=g) * scale + shift).to(dtype)


# ---- the recurrence ---------------------------------------------------------------------------------------------------------------------------


def recurrence_64(gate, update, first=None, state=None, d_h=None, d_last=None):
    """the formulas step by step, [T, N, D] on the CPU, with the running error bounds of every result"""
    a, b = gate.double(), update.double()
    T = a.shape[0]
    cut = torch.zeros(a.shape[:2], dtype=torch.bool) if first is None else first.bool()
    cut = cut[:, :, None]
    start = torch.zeros(a.shape[1:], dtype=torch.float64) if state is None else state.double()
    out = {"h": torch.empty_like(b), "E_h": torch.empty_like(b)}
    h, S, E = start, start.abs(), torch.zeros_like(start)
    before, E_before = [], []
    for t in range(T):
        before.append(h), E_before.append(E)
        h = torch.where(cut[t], b[t], a[t] * h + b[t])
        S = torch.where(cut[t], b[t].abs(), a[t].abs() * S + b[t].abs())
        E = torch.where(cut[t], torch.zeros_like(E), a[t].abs() * E) + 8 * U * S
        out["h"][t], out["E_h"][t] = h, E
    out["last"], out["E_last"] = h, E
    if d_h is not None or d_last is not None:
        for k in ("d_gate", "d_update", "E_d_gate", "E_d_update"):
            out[k] = torch.empty_like(b)
        g = torch.zeros_like(start) if d_last is None else d_last.double()
        S, E = g.abs(), torch.zeros_like(g)
        for t in reversed(range(T)):
            d = torch.zeros_like(g) if d_h is None else d_h[t].double()
            g, S = g + d, S + d.abs()
            E = E + 8 * U * S
            out["d_update"][t], out["E_d_update"][t] = g, E
            zero = torch.zeros_like(g)
            out["d_gate"][t] = torch.where(cut[t], zero, g * before[t])
            out["E_d_gate"][t] = torch.where(cut[t], zero, g.abs() * E_before[t] + E * before[t].abs() + E * E_before[t] + U * (g * before[t]).abs())
            g, S, E = (torch.where(cut[t], zero, k * x) for k, x in ((a[t], g), (a[t].abs(), S), (a[t].abs(), E)))
        out["d_state"], out["E_d_state"] = g, E + 8 * U * S
    return out


def recurrence_inputs(T, N, D, dtype, seed, first=True, state=True, layout="tnd"):
    g = gen(seed)
    dt = DTYPES[dtype]
    gate = torch.sigmoid(rand((T, N, D), g, scale=1.5, shift=2.0)).to(dt)
    gate[rand((T, N, D), g) > 2.0] *= -1  # gates of either sign, and some beyond one
    gate[rand((T, N, D), g) > 2.5] *= 1.25
    update = rand((T, N, D), g, dt)
    f = (torch.rand((T, N), generator=g) < 0.05).to(torch.uint8) * 3 if first else None  # any value but zero is set
    s = rand((N, D), g) if state else None

    def put(x):
        if layout == "tnd":
            return x.cuda()
        if layout == "ntd":  # a batch-major window
            return x.transpose(0, 1).contiguous().cuda().transpose(0, 1)
        if layout == "slice":  # every second step of a wider, longer tensor, at an odd offset
            wide = torch.full((2 * T + 1, N + 1, 2 * D + 3), float("nan"), dtype=x.dtype)
            view = wide[1::2, 1:, 3:3 + D]
            view.copy_(x)
            return wide.cuda()[1::2, 1:, 3:3 + D]
        wide = torch.full((T, N, 2 * D), float("nan"), dtype=x.dtype)  # "strided": every second channel
        wide[:, :, ::2] = x
        return wide.cuda()[:, :, ::2]

    return gate, update, f, s, put


RECURRENCES = [
    (1, 1, 1, "f32", True, True, "tnd"), (1, 5, 64, "bf16", True, True, "tnd"), (2, 3, 7, "f16", True, False, "tnd"), (17, 4, 128, "bf16", True, True, "tnd"),
    (63, 2, 32, "f32", False, True, "tnd"), (64, 1, 256, "bf16", True, True, "tnd"), (65, 3, 40, "f16", True, True, "ntd"), (127, 9, 24, "bf16", False, False, "slice"),
    (129, 2, 33, "f32", True, True, "strided"), (256, 8, 64, "bf16", True, True, "ntd"), (1000, 1, 5, "f32", True, True, "tnd"), (2049, 1, 16, "f16", False, True, "tnd"),
    (5000, 2, 3, "bf16", True, True, "ntd"), (31, 1, 2000, "f32", True, False, "slice"), (40, 300, 1, "bf16", True, True, "strided"), (7, 129, 65, "f16", True, True, "tnd"),
    (12345, 1, 1, "f32", True, True, "tnd"), (3, 700, 100, "bf16", True, True, "tnd"), (4, 300, 257, "f16", True, False, "ntd"), (1, 2100, 133, "f32", True, True, "slice"),
    (1, 9000, 61, "bf16", True, True, "tnd"), (4, 40, 30, "f32", False, True, "strided"), (5, 900, 150, "bf16", True, True, "tnd"), (100, 700, 101, "bf16", True, True, "ntd"),
    (20000, 1, 70, "bf16", True, True, "slice"), (200, 33, 500, "f32", True, True, "tnd"), (150, 64, 257, "bf16", True, True, "ntd"), (97, 5, 3301, "f16", False, True, "slice"),
]


@pytest.mark.parametrize("T,N,D,dtype,first,state,layout", RECURRENCES)
def test_gated_recurrence(T, N, D, dtype, first, state, layout):
    gate, update, f, s, put = recurrence_inputs(T, N, D, dtype, T + N + D, first, state, layout)
    g = gen(5)
    d_h, d_last = rand((T, N, D), g, DTYPES[dtype]), rand((N, D), g)
    want = recurrence_64(gate, update, f, s, d_h, d_last)
    a, b = put(gate).requires_grad_(), put(update).requires_grad_()
    fc, sc = None if f is None else f.cuda(), None if s is None else s.cuda().requires_grad_()
    h, last = ops().gated_recurrence(a, b, fc, sc)
    dt = DTYPES[dtype]
    assert h.dtype == dt and last.dtype == torch.float32
    check(h, want["h"], want["E_h"] + rounding(want["h"], dt), "h")
    check(last, want["last"], want["E_last"] + TINY[torch.float32], "state")
    leaves = [a, b] + ([sc] if state else [])
    got = torch.autograd.grad([h, last], leaves, [put(d_h), d_last.cuda()])
    h_read = want["E_h"] + rounding(want["h"], dt)  # the backward pass may read h as it was returned
    more = torch.cat([torch.zeros(1, N, D), h_read[:-1]]) * (want["d_update"].abs() + want["E_d_update"])
    check(got[1], want["d_update"], want["E_d_update"] + rounding(want["d_update"], dt), "d_update")
    check(got[0], want["d_gate"], want["E_d_gate"] + more + rounding(want["d_gate"], dt), "d_gate")
    if state:
        check(got[2], want["d_state"], want["E_d_state"] + TINY[torch.float32], "d_state")
    with torch.no_grad():  # the call without gradients gives the same bits
        h2, last2 = ops().gated_recurrence(a, b, fc, sc)
    assert torch.equal(h2, h) and torch.equal(last2, last)


@pytest.mark.parametrize("T", [1, 70, 3000])
def test_gated_recurrence_cuts_whatever_is_behind_the_first_step(T):
    """NaN and infinities in the gates at a cut, in the state before it and in the steps of the other episode: nothing of them passes the cut, in
    either direction"""
    N, D, at = 3, 10, T // 2
    gate, update, f, s, _ = recurrence_inputs(T, N, D, "f32", 3)
    f.zero_()
    f[at, 1] = 1
    bad = [x.clone() for x in (gate, update, s)]
    bad[0][at, 1] = float("nan")
    bad[0][:at, 1] = float("inf")
    bad[1][:at, 1] = float("nan")
    bad[2][1] = float("-inf")
    a, b, s0 = (x.cuda().requires_grad_() for x in bad)
    h, last = ops().gated_recurrence(a, b, f.cuda(), s0)
    want = recurrence_64(gate, update, f, s, torch.ones(T, N, D), None)
    rows = [0, 2]
    check(h[:, rows], want["h"][:, rows], want["E_h"][:, rows] + rounding(want["h"][:, rows], torch.float32), "other envs")
    check(h[at:, 1], want["h"][at:, 1], want["E_h"][at:, 1] + rounding(want["h"][at:, 1], torch.float32), "behind the cut")
    check(last, want["last"], want["E_last"] + TINY[torch.float32], "state")
    d = torch.autograd.grad(h.sum(), [a, b, s0])  # the incoming gradient is an expanded scalar
    check(d[1][at:, 1], want["d_update"][at:, 1], want["E_d_update"][at:, 1] + rounding(want["d_update"][at:, 1], torch.float32), "d_update behind the cut")
    assert (d[0][at, 1] == 0).all()
    if at:
        check(d[1][at - 1, 1], torch.ones(D, dtype=torch.float64), torch.zeros(()), "the step before the cut gets its own gradient alone")
    else:
        assert (d[2][1] == 0).all()
    assert d[2][rows].isfinite().all()


def test_gated_recurrence_takes_two_dimensions_no_steps_and_expanded_gates():
    o = ops()
    g = gen(1)
    gate, update, state = torch.rand((50, 30), generator=g), rand((50, 30), g), rand((30,), g)
    h, last = o.gated_recurrence(gate.cuda(), update.cuda(), None, state.cuda())
    want = recurrence_64(gate[:, :, None], update[:, :, None], None, state[:, None])
    check(h, want["h"][:, :, 0], want["E_h"][:, :, 0] + rounding(want["h"][:, :, 0], torch.float32), "h")
    assert last.shape == (30,)
    h, last = o.gated_recurrence(gate[:0].cuda(), update[:0].cuda(), None, state.cuda())
    assert h.shape == (0, 30) and torch.equal(last.cpu(), state)
    h, last = o.gated_recurrence(gate[:, :0].cuda(), update[:, :0].cuda())
    assert h.shape == (50, 0) and last.shape == (0,)
    out = state.cuda().clone()
    with torch.no_grad():
        o.gated_recurrence(gate[:0].cuda(), update[:0].cuda(), None, state.cuda(), state_out=out)
    assert torch.equal(out.cpu(), state)
    # one decay per channel, shared by all steps and envs: its gradient is the sum over them
    T, N, D = 40, 6, 32
    decay = torch.rand(D, generator=g).cuda().requires_grad_()
    update = rand((T, N, D), g)
    h, last = o.gated_recurrence(decay.expand(T, N, D), update.cuda())
    (d,) = torch.autograd.grad(h.sum(), decay)
    want = recurrence_64(decay.detach().cpu().expand(T, N, D), update, None, None, torch.ones(T, N, D))
    tol = (want["E_d_gate"] + rounding(want["d_gate"], torch.float32)).sum((0, 1)) + want["d_gate"].abs().sum((0, 1)) * U * T * N + (want["E_h"].sum((0, 1)) * want["d_update"].abs().amax((0, 1)))
    check(d, want["d_gate"].sum((0, 1)), tol, "shared gate")


def test_gated_recurrence_of_one_tensor_as_gate_and_update():
    g = gen(2)
    x = torch.rand((33, 2, 20), generator=g)
    a = x.cuda().requires_grad_()
    h, _ = ops().gated_recurrence(a, a)
    (d,) = torch.autograd.grad(h.sum(), a)
    w = recurrence_64(x, x, None, None, torch.ones_like(x))
    check(d, w["d_gate"] + w["d_update"], w["E_d_gate"] + w["E_d_update"] + (w["E_h"] + rounding(w["h"], torch.float32)).amax() * w["d_update"].abs() + 4 * U * (w["d_gate"].abs() + w["d_update"].abs()), "sum of both gradients")


def test_gated_recurrence_gradients_agree_with_differences():
    """f(step s) = <h(x + s d), w> is a polynomial in s: (f(s) - f(-s)) / 2s = f' + s^2 f''' / 6 + ...; the third derivative of 6 steps' products is
    computed in 64 bits, and the two values of f are off by their running error bounds"""
    T, N, D, s = 6, 2, 3, 2.0 ** -5
    gate, update, f, state, _ = recurrence_inputs(T, N, D, "f32", 9)
    g = gen(4)
    w = rand((T, N, D), g)
    way = [rand(x.shape, g) for x in (gate, update, state)]

    def at(k, x64=False):
        moved = [x.double() + k * d.double() if x64 else x + k * d for x, d in zip((gate, update, state), way)]
        if x64:
            return float((recurrence_64(moved[0], moved[1], f, moved[2])["h"] * w.double()).sum())
        h, _ = ops().gated_recurrence(moved[0].cuda(), moved[1].cuda(), f.cuda(), moved[2].cuda())
        bound = recurrence_64(moved[0], moved[1], f, moved[2])
        slack = ((bound["E_h"] + rounding(bound["h"], torch.float32) + 16 * U * bound["h"].abs().amax()) * w.abs().double()).sum()
        return float((h.double().cpu() * w.double()).sum()), float(slack)

    leaves = [x.cuda().requires_grad_() for x in (gate, update, state)]
    h, _ = ops().gated_recurrence(leaves[0], leaves[1], f.cuda(), leaves[2])
    d = torch.autograd.grad(h, leaves, w.cuda())
    slope = sum(float((x.double().cpu() * y.double()).sum()) for x, y in zip(d, way))
    (hi, e1), (lo, e2) = at(s), at(-s)
    third = (at(2 * s, True) - 2 * at(s, True) + 2 * at(-s, True) - at(-2 * s, True)) / (2 * s ** 3)
    assert abs((hi - lo) / (2 * s) - slope) <= abs(third) * s * s / 6 * 2 + (e1 + e2) / (2 * s) + 1e-5 * abs(slope) + 1e-6


def test_gated_recurrence_in_place_single_steps_equal_the_window():
    T, N, D = 24, 7, 48
    gate, update, f, s, _ = recurrence_inputs(T, N, D, "bf16", 8)
    gate, update, f = gate.cuda(), update.cuda(), f.cuda()
    with torch.no_grad():
        state = s.cuda()
        steps = [ops().gated_recurrence(gate[t:t + 1], update[t:t + 1], f[t:t + 1], state, state_out=state)[0] for t in range(T)]
    want = recurrence_64(gate.cpu(), update.cpu(), f.cpu(), s)
    check(torch.cat(steps), want["h"], want["E_h"] + rounding(want["h"], torch.bfloat16), "steps")
    check(state, want["last"], want["E_last"], "state moved in place")
    for T in (300, 9000):  # a state moved on in place by a whole window, one that is cut into pieces too
        gate, update, f, s, _ = recurrence_inputs(T, 1, 20, "f32", 8)
        state = s.cuda()
        with torch.no_grad():
            h, got = ops().gated_recurrence(gate.cuda(), update.cuda(), f.cuda(), state, state_out=state)
        assert got.data_ptr() == state.data_ptr()
        want = recurrence_64(gate, update, f, s)
        check(h, want["h"], want["E_h"] + rounding(want["h"], torch.float32), "h")
        check(state, want["last"], want["E_last"], "state")


def test_gated_recurrence_refuses_a_state_out_inside_of_its_inputs():
    x = torch.zeros((6, 2, 4), device="cuda")
    state = torch.zeros((3, 4), device="cuda")
    with torch.no_grad():
        for out, kw in ((x[0], {}), (x[5], {}), (state[1:], {"state": state[:2]}), (state.view(-1)[:8].view(2, 4), {"state": state.view(-1)[:8].view(4, 2).T})):
            with pytest.raises(ValueError):
                ops().gated_recurrence(x, x, state_out=out, **kw)
        rows = torch.zeros((2, 2, 4), device="cuda")
        ops().gated_recurrence(x, x, state=rows[0], state_out=rows[1])  # neighbours in one buffer are no overlap


def test_a_state_that_was_moved_on_in_place_is_not_used_by_an_older_graph():
    g = gen(3)
    gate, update, state = torch.rand((4, 2, 8), generator=g).cuda().requires_grad_(), rand((4, 2, 8), g).cuda(), rand((2, 8), g).cuda()
    h, _ = ops().gated_recurrence(gate, update, None, state)
    with torch.no_grad():
        ops().gated_recurrence(gate, update, None, state, state_out=state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        h.sum().backward()


def test_gated_recurrence_reaches_beyond_32_bits():
    """3 x 2^30 elements of output: gates and updates are expanded scalars, so that h[t] = 2 - 2^-t"""
    T, D = 3 << 20, 1024
    one = torch.ones((), dtype=torch.bfloat16, device="cuda")
    with torch.no_grad():
        h, last = ops().gated_recurrence((one * 0.5).expand(T, 1, D), one.expand(T, 1, D))
    assert h.numel() * 2 > 1 << 32 and (last == 2).all()
    for t in (0, 1, 2, 100, T // 2, T - 1):
        assert (h[t] == 2 - 2.0 ** -min(t, 100)).all(), t
    assert (h[1 << 20:, 0, ::257] == 2).all()


# ---- advantages -------------------------------------------------------------------------------------------------------------------------------


def advantages_64(rew, values, first, gamma, lam):
    r, v, live = rew.double(), values.double(), first == 0
    T = r.shape[0]
    adv, E_adv = torch.empty_like(r), torch.empty_like(r)
    zero = torch.zeros_like(r[0])
    A, S, E = zero, zero, zero
    g32, gl32 = float(np.float32(gamma)), float(np.float32(np.float32(gamma) * np.float32(lam)))
    for t in reversed(range(T)):
        nxt = torch.where(live[t + 1], v[t + 1], zero)
        delta, size = r[t] + g32 * nxt - v[t], r[t].abs() + g32 * nxt.abs() + v[t].abs()
        A = torch.where(live[t + 1], gl32 * A, zero) + delta
        S = torch.where(live[t + 1], gl32 * S, zero) + size
        E = torch.where(live[t + 1], gl32 * E, zero) + 8 * U * S
        adv[t], E_adv[t] = A, E
    return adv, E_adv, adv + v[:-1], E_adv + U * (adv + v[:-1]).abs()


@pytest.mark.parametrize("T,N,dtype,gamma,lam,layout", [
    (1, 1, "f32", 0.999, 0.95, "tn"), (2, 65, "bf16", 0.99, 0.9, "tn"), (16, 64, "f32", 0.999, 0.95, "tn"), (31, 1000, "f16", 0.999, 0.95, "nt"), (64, 3, "f32", 1.0, 1.0, "tn"),
    (65, 130, "bf16", 0.9, 0.0, "nt"), (257, 512, "f32", 0.999, 0.95, "slice"), (1000, 7, "f16", 0.0, 0.95, "tn"), (4097, 2, "f32", 0.999, 0.95, "nt"), (10007, 1, "bf16", 1.0, 1.0, "tn"),
    (5, 70000, "f32", 0.999, 0.95, "tn"),
    (300, 8195, "f32", 0.999, 0.95, "tn"), (70, 20001, "bf16", 0.999, 0.95, "nt"), (7, 9000, "f32", 0.999, 0.95, "tn"),
])
def test_advantages(T, N, dtype, gamma, lam, layout):
    g = gen(T + N)
    rew = torch.where(torch.rand((T, N), generator=g) < 0.1, 10 * torch.rand((T, N), generator=g), torch.zeros(()))
    values = rand((T + 1, N), g, DTYPES[dtype], 2.0, 5.0)
    first = (torch.rand((T + 1, N), generator=g) < 0.03)
    values[1:][first[1:]] = float("nan")  # the value of the observation that replaced an ended episode's last one is not looked at ...
    values[:-1][first[:-1]] = 1.0  # ... for the step that ended; the next step starts from it
    if first[-1].any():
        values[-1][first[-1]] = float("inf")

    def put(x):
        if layout == "nt":
            return x.T.contiguous().cuda().T
        if layout == "slice":
            wide = torch.zeros((2 * x.shape[0], x.shape[1] + 5), dtype=x.dtype)
            wide[::2, 3:-2] = x
            return wide.cuda()[::2, 3:-2]
        return x.cuda()

    got = ops().advantages(put(rew), put(values), put(first.to(torch.uint8) * 255) if layout == "nt" else put(first), gamma=gamma, lam=lam)
    adv, E_adv, ret, E_ret = advantages_64(rew, values, first, gamma, lam)
    check(got[0], adv, E_adv + TINY[torch.float32], "advantages")
    check(got[1], ret, E_ret + TINY[torch.float32], "returns")


def test_advantages_of_nothing():
    for T, N in ((0, 4), (4, 0)):
        adv, ret = ops().advantages(torch.zeros((T, N), device="cuda"), torch.zeros((T + 1, N), device="cuda"), torch.zeros((T + 1, N), dtype=torch.uint8, device="cuda"), gamma=0.9, lam=0.9)
        assert adv.shape == ret.shape == (T, N)


# ---- rows of logits ----------------------------------------------------------------------------------------------------------------------------


class Rows64:
    """log p, p, entropy of rows [B, A] in 64 bits, and how far 32-bit sums may be off"""

    def __init__(self, logits):
        x = logits.double()
        self.m = x.amax(1, keepdim=True)
        self.empty = (self.m == float("-inf"))[:, 0]
        self.x = torch.where(self.empty[:, None], torch.full_like(x, float("-inf")), x - torch.where(self.empty[:, None], torch.zeros_like(self.m), self.m))
        e = self.x.exp()
        self.s = e.sum(1, keepdim=True)
        self.p = torch.where(self.empty[:, None], torch.zeros_like(e), e / self.s)
        self.logp = self.x - self.s.log()
        xf = torch.where(self.p > 0, self.x, torch.zeros_like(self.x))  # where p underflows, nothing is added
        self.finite_logp = torch.where(self.p > 0, self.logp, torch.zeros_like(self.x))
        self.H = -(self.p * self.finite_logp).sum(1)
        self.mean_x, self.mean_x2 = (self.p * xf.abs()).sum(1), (self.p * xf * xf).sum(1)
        n = logits.shape[1]
        self.rel_s = U * (2 * self.mean_x + 3 + n / 64 + 32)  # of the sum
        self.T_logp = (self.rel_s[:, None] + U * (2 * xf.abs() + 2 * self.finite_logp.abs() + 2 * self.s.log().abs() + 8))  # of log p[j], absolute
        self.T_H = self.rel_s * (1 + self.mean_x) + U * (2 * self.mean_x2 + 4 * self.mean_x + (n / 64 + 32) * self.mean_x + 4 * self.H + 2 * self.s.log()[:, 0].abs() + 8)
        self.rel_p = self.rel_s[:, None] + U * (2 * xf.abs() + 8)


def pick(x, actions):
    return x.gather(1, actions.long()[:, None])[:, 0]


def put_rows(x, layout):
    """[B, A] rows as the tensor that the call gets"""
    B, A = x.shape
    if layout == "plain":
        return x.cuda()
    if layout == "pitch":  # rows of a wider tensor, at an odd offset
        wide = torch.full((B, A + 7), float("nan"), dtype=x.dtype)
        wide[:, 3:3 + A] = x
        return wide.cuda()[:, 3:3 + A]
    wide = torch.full((2, B // 2 + 3, A), float("nan"), dtype=x.dtype)  # "window": [2, B / 2, A] out of longer windows
    wide[:, :B // 2] = x.reshape(2, B // 2, A)
    return wide.cuda()[:, :B // 2]


LOGITS = [
    (1, 1, "f32", "plain"), (1, 2, "bf16", "plain"), (3, 15, "f32", "plain"), (64, 15, "bf16", "plain"), (130, 15, "f16", "pitch"), (1000, 15, "bf16", "window"), (257, 16, "f32", "plain"),
    (65, 7, "bf16", "plain"), (100, 63, "f16", "window"), (77, 64, "bf16", "plain"), (77, 65, "f32", "plain"), (40, 128, "bf16", "pitch"), (33, 1000, "bf16", "plain"), (8, 1023, "f16", "pitch"),
    (5, 4099, "f32", "plain"), (300, 4096, "bf16", "plain"), (2, 32001, "bf16", "plain"), (1, 131072, "f16", "plain"), (3, 50021, "bf16", "pitch"), (1, 100003, "f32", "plain"), (6, 20000, "f32", "window"),
    (129, 16, "f32", "pitch"), (514, 16, "f32", "window"), (1000, 16, "f32", "plain"), (70, 17, "bf16", "plain"), (130, 31, "f16", "window"), (66, 24, "f32", "plain"), (200, 9, "bf16", "pitch"),
    (66, 8, "f16", "plain"), (129, 32, "bf16", "plain"),
    (321, 32, "f32", "plain"), (66, 32, "f32", "window"), (65, 32, "f32", "pitch"), (193, 25, "f32", "plain"), (70, 31, "f32", "pitch"), (500, 23, "f32", "plain"), (259, 20, "f16", "plain"),
    (321, 33, "bf16", "plain"), (130, 48, "f16", "window"), (193, 49, "bf16", "pitch"), (259, 63, "f16", "plain"), (129, 64, "bf16", "pitch"), (129, 55, "bf16", "plain"),
    (130, 3, "bf16", "pitch"), (66, 2, "f32", "window"), (130, 24, "f32", "window"), (195, 8, "bf16", "pitch"), (70, 5, "f32", "pitch"), (259, 40, "f16", "pitch"),
    (33, 90, "bf16", "plain"), (20, 150, "f16", "pitch"), (18, 190, "bf16", "window"), (21, 300, "bf16", "plain"), (17, 380, "f16", "plain"), (9, 600, "bf16", "pitch"), (9, 700, "f16", "plain"),
    (5, 1200, "bf16", "plain"), (6, 1500, "bf16", "window"), (5, 2047, "bf16", "plain"), (50, 45, "f32", "plain"), (40, 70, "f32", "window"), (30, 95, "f32", "pitch"), (19, 155, "f32", "plain"),
    (17, 190, "f32", "plain"), (12, 310, "f32", "window"), (9, 380, "f32", "plain"), (7, 601, "f32", "pitch"), (5, 767, "f32", "plain"), (5, 1277, "f32", "plain"), (3, 2040, "f32", "plain"),
]


def row_inputs(B, A, dtype, seed, scale=3.0):
    g = gen(seed)
    x = rand((B, A), g, DTYPES[dtype], scale)
    return g, x, torch.randint(0, A, (B,), generator=g, dtype=torch.int32)


@pytest.mark.parametrize("B,A,dtype,layout", LOGITS)
@pytest.mark.parametrize("shift", [0.0, 500.0])
def test_action_logprobs(B, A, dtype, layout, shift):
    g, x, actions = row_inputs(B, A, dtype, B + A)
    x = (x.float() + shift).to(x.dtype)
    if A > 2:
        x[0, 1] = float("-inf")  # an action that cannot be taken
        actions[0] = 0
    w = Rows64(x)
    t = put_rows(x, layout)
    lead = t.shape[:-1]
    t.requires_grad_()
    logp, entropy = ops().action_logprobs(t, (actions.long() if B % 2 else actions).cuda().view(lead))
    assert logp.shape == entropy.shape == lead and logp.dtype == entropy.dtype == torch.float32
    check(logp.view(B), pick(w.logp, actions), pick(w.T_logp, actions), "log-probabilities")
    check(entropy.view(B), w.H, w.T_H, "entropy")
    d_logp, d_entropy = rand((B,), g), rand((B,), g)
    (d,) = torch.autograd.grad([logp, entropy], [t], [d_logp.cuda().view(lead), d_entropy.cuda().view(lead)])
    onehot = torch.zeros_like(w.p).scatter_(1, actions.long()[:, None], 1.0)
    gl, ge = d_logp.double()[:, None], d_entropy.double()[:, None]
    both = torch.where(w.p > 0, w.finite_logp + w.H[:, None], torch.zeros_like(w.p))
    want = gl * (onehot - w.p) - ge * w.p * both
    # lse is held in 32 bits between the passes: off by U |lse| more, which p and log p inherit
    lse = U * (w.m.abs() + w.s.log().abs()) * 2
    tol = gl.abs() * w.p * (w.rel_p + lse) + ge.abs() * w.p * (both.abs() * (w.rel_p + lse) + w.T_logp + w.T_H[:, None] + lse) + 8 * U * (gl.abs() * (onehot + w.p) + ge.abs() * w.p * both.abs())
    check(d.view(B, A), want, tol + rounding(want, x.dtype), "gradient")


def test_action_logprobs_where_little_is_left():
    """masked columns of -inf and of the type's lowest value, rows with one column left or none, actions outside the columns"""
    inf, nan, low = float("inf"), float("nan"), torch.finfo(torch.float32).min
    for A in (5, 200, 9000):
        x = torch.full((8, A), -inf)
        x[0, 2] = 3.0                                # one column left
        x[1] = low                                   # all of the lowest value: uniform
        x[2] = low
        x[2, 1] = 7.0                                # one column far over the others
        x[4, :2] = 0.0                               # two columns left; row 3: none
        x[5, :2] = 0.0
        x[6, :2] = 0.0
        x[7] = 0.5
        x[7, 1] = nan
        actions = torch.tensor([2, 4, 1, 0, 3, -1, A, 0])
        t = x.cuda().requires_grad_()
        logp, entropy = ops().action_logprobs(t, actions.cuda())
        n, two = float(np.log(A)), float(np.log(2.0))
        check(logp, torch.tensor([0.0, -n, 0.0, -inf, -inf, nan, nan, nan], dtype=torch.float64), torch.tensor(64 * U + 4 * U * n + A / 64 * U), f"log-probabilities of {A}")
        check(entropy, torch.tensor([0.0, n, 0.0, 0.0, two, two, two, nan], dtype=torch.float64), torch.tensor(64 * U + 4 * U * n + A / 64 * U), f"entropy of {A}")
        up = torch.tensor([1.0, 1.0, 1.0, 1.0, 1.0, 1.0, 0.0, 0.0]).cuda()
        (d,) = torch.autograd.grad([logp, entropy], [t], [up, up * 0.5])
        assert (d[0] == 0).all() and (d[3] == 0).all(), "certain and empty rows"
        assert d[5].isnan().all() and (d[6] == 0).all() and (d[7] == 0).all(), "unknown actions; rows that nothing comes in for"
        want = torch.zeros(A, dtype=torch.float64)
        want[:2], want[3] = -0.5, 1.0  # 1[j = a] - p[j] with p = 1/2, 1/2, 0, ..., a = 3 a masked column; the entropy is at its largest, log p + H = 0
        check(d[4], want, torch.tensor(64 * U), "masked action")
        assert d[1:3].isfinite().all()


@pytest.mark.parametrize("A", [5, 40, 200, 9000])
def test_rows_with_nan_and_infinities(A):
    """NaN wherever a NaN or +inf is among the logits, as log_softmax has it; the rows beside them are as without"""
    inf, nan = float("inf"), float("nan")
    g, x, actions = row_inputs(6, A, "f32", A)
    clean = x.clone()
    x[1] = nan
    x[2, A - 1] = nan
    x[3, 0] = inf
    x[4] = -inf
    x[4, 1] = nan
    t = x.cuda().requires_grad_()
    logp, entropy = ops().action_logprobs(t, actions.cuda())
    out = ops().policy_loss(t, actions.cuda(), logp.detach(), torch.ones(6, device="cuda"), entropy_coef=0.1)
    (d,) = torch.autograd.grad([logp.sum() + entropy.sum()], t, retain_graph=True)
    (e,) = torch.autograd.grad(out.loss, t)
    for r in (1, 2, 3, 4):
        assert logp[r].isnan() and entropy[r].isnan() and d[r].isnan().all() and e[r].isnan().all(), r
    assert out.loss.isnan()
    w = Rows64(clean)
    for r in (0, 5):
        check(logp[r], pick(w.logp, actions)[r], pick(w.T_logp, actions)[r], "log-probability")
        assert d[r].isfinite().all() and e[r].isfinite().all()


def test_policy_loss_against_a_reference_that_excludes_an_action():
    """KL is infinite where the reference has no probability and the policy has; not where the policy has none either"""
    inf = float("inf")
    for A in (6, 500):
        g, x, actions, old, adv = policy_inputs(4, A, "f32", 5)
        ref = x + rand((4, A), g, scale=0.3)
        x[1, 3] = ref[1, 3] = -inf
        actions[1] = 0
        old[1] = float(Rows64(x).logp[1, 0])
        want = policy_64(x, actions, old, adv, 0.2, 0.2, 0.2, 0.0, None, ref)
        out = ops().policy_loss(x.cuda(), actions.cuda(), old.cuda(), adv.cuda(), kl_coef=0.2, ref_logits=ref.cuda())
        check(out.loss, want[0], want[1], "loss")
        check(out.stats, want[2], want[3], "stats")
        ref[2, 1] = -inf
        out = ops().policy_loss(x.cuda(), actions.cuda(), old.cuda(), adv.cuda(), kl_coef=0.2, ref_logits=ref.cuda())
        assert out.stats[1].item() == inf and out.loss.item() == inf
        out = ops().policy_loss(x.cuda(), actions.cuda(), old.cuda(), adv.cuda(), kl_coef=0.0, ref_logits=ref.cuda())
        assert out.stats[1].item() == inf and out.loss.isfinite()


def test_rows_reach_beyond_32_bits():
    """70 000 rows of 32 768 columns: the last rows against the same rows alone"""
    B, A = 70000, 32768
    x = torch.zeros((B, A), dtype=torch.bfloat16, device="cuda")
    g, tail, actions = row_inputs(5, A, "bf16", 1)
    x[-5:] = tail.cuda()
    a = torch.zeros(B, dtype=torch.int32, device="cuda")
    a[-5:] = actions.cuda()
    alone = tail.cuda().requires_grad_()
    logp, entropy = ops().action_logprobs(x, a)
    w = Rows64(tail)
    check(logp[-5:], pick(w.logp, actions), pick(w.T_logp, actions), "log-probabilities")
    check(logp[:-5], torch.full((B - 5,), -np.log(A), dtype=torch.float64), torch.tensor(64 * U + 8 * U * np.log(A) + A / 64 * U), "uniform rows")
    x.requires_grad_()
    ones, valid = torch.ones(B, device="cuda"), torch.zeros(B, dtype=torch.uint8, device="cuda")
    valid[-5:] = 1
    (d,) = torch.autograd.grad(ops().policy_loss(x, a, logp, ones, valid=valid).loss, x)
    (e,) = torch.autograd.grad(ops().policy_loss(alone, actions.cuda(), logp[-5:], ones[-5:]).loss, alone)
    # another number of lanes for a row: sums in another order, bounded as ever; then half a step of bfloat16 each
    tol = 2 * (w.rel_p * w.p / 5 + 16 * U * (1 + w.p) / 5) + rounding(e.double().cpu(), torch.bfloat16) * 2
    check(d[-5:], e.double().cpu(), tol, "gradient of the last rows")
    assert not d[:-5].any()


@pytest.mark.parametrize("shape", [(0, 5), (3, 0, 5)])
def test_rows_of_nothing(shape):
    x = torch.zeros(shape, device="cuda", requires_grad=True)
    lead = shape[:-1]
    a, f = torch.zeros(lead, dtype=torch.int32, device="cuda"), torch.zeros(lead, device="cuda")
    logp, entropy = ops().action_logprobs(x, a)
    assert logp.shape == entropy.shape == lead
    out = ops().policy_loss(x, a, f, f)
    assert out.loss.item() == 0 and (out.stats == 0).all()
    (d,) = torch.autograd.grad(out.loss, x)
    assert d.shape == shape


def policy_64(x, actions, old, adv, low, high, kl_coef, entropy_coef, valid=None, ref=None, ref_logp=None):
    """loss, stats, gradient and their tolerances, from the definition"""
    w = Rows64(x)
    A, B = x.shape[1], x.shape[0]
    use = torch.ones(B, dtype=torch.bool, device=x.device) if valid is None else valid.bool()
    n = max(1, int(use.sum()))
    use = use & ~w.empty
    logp, T = pick(w.logp, actions), pick(w.T_logp, actions)
    ratio, adv = (logp - old.double()).exp(), adv.double()
    T_ratio = ratio * (T + U * (2 * (logp - old.double()).abs() + 8))
    plain, held = ratio * adv, ratio.clamp(1 - low, 1 + high) * adv
    near = (ratio - (1 - low)).abs().minimum((ratio - (1 + high)).abs()) <= T_ratio + 4 * U
    assert not (near & use).any(), "an input lies on the border of the clip range, where the gradient jumps"
    out = plain > held
    policy, T_policy = -torch.minimum(plain, held), adv.abs() * (T_ratio + 4 * U * ratio)
    c = torch.where(out, torch.zeros_like(plain), -plain)
    T_c = torch.where(out, torch.zeros_like(plain), T_policy)
    per, T_per = entropy_coef * (w.finite_logp + w.H[:, None]), abs(entropy_coef) * (w.T_logp + w.T_H[:, None])
    kl, T_kl = torch.zeros_like(logp), torch.zeros_like(logp)
    if ref is not None:
        q = Rows64(ref)
        off = torch.where(w.p > 0, w.logp - q.logp, torch.zeros_like(w.p))
        raw = torch.where(w.p > 0, w.x - q.x, torch.zeros_like(w.p))
        kl = (w.p * off).sum(1)
        weight = (w.p * raw.abs() * (w.rel_s[:, None] + w.rel_p + U * (A / 64 + 32))).sum(1) + (w.p * (w.x.abs() + q.x.abs()).nan_to_num(0, 0, 0)).sum(1) * 4 * U
        T_kl = weight + w.rel_s + q.rel_s + 8 * U * ((q.s / w.s).log()[:, 0].abs() + 1)
        T_off = w.T_logp + U * (2 * q.x.abs() + 2 * q.logp.abs()).nan_to_num(0, 0, 0) + q.rel_s[:, None] + U * (8 + 2 * q.s.log().abs())
        per, T_per = per + kl_coef * (off - kl[:, None]), T_per + kl_coef * (T_off + T_kl[:, None] + 4 * U * off.abs())
    elif ref_logp is not None:
        z = ref_logp.double() - logp
        kl = z.expm1() - z
        T_z = T + U * z.abs()
        T_kl = (z.exp() + 1) * T_z + U * 8 * (z.expm1().abs() + z.abs())
        c = c - kl_coef * z.expm1()
        T_c = T_c + kl_coef * (z.exp() * T_z + 8 * U * z.expm1().abs())
    onehot = torch.zeros_like(w.p).scatter_(1, actions.long()[:, None], 1.0)
    c, T_c = c[:, None], T_c[:, None]
    d = (c * (onehot - w.p) + w.p * per) / n
    T_d = (T_c * (onehot + w.p) + c.abs() * w.p * w.rel_p + w.p * (per.abs() * w.rel_p + T_per) + 8 * U * (c.abs() * (onehot + w.p) + w.p * per.abs())) / n
    d, T_d = (torch.where(use[:, None], v, torch.zeros_like(v)) for v in (d, T_d))

    def mean(v):
        return torch.where(use, v, torch.zeros_like(v)).sum() / n

    clipped = ((ratio < 1 - low) | (ratio > 1 + high)).double()
    stats = torch.stack([mean(policy), mean(kl), mean(w.H), mean(clipped)])
    T_stats = torch.stack([mean(T_policy), mean(T_kl), mean(w.T_H), torch.zeros((), dtype=torch.float64, device=x.device)]) + 2 * U * stats.abs() + TINY[torch.float32]
    loss = stats[0] + kl_coef * stats[1] - entropy_coef * stats[2]
    T_loss = T_stats[0] + kl_coef * T_stats[1] + abs(entropy_coef) * T_stats[2] + 4 * U * (stats[0].abs() + kl_coef * stats[1].abs() + abs(entropy_coef) * stats[2].abs())
    return loss, T_loss, stats, T_stats, d, T_d


def policy_inputs(B, A, dtype, seed, low=0.2, high=0.2):
    g, x, actions = row_inputs(B, A, dtype, seed)
    logp = pick(Rows64(x).logp, actions)
    step = rand((B,), g, scale=0.15).double()
    for border in (np.log(1 - low), np.log(1 + high)):  # off the border
        step = torch.where((step - border).abs() < 1e-3, step + 4e-3, step)
    return g, x, actions, (logp - step).float(), rand((B,), g)


@pytest.mark.parametrize("B,A,dtype,layout", LOGITS)
@pytest.mark.parametrize("ref", ["none", "logprobs", "logits"])
def test_policy_loss(B, A, dtype, layout, ref):
    low, high = (0.2, 0.2) if B % 2 else (0.1, 0.28)
    g, x, actions, old, adv = policy_inputs(B, A, dtype, 7 * B + A, low, high)
    lead = put_rows(x, layout).shape[:-1]
    valid = (torch.rand(B, generator=g) < 0.8).to(torch.uint8) * 2 if B > 2 else None
    ref_x = (x.float() + rand((B, A), g, scale=0.5)).to(x.dtype) if ref == "logits" else None
    ref_logp = (old + rand((B,), g, scale=0.3)) if ref == "logprobs" else None
    kl_coef = 0.0 if ref == "none" else 0.3
    loss, T_loss, stats, T_stats, d, T_d = policy_64(x, actions, old, adv, low, high, kl_coef, 0.02, valid, ref_x, ref_logp)
    if valid is not None:  # whatever rows that are not valid hold
        for v in (x, ref_x, old, adv, ref_logp):
            if v is not None:
                v[valid == 0] = float("nan")
        actions[valid == 0] = -1
    t = put_rows(x, layout).requires_grad_()

    def flat(v):
        return None if v is None else v.cuda().view(lead)

    kw = dict(clip=low if low == high else (low, high), kl_coef=kl_coef, entropy_coef=0.02, valid=flat(valid), ref_logprobs=flat(ref_logp),
              ref_logits=None if ref_x is None else put_rows(ref_x, "plain").view(t.shape))
    out = ops().policy_loss(t, flat(actions), flat(old), flat(adv), **kw)
    check(out.loss, loss, T_loss, "loss")
    check(out.stats, stats, T_stats, "stats")
    assert not out.stats.requires_grad
    (got,) = torch.autograd.grad(out.loss, t, retain_graph=True)
    check(got.view(B, A), d, T_d + rounding(d, x.dtype), "gradient")
    (more,) = torch.autograd.grad(out.loss * 8.0, t)  # a second pass over the same graph, under another scale; the first one's answer stays
    check(more.view(B, A), d * 8, T_d * 8 + rounding(d * 8, x.dtype), "gradient of 8 times the loss")
    check(got.view(B, A), d, T_d + rounding(d, x.dtype), "gradient, still")
    with torch.no_grad():
        again = ops().policy_loss(t, flat(actions), flat(old), flat(adv), **kw)
    assert torch.equal(again.loss, out.loss.detach()) and torch.equal(again.stats, out.stats)


@pytest.mark.parametrize("B,A,dtype", [(130, 15, "bf16"), (70, 16, "f32"), (257, 31, "f32"), (66, 5, "f16"), (129, 200, "bf16")])
def test_policy_loss_beside_a_reference_laid_out_otherwise(B, A, dtype):
    g, x, actions, old, adv = policy_inputs(B, A, dtype, B + 3 * A)
    ref = (x.float() + rand((B, A), g, scale=0.5)).to(x.dtype)
    loss, T_loss, stats, T_stats, d, T_d = policy_64(x, actions, old, adv, 0.2, 0.2, 0.3, 0.02, None, ref, None)
    for ours, theirs in (("plain", "pitch"), ("pitch", "plain"), ("pitch", "pitch")):
        t = put_rows(x, ours).requires_grad_()
        out = ops().policy_loss(t, actions.cuda(), old.cuda(), adv.cuda(), kl_coef=0.3, entropy_coef=0.02, ref_logits=put_rows(ref, theirs))
        check(out.loss, loss, T_loss, "loss")
        check(out.stats, stats, T_stats, "stats")
        (got,) = torch.autograd.grad(out.loss, t)
        check(got, d, T_d + rounding(d, x.dtype), "gradient")


@pytest.mark.parametrize("B,A,dtype,ref", [(513, 20011, "f32", True), (515, 40003, "bf16", True), (600, 5000, "f16", True), (520, 33333, "bf16", False), (1030, 2500, "f32", False),
                                           (520, 6000, "bf16", False), (515, 8101, "bf16", True), (513, 9999, "f16", False), (513, 2900, "f32", True), (600, 4090, "f32", False),
                                           (530, 5100, "f32", True), (515, 9001, "f32", False)])
def test_policy_loss_of_many_long_rows(B, A, dtype, ref):
    """rows of several batches, enough of them to fill the card; the 64-bit loss on the GPU for its time"""
    g = torch.Generator(device="cuda").manual_seed(A)
    x = (3 * torch.randn((B, A), generator=g, device="cuda")).to(DTYPES[dtype])
    r = (x.float() + 0.5 * torch.randn((B, A), generator=g, device="cuda")).to(x.dtype) if ref else None
    actions = torch.randint(0, A, (B,), generator=g, device="cuda")
    actions[:4] = torch.tensor([0, 1, A - 2, A - 1])
    step = 0.15 * torch.randn(B, generator=g, device="cuda").double()
    for border in (np.log(0.8), np.log(1.2)):
        step = torch.where((step - border).abs() < 1e-3, step + 4e-3, step)
    old, adv = (pick(Rows64(x).logp, actions) - step).float(), torch.randn(B, generator=g, device="cuda")
    valid = torch.rand(B, generator=g, device="cuda") < 0.9
    want = [v.cpu() for v in policy_64(x, actions, old, adv, 0.2, 0.2, 0.3 if ref else 0.0, 0.02, valid, r)]
    wide = torch.full((B, A + 5), float("nan"), dtype=x.dtype, device="cuda")
    wide[:, 2:2 + A] = x
    t = wide[:, 2:2 + A].requires_grad_()
    out = ops().policy_loss(t, actions, old, adv, kl_coef=0.3 if ref else 0.0, ref_logits=r, entropy_coef=0.02, valid=valid)
    check(out.loss, want[0], want[1], "loss")
    check(out.stats, want[2], want[3], "stats")
    (d,) = torch.autograd.grad(out.loss, t, retain_graph=True)
    check(d, want[4], want[5] + rounding(want[4], x.dtype), "gradient")
    (d,) = torch.autograd.grad(out.loss * 4, t)
    check(d, want[4] * 4, want[5] * 4 + rounding(want[4] * 4, x.dtype), "gradient of 4 times the loss")


@pytest.mark.parametrize("A", [6, 300])
def test_policy_loss_where_little_is_left(A):
    g, x, actions, old, adv = policy_inputs(12, A, "f32", 3)
    x[2] = float("-inf")  # an empty row counts, with nothing to add
    x[3, 1:] = float("-inf")
    actions[3] = 0
    old[3] = 0.0
    want = policy_64(x, actions, old, adv, 0.2, 0.2, 0.0, 0.5)
    t = x.cuda().requires_grad_()
    args = actions.cuda(), old.cuda(), adv.cuda()
    out = ops().policy_loss(t, *args, entropy_coef=0.5)
    check(out.loss, want[0], want[1], "loss")
    check(out.stats, want[2], want[3], "stats")
    (d,) = torch.autograd.grad(out.loss, t)
    check(d, want[4], want[5] + rounding(want[4], torch.float32), "gradient")
    # no valid row at all: nothing is looked at
    t = torch.full((12, A), float("nan"), device="cuda", requires_grad=True)
    nan = torch.full((12,), float("nan"), device="cuda")
    out = ops().policy_loss(t, args[0] * 0 - 1, nan, nan, valid=torch.zeros(12, dtype=torch.bool, device="cuda"), ref_logprobs=nan, kl_coef=1.0, entropy_coef=1.0)
    (d,) = torch.autograd.grad(out.loss, t)
    assert out.loss.item() == 0 and (out.stats == 0).all() and (d == 0).all()
    # an action outside the columns: NaN for the loss and for its row, not for the others
    t = x.cuda().requires_grad_()
    bad = actions.clone()
    bad[5] = A
    out = ops().policy_loss(t, bad.cuda(), *args[1:], entropy_coef=0.5)
    (d,) = torch.autograd.grad(out.loss, t)
    assert out.loss.isnan() and d[5].isnan().all() and d[[0, 1, 2, 3, 4, 6, 7, 8, 9, 10, 11]].isfinite().all()


def test_policy_loss_gradient_agrees_with_differences():
    """second-order error of the central difference from the 64-bit loss's own third difference; the two losses are off by their tolerances"""
    B, A, s = 16, 15, 2.0 ** -6
    g, x, actions, old, adv = policy_inputs(B, A, "f32", 11)
    old = old - 0.05  # no row crosses a border of the clip range on the way
    way = rand((B, A), g, scale=0.02)
    ref = x + rand((B, A), g, scale=0.5)
    kw = dict(kl_coef=0.3, entropy_coef=0.1, ref_logits=ref.cuda())

    def at(k):
        moved = x + k * way
        loss = ops().policy_loss(moved.cuda(), actions.cuda(), old.cuda(), adv.cuda(), **kw).loss
        want = policy_64(moved, actions, old, adv, 0.2, 0.2, 0.3, 0.1, None, ref)
        return loss.item(), float(want[1]), float(want[0])

    t = x.cuda().requires_grad_()
    (d,) = torch.autograd.grad(ops().policy_loss(t, actions.cuda(), old.cuda(), adv.cuda(), **kw).loss, t)
    slope = float((d.double().cpu() * way.double()).sum())
    hi, lo, hi2, lo2 = at(s), at(-s), at(2 * s), at(-2 * s)
    third = (hi2[2] - 2 * hi[2] + 2 * lo[2] - lo2[2]) / (2 * s ** 3)
    slack = 2 * abs(third) * s * s / 6 + (hi[1] + lo[1]) / (2 * s) + 4 * U * float((x.abs() * d.abs().cpu()).sum()) / s + 1e-6
    assert abs((hi[0] - lo[0]) / (2 * s) - slope) <= slack
    assert slack < 0.2 * abs(slope) + 1e-3


# ---- streams, graphs, many at once ---------------------------------------------------------------------------------------------------------------


def window_step(x, w):
    """a run of all of them, as an update of a recurrent policy makes it; returns outputs and gradients"""
    o = ops()
    adv, ret = o.advantages(x["rew"], x["values"], x["first"], gamma=0.999, lam=0.95)
    h, last = o.gated_recurrence(x["gate"], x["update"], x["first"][:-1], x["state"])
    logits = h @ w
    logp, entropy = o.action_logprobs(logits, x["actions"])
    out = o.policy_loss(logits, x["actions"], x["old"], adv, entropy_coef=0.01, valid=x["valid"], ref_logprobs=x["ref"], kl_coef=0.1)
    d = torch.autograd.grad([out.loss, entropy], [x["gate"], x["update"], x["state"], w], [torch.ones_like(out.loss), torch.full_like(entropy, 1e-4)])
    return (adv, ret, h.detach(), last.detach(), logp.detach(), out.loss.detach(), out.stats, *d)


def window_inputs(T, N, D, A, seed):
    g = gen(seed)
    x = {"rew": torch.rand((T, N), generator=g), "values": rand((T + 1, N), g), "first": (torch.rand((T + 1, N), generator=g) < 0.05).to(torch.uint8),
         "gate": torch.sigmoid(rand((T, N, D), g, shift=1.0)), "update": rand((T, N, D), g), "state": rand((N, D), g), "actions": torch.randint(0, A, (T, N), generator=g, dtype=torch.int32),
         "old": rand((T, N), g, scale=0.1, shift=-2.7), "ref": rand((T, N), g, scale=0.1, shift=-2.7), "valid": torch.rand((T, N), generator=g) < 0.9}
    x = {k: v.cuda() for k, v in x.items()}
    for k in ("gate", "update", "state"):
        x[k].requires_grad_()
    return x, rand((D, A), g, scale=0.3).cuda().requires_grad_()


def window_64(x, w):
    """the same update in 64 bits on the CPU, differentiated by torch"""
    x = {k: v.detach().cpu() for k, v in x.items()}
    gate, update, state, w = (v.detach().cpu().double().requires_grad_() for v in (x["gate"], x["update"], x["state"], w))
    adv, _, ret, _ = advantages_64(x["rew"], x["values"], x["first"], 0.999, 0.95)
    h, hs = state, []
    for t in range(gate.shape[0]):
        h = torch.where(x["first"][t].bool()[:, None], update[t], gate[t] * h + update[t])
        hs.append(h)
    hs = torch.stack(hs)
    dist = torch.log_softmax(hs @ w, -1)
    logp, entropy = dist.gather(-1, x["actions"].long()[..., None])[..., 0], -(dist.exp() * dist).sum(-1)
    ratio = (logp - x["old"].double()).exp()
    z = x["ref"].double() - logp
    row = -torch.minimum(ratio * adv, ratio.clamp(0.8, 1.2) * adv) + 0.1 * (z.exp() - z - 1) - 0.01 * entropy
    loss = row[x["valid"]].mean()
    d = torch.autograd.grad(loss + 1e-4 * entropy.sum(), [gate, update, state, w])
    return (adv, ret, hs.detach(), h.detach(), logp.detach(), loss.detach(), None, *d)


@pytest.mark.parametrize("T,N,D,A", [(20, 6, 32, 15), (130, 3, 16, 40)])
def test_a_window_with_all_operators(T, N, D, A):
    x, w = window_inputs(T, N, D, A, T)
    got, want = window_step(x, w), window_64(x, w)
    names = ("adv", "ret", "h", "state", "logp", "loss", "stats", "d_gate", "d_update", "d_state", "d_w")
    for name, a, b in zip(names, got, want):
        if b is None:
            continue
        # sums of up to T N A products in 32 bits, relative to the size of the whole result (the element-wise bounds are the other tests' matter)
        off = float((a.double().cpu() - b).norm() / b.norm())
        assert off < 64 * U * np.sqrt(T * N), (name, off)


def test_streams_and_captured_graphs():
    """two graphs that are captured one after the other and replayed in turn, with eager work and synchronizations between; every replay equals the eager
    result bit for bit.  And a pass on another stream while this one works."""
    sets = [window_inputs(40, 5, 16, 15, 100), window_inputs(70, 4, 24, 33, 200)]
    eager = [window_step(*s) for s in sets]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = window_step(*sets[0])
    here = window_step(*sets[1])
    side.synchronize()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, eager[0])) and all(torch.equal(a, b) for a, b in zip(here, eager[1]))
    del other, here
    graphs, outs = [], []
    for s in sets:
        with torch.cuda.stream(side):  # as the capture needs it: warmed up on its stream
            window_step(*s)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(window_step(*s))
        graphs.append(graph)
    for k in range(4):
        for graph, out, want in zip(graphs, outs, eager):
            for v in out:
                v.zero_()
            graph.replay()
            noise = ops().action_logprobs(torch.randn(100, 15, device="cuda"), torch.zeros(100, dtype=torch.int32, device="cuda"))
            torch.cuda.synchronize()
            for i, (a, b) in enumerate(zip(out, want)):
                assert torch.equal(a, b), (k, i)
            assert noise[0].isfinite().all()


def test_single_steps_in_a_captured_graph_move_the_state_on():
    N, D, A = 64, 32, 15
    g = gen(6)
    gate, update, state, w = torch.rand((1, N, D), generator=g).cuda(), rand((1, N, D), g).cuda(), rand((N, D), g).cuda(), rand((D, A), g).cuda()
    first, actions = torch.zeros((1, N), dtype=torch.uint8, device="cuda"), torch.zeros((1, N), dtype=torch.int32, device="cuda")

    def act(state):
        with torch.no_grad():
            h, _ = ops().gated_recurrence(gate, update, first, state, state_out=state)
            return ops().action_logprobs(h @ w, actions)

    eager_state, graph_state = state.clone(), state.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        act(state.clone())
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        logp, entropy = act(graph_state)
    graph_state.copy_(state)
    for k in range(5):
        first.fill_(1 if k == 3 else 0)
        want = act(eager_state)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(graph_state, eager_state) and torch.equal(logp, want[0]) and torch.equal(entropy, want[1]), k


def test_forward_and_backward_in_graphs_of_their_own():
    """as torch.cuda.make_graphed_callables captures them: the backward graph cannot know what the forward one wrote, and serves every scale"""
    g, x, actions, old, adv = policy_inputs(300, 15, "f32", 21)
    args = actions.cuda(), old.cuda(), adv.cuda()

    class Loss(torch.nn.Module):
        def forward(self, logits):
            return ops().policy_loss(logits, *args, entropy_coef=0.05).loss

    graphed = torch.cuda.make_graphed_callables(Loss(), (torch.zeros((300, 15), device="cuda", requires_grad=True),))
    for k, scale in enumerate((3.0, 1.0, 0.5, 1.0)):
        values = x + 0.01 * k
        t = values.cuda().requires_grad_()
        (d,) = torch.autograd.grad(graphed(t) * scale, t)
        torch.cuda.synchronize()
        u = values.cuda().requires_grad_()
        (e,) = torch.autograd.grad(Loss()(u) * scale, u)
        assert torch.equal(d, e), scale


def test_gradients_of_gradients_are_refused():
    x, w = window_inputs(8, 3, 4, 15, 7)
    logits = torch.zeros((8, 3, 15), device="cuda", requires_grad=True)
    h, _ = ops().gated_recurrence(x["gate"], x["update"], x["first"][:-1], x["state"])
    logp, _ = ops().action_logprobs(logits, x["actions"])
    for y, leaf in ((h.sum(), x["gate"]), (logp.sum(), logits), (ops().policy_loss(logits, x["actions"], x["old"], x["rew"]).loss, logits)):
        (d,) = torch.autograd.grad(y, leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="once"):
            d.sum().backward()


def test_two_host_threads_and_streams():
    """each with a stream of its own, the same work at the same time: the results are those of one after the other"""
    import threading

    sets = [window_inputs(60, 4, 16, 15, 300 + k) for k in range(3)]
    alone = [window_step(*s) for s in sets]
    torch.cuda.synchronize()
    got, errors = [None] * 3, []

    def work(k):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(5):
                    got[k] = window_step(*sets[k])
            stream.synchronize()
        except Exception as e:  # handed to the test's own thread
            errors.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for a, b in zip(got, alone):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_repeated_calls_give_the_same_bits():
    x, w = window_inputs(200, 9, 8, 15, 1)
    a, b = window_step(x, w), window_step(x, w)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


# ---- next to the environments --------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("names,devices", [("coinrun", 1), ("bigfish,maze", 1)])
def test_rollout_of_a_handle_feeds_the_operators(names, devices):
    """torch_view.Rollout collects what env.observe() returned, and its advantages are those of the collected window"""
    from procgen_amd import ProcgenGym3Env, torch_view

    n, T = 32, 12
    env = ProcgenGym3Env(n, names, rand_seed=5, use_generated_assets=True)
    window = torch_view.Rollout(env, T)
    rng = np.random.RandomState(0)
    rew, _, first = env.observe()
    window.record()
    with pytest.raises(ValueError):
        window.advantages(torch.zeros((T + 1, n), device="cuda"), gamma=0.9, lam=0.9)
    for part in range(2):  # a second window begins where the first one ended
        rews, firsts, acts = [], [np.array(first)], []
        for t in range(T):
            acts.append(rng.randint(0, 15, size=n).astype(np.int32))
            if t == 4:
                acts[-1][3] = -1  # a forced reset
            env.act(acts[-1])
            rew, _, first = env.observe()
            window.record()
            rews.append(np.array(rew)), firsts.append(np.array(first))
        assert firsts[5][3] == 1
        rews, firsts = torch.tensor(np.stack(rews)), torch.tensor(np.stack(firsts).astype(np.uint8))
        assert torch.equal(window.rew.cpu(), rews) and torch.equal(window.first.cpu(), firsts) and np.array_equal(window.action.cpu().numpy(), np.stack(acts))
        values = rand((T + 1, n), gen(part))
        adv, ret = window.advantages(values.cuda(), gamma=0.999, lam=0.95)
        want = advantages_64(rews, values, firsts, 0.999, 0.95)
        check(adv, want[0], want[1], "advantages")
        check(ret, want[2], want[3], "returns")
        valid = window.action >= 0  # a forced reset's action has no log-probability
        logits = rand((T, n, 15), gen(9 + part)).cuda().requires_grad_()
        logp, _ = ops().action_logprobs(logits.detach(), window.action)
        assert torch.equal(logp.isnan(), ~valid)
        out = ops().policy_loss(logits, window.action, logp, adv, valid=valid)
        (d,) = torch.autograd.grad(out.loss, logits)
        assert abs(out.loss.item() + adv[valid].double().mean().item()) < 1e-5 and d.isfinite().all() and (d[~valid] == 0).all()  # ratio 1: the loss is minus the mean advantage
        same = window.policy_loss(logits, logp, adv)
        assert torch.equal(same.loss, out.loss) and torch.equal(same.stats, out.stats) and torch.equal(window.action_logprobs(logits.detach())[0].nan_to_num(9.0), logp.nan_to_num(9.0))
        half = window.policy_loss(logits, logp, adv, valid=torch.arange(n, device="cuda").expand(T, n) % 2)
        assert abs(half.loss.item() + adv[:, 1::2][valid[:, 1::2]].double().mean().item()) < 1e-5
        gate, update = torch.rand((T, n, 8), generator=gen(part)).cuda(), rand((T, n, 8), gen(20 + part)).cuda()
        memory = torch.zeros((n, 8), device="cuda") if part == 0 else memory
        want = recurrence_64(gate.cpu(), update.cpu(), firsts[:-1], memory.cpu())
        h, memory = window.recurrence(gate, update, memory)
        check(h, want["h"], want["E_h"] + rounding(want["h"], torch.float32), "memory over the window")
        with pytest.raises(ValueError):
            window.record()
        window.restart()
    env.close()
