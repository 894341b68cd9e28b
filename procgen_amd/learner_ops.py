"""
Learner operators over a rollout: what a policy gradient needs of a window of T steps of N envs, computed on the GPU where torch_view's tensors
already are.  Entry points of libenv.so (include/procgen_amd_learner.h); hand-written kernels, no CPU path.

    views = torch_view.device_views(env)                         # rew, first, action of every step, on the GPU
    h, memory = gated_recurrence(gate, update, first, memory)    # the policy's memory over the window, cut where an episode begins
    logp, entropy = action_logprobs(logits, actions)             # what the rollout stores about its own actions
    adv, ret = advantages(rew, values, first, gamma=0.999, lam=0.95)
    out = policy_loss(logits, actions, logp, adv, entropy_coef=0.01)
    out.loss.backward()

Every operator runs on the current stream of its tensors' device, does not synchronise, keeps nothing between calls and can be captured into a graph.
Tensors may be strided (batch-major windows, slices, expanded dimensions); arguments that an operator does not take raise TypeError or ValueError
before anything runs.  Element types: float32, float16, bfloat16; sums, states and statistics are held in 32 bits or more.
"""
import ctypes as C
import os
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from .env import DEFAULT_LIB_DIR

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}  # enum procgen_amd_dtype


class _Array3(C.Structure):  # struct procgen_amd_array3
    _fields_ = [("data", C.c_void_p), ("t_stride", C.c_longlong), ("n_stride", C.c_longlong), ("d_stride", C.c_longlong)]


class _Recurrence(C.Structure):  # struct procgen_amd_recurrence
    _fields_ = [("dtype", C.c_int), ("T", C.c_int), ("N", C.c_int), ("D", C.c_int), ("gate", _Array3), ("update", _Array3), ("h", _Array3),
                ("first", C.c_void_p), ("first_t_stride", C.c_longlong), ("first_n_stride", C.c_longlong), ("state", C.c_void_p), ("state_out", C.c_void_p),
                ("checkpoints", C.c_void_p), ("workspace", C.c_void_p), ("d_h", _Array3), ("d_gate", _Array3), ("d_update", _Array3),
                ("d_state_out", C.c_void_p), ("d_state", C.c_void_p)]


class _Advantage(C.Structure):  # struct procgen_amd_advantage
    _fields_ = [("dtype", C.c_int), ("T", C.c_int), ("N", C.c_int), ("rew", C.c_void_p), ("rew_t_stride", C.c_longlong), ("rew_n_stride", C.c_longlong),
                ("values", C.c_void_p), ("values_t_stride", C.c_longlong), ("values_n_stride", C.c_longlong),
                ("first", C.c_void_p), ("first_t_stride", C.c_longlong), ("first_n_stride", C.c_longlong), ("gamma", C.c_float), ("lam", C.c_float),
                ("adv", C.c_void_p), ("ret", C.c_void_p), ("workspace", C.c_void_p)]


class _Rows(C.Structure):  # struct procgen_amd_rows
    _fields_ = [("dtype", C.c_int), ("rows", C.c_longlong), ("columns", C.c_longlong), ("inner", C.c_longlong), ("logits", C.c_void_p),
                ("outer_stride", C.c_longlong), ("inner_stride", C.c_longlong), ("actions", C.c_void_p), ("actions_are_64_bit", C.c_int),
                ("d_logits", C.c_void_p), ("workspace", C.c_void_p)]


class _Policy(C.Structure):  # struct procgen_amd_policy
    _fields_ = [("old_logprobs", C.c_void_p), ("adv", C.c_void_p), ("valid", C.c_void_p), ("ref_logits", C.c_void_p), ("ref_outer_stride", C.c_longlong),
                ("ref_inner_stride", C.c_longlong), ("ref_logprobs", C.c_void_p), ("clip_low", C.c_float), ("clip_high", C.c_float), ("kl_coef", C.c_float),
                ("entropy_coef", C.c_float), ("scale", C.c_void_p), ("loss", C.c_void_p), ("stats", C.c_void_p), ("resume", C.c_int)]


class _Library:
    """the entry points, loaded when an operator first runs"""

    def __init__(self):
        self.lib = None

    def __getattr__(self, name):
        if self.lib is None:
            lib = C.CDLL(os.path.join(DEFAULT_LIB_DIR, "libenv.so"))
            P, I, L = C.c_void_p, C.c_int, C.c_longlong
            for fn, res, args in (("recurrence_checkpoints", L, [I]), ("recurrence_workspace", L, [I, I, I]), ("recurrence_forward", I, [P, I, P]),
                                  ("recurrence_backward", I, [P, I, P]), ("advantages", I, [P, I, P]), ("rows_workspace", L, [L, L]),
                                  ("action_logprobs", I, [P, P, P, P, I, P]), ("action_logprobs_backward", I, [P, P, P, P, P, I, P]), ("policy_loss", I, [P, P, I, P]), ("capture_id", L, [P])):
                f = getattr(lib, "procgen_amd_" + fn)
                f.restype, f.argtypes = res, args
                setattr(self, fn, f)
            self.lib = lib
            return getattr(self, name)
        raise AttributeError(name)


_lib = _Library()


def _run(fn, name, device, *args):
    rc = fn(*args, device.index, torch.cuda.current_stream(device).cuda_stream)
    if rc:
        raise RuntimeError(f"{name}: " + ("the library refused the arguments" if rc < 0 else f"HIP error {rc}"))


def _need(ok, message, kind=ValueError):
    if not ok:
        raise kind(message)


def _tensor(x, what, dtypes, shape=None):
    _need(isinstance(x, torch.Tensor), f"{what} has to be a tensor", TypeError)
    _need(x.dtype in dtypes, f"{what} has to be {' or '.join(str(d).replace('torch.', '') for d in dtypes)}, not {x.dtype}", TypeError)
    _need(shape is None or tuple(x.shape) == tuple(shape), f"{what} has to have the shape {tuple(shape) if shape is not None else ''}, not {tuple(x.shape)}")


def _on_gpu(*tensors):
    """the one device all of them are on"""
    device = tensors[0].device
    _need(device.type == "cuda", f"the learner operators run on the GPU only: a tensor is on {device}")
    for x in tensors:
        _need(x is None or x.device == device, f"the tensors are on different devices ({device} and {x.device if x is not None else ''})")
    return device


def _constant(x, what):
    _need(x is None or not (x.requires_grad and torch.is_grad_enabled()), f"{what} is a constant to this operator and gets no gradient: detach it")


def _number(x, what, low=float("-inf"), high=float("inf")):
    _need(isinstance(x, (int, float)) and not isinstance(x, bool), f"{what} has to be a number", TypeError)
    _need(low <= x <= high, f"{what} has to lie in [{low}, {high}], not {x}")


_FLAGS = (torch.uint8, torch.bool)
_F32 = (torch.float32,)


def _array3(x):
    return _Array3(x.data_ptr(), *x.stride())


def _bytes(n, device):
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


def _ptr(x):
    return None if x is None else x.data_ptr()


# ---- the memory of a policy ------------------------------------------------------------------------------------------------------------------


def _recurrence_args(gate, update, first, state, checkpoints):
    T, N, D = gate.shape
    a = _Recurrence(dtype=_DTYPES[gate.dtype], T=T, N=N, D=D, gate=_array3(gate), update=_array3(update), state=_ptr(state), checkpoints=_ptr(checkpoints))
    if first is not None:
        a.first, a.first_t_stride, a.first_n_stride = first.data_ptr(), first.stride(0), first.stride(1)
    work = _bytes(_lib.recurrence_workspace(T, N, D), gate.device)
    a.workspace = _ptr(work)
    return a, work


def _recurrence_forward(gate, update, first, state, state_out, checkpoints=None):
    h = torch.empty_like(update)
    last = state_out if state_out is not None else torch.empty(gate.shape[1:], dtype=torch.float32, device=gate.device)
    a, work = _recurrence_args(gate, update, first, state, checkpoints)
    a.h, a.state_out = _array3(h), last.data_ptr()
    _run(_lib.recurrence_forward, "gated_recurrence", gate.device, C.addressof(a))
    return h, last


class _GatedRecurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, update, first, state):
        checkpoints = torch.empty((_lib.recurrence_checkpoints(gate.shape[0]), *gate.shape[1:]), dtype=torch.float32, device=gate.device)
        h, last = _recurrence_forward(gate, update, first, state, None, checkpoints)
        ctx.save_for_backward(gate, update, first, state, checkpoints)
        return h, last

    @staticmethod
    @once_differentiable
    def backward(ctx, d_h, d_last):
        gate, update, first, state, checkpoints = ctx.saved_tensors
        a, work = _recurrence_args(gate, update, first, state, checkpoints)
        d_gate = d_update = d_state = None
        if d_h is not None:
            a.d_h = _array3(d_h)
        if d_last is not None:
            d_last = d_last.contiguous()
            a.d_state_out = d_last.data_ptr()
        if ctx.needs_input_grad[0]:
            d_gate = torch.empty_like(gate)
            a.d_gate = _array3(d_gate)
        if ctx.needs_input_grad[1]:
            d_update = torch.empty_like(update)
            a.d_update = _array3(d_update)
        if ctx.needs_input_grad[3]:
            d_state = torch.empty_like(state)
            a.d_state = d_state.data_ptr()
        _run(_lib.recurrence_backward, "gated_recurrence", gate.device, C.addressof(a))
        return d_gate, d_update, None, d_state


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in tensors)


def gated_recurrence(gate, update, first=None, state=None, state_out=None):
    """h[t] = gate[t] * h[t-1] + update[t] along the steps of a window, each env and channel a chain of its own; where first[t] is set an episode
    begins and h[t] = update[t].  Returns (h, state): h [T, N, D] in the inputs' type, and the state behind the last step, float32 [N, D], to begin the
    next window or the next single step (T = 1) with.

    gate, update: [T, N, D] (or [T, N]) float32, float16 or bfloat16, any strides; first: [T, N] uint8 or bool, None: no episode begins; state:
    float32 [N, D] (or [N]), None: zeros.  state_out: a float32 buffer that takes the new state, `state` itself to move it on in place; only without
    gradients.  Differentiable in gate, update and state, once."""
    _tensor(gate, "gate", tuple(_DTYPES))
    _need(gate.dim() in (2, 3), f"gate has to be [T, N, D] or [T, N], not {tuple(gate.shape)}")
    _tensor(update, "update", (gate.dtype,), gate.shape)
    lead, per_env = gate.shape[:2], gate.shape[1:]
    if first is not None:
        _tensor(first, "first", _FLAGS, lead)
    if state is not None:
        _tensor(state, "state", _F32, per_env)
    if state_out is not None:
        _tensor(state_out, "state_out", _F32, per_env)
        _need(state_out.is_contiguous(), "state_out has to be contiguous")
        _need(not _wants_grad(gate, update, state, state_out),
              "state_out overwrites a state: call under torch.no_grad(), or take the returned state")
    _on_gpu(gate, update, first, state, state_out)
    flat = gate.dim() == 2
    if flat:
        gate, update = gate.unsqueeze(2), update.unsqueeze(2)
        state = state.unsqueeze(1) if state is not None else None
        state_out = state_out.unsqueeze(1) if state_out is not None else None
    if state is not None:
        state = state.contiguous()
    if gate.numel() == 0:  # no step or no chain: the state stays
        h = (update + gate) * 1
        last = state * 1 if state is not None else torch.zeros(gate.shape[1:], dtype=torch.float32, device=gate.device)
        if state_out is not None:
            last = state_out.copy_(last)
    elif _wants_grad(gate, update, state):
        h, last = _GatedRecurrence.apply(gate, update, first, state)
    else:
        h, last = _recurrence_forward(gate, update, first, state, state_out)
    return (h.squeeze(2), last.squeeze(1)) if flat else (h, last)


# ---- advantages ------------------------------------------------------------------------------------------------------------------------------


def advantages(rew, values, first, *, gamma, lam):
    """Generalized advantages and returns of a window, float32 [T, N] each:
    delta[t] = rew[t] + gamma * v[t+1] - v[t], adv[t] = delta[t] + gamma * lam * adv[t+1], ret = adv + v, where v[t+1] and adv[t+1] count as zero
    where first[t+1] is set: the episode of step t ended with it.

    rew: float32 [T, N], rew[t] earned by the action of step t; values: [T + 1, N] float32, float16 or bfloat16, the last row the value of the
    observation behind the window; first: [T + 1, N] uint8 or bool (torch_view's `first` of the observations 0 .. T).  Targets are constants of the
    losses made from them: no gradient."""
    _tensor(rew, "rew", _F32)
    _need(rew.dim() == 2, f"rew has to be [T, N], not {tuple(rew.shape)}")
    T, N = rew.shape
    _tensor(values, "values", tuple(_DTYPES), (T + 1, N))
    _tensor(first, "first", _FLAGS, (T + 1, N))
    _number(gamma, "gamma", 0.0, 1.0)
    _number(lam, "lam", 0.0, 1.0)
    _constant(rew, "rew")
    _constant(values, "values")
    device = _on_gpu(rew, values, first)
    adv = torch.empty((T, N), dtype=torch.float32, device=device)
    ret = torch.empty((T, N), dtype=torch.float32, device=device)
    if T and N:
        a = _Advantage(_DTYPES[values.dtype], T, N, rew.data_ptr(), *rew.stride(), values.data_ptr(), *values.stride(), first.data_ptr(), *first.stride(),
                       gamma, lam, adv.data_ptr(), ret.data_ptr(), None)
        work = _bytes(_lib.recurrence_workspace(T, N, 1), device)
        a.workspace = _ptr(work)
        _run(_lib.advantages, "advantages", device, C.addressof(a))
    return adv, ret


# ---- rows of logits --------------------------------------------------------------------------------------------------------------------------


def _layout(x, what):
    """(inner, outer stride, inner stride) of the rows of x [..., columns]: the leading dimensions as at most two strided ones"""
    dims = []
    for size, stride in zip(x.shape[:-1], x.stride()[:-1]):
        if size == 1:
            continue
        if dims and dims[-1][1] == stride * size:
            dims[-1] = (dims[-1][0] * size, stride)
        else:
            dims.append((size, stride))
    _need(x.shape[-1] == 1 or x.stride(-1) == 1, f"the columns of {what} have to be contiguous")
    _need(len(dims) <= 2, f"the leading dimensions of {what} are strided in more than two ways: make it contiguous")
    if len(dims) == 2:
        return dims[1][0], dims[0][1], dims[1][1]
    return 1, dims[0][1] if dims else 0, 0


def _rows(logits, actions):
    inner, outer_stride, inner_stride = _layout(logits, "logits")
    columns = logits.shape[-1]
    return _Rows(_DTYPES[logits.dtype], logits.numel() // columns, columns, max(1, inner), logits.data_ptr(), outer_stride, inner_stride, actions.data_ptr(), actions.dtype == torch.int64)


def _check_rows(logits, actions):
    _tensor(logits, "logits", tuple(_DTYPES))
    _need(logits.dim() >= 1 and logits.shape[-1] >= 1, "logits have to be [..., columns] with one column at least")
    _tensor(actions, "actions", (torch.int32, torch.int64), logits.shape[:-1])


def _action_logprobs(logits, actions, grad):
    device = logits.device
    logp, entropy = (torch.empty(logits.shape[:-1], dtype=torch.float32, device=device) for _ in range(2))
    lse = torch.empty_like(logp) if grad else None
    a = _rows(logits, actions)
    work = _bytes(_lib.rows_workspace(a.rows, a.columns), device)
    a.workspace = work.data_ptr()
    _run(_lib.action_logprobs, "action_logprobs", device, C.addressof(a), logp.data_ptr(), entropy.data_ptr(), _ptr(lse))
    return logp, entropy, lse


class _ActionLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, actions):
        logp, entropy, lse = _action_logprobs(logits, actions, True)
        ctx.save_for_backward(logits, actions, lse, entropy)
        return logp, entropy

    @staticmethod
    @once_differentiable
    def backward(ctx, d_logp, d_entropy):
        logits, actions, lse, entropy = ctx.saved_tensors
        d_logits = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        a = _rows(logits, actions)
        a.d_logits = d_logits.data_ptr()
        d_logp, d_entropy = (None if x is None else x.contiguous() for x in (d_logp, d_entropy))
        _run(_lib.action_logprobs_backward, "action_logprobs", logits.device, C.addressof(a), lse.data_ptr(), entropy.data_ptr(), _ptr(d_logp), _ptr(d_entropy))
        return d_logits, None


def action_logprobs(logits, actions):
    """(logp, entropy), float32 [...]: the log-probability of actions[...] under softmax(logits[..., :]) and the entropy of that distribution.

    logits: [..., columns] float32, float16 or bfloat16, columns contiguous; actions: [...] int32 or int64.  A column of -inf is an action that
    cannot be taken; a row of nothing else has log-probability -inf, entropy 0 and a zero gradient.  An action outside [0, columns) -- the -1 of a forced
    reset -- has no log-probability: NaN, and a NaN gradient unless its gradients coming in are zero.  Differentiable in logits, once."""
    _check_rows(logits, actions)
    _on_gpu(logits, actions)
    _layout(logits, "logits")
    if logits.numel() == 0:
        empty = logits.sum(-1, dtype=torch.float32)
        return empty, empty * 1
    actions = actions.contiguous()
    if _wants_grad(logits):
        return _ActionLogprobs.apply(logits, actions)
    return _action_logprobs(logits, actions, False)[:2]


class PolicyLoss(NamedTuple):
    loss: torch.Tensor   # float32, differentiable in the logits
    stats: torch.Tensor  # float32 [4]: the means of -objective, KL, entropy and of (ratio outside the clip range), constants


def _policy_args(coefs, work, logits, actions, old, adv, valid, ref_logits, ref_logprobs):
    a = _rows(logits, actions)
    a.workspace = work.data_ptr()
    clip, kl_coef, entropy_coef = coefs
    q = _Policy(old.data_ptr(), adv.data_ptr(), _ptr(valid), _ptr(ref_logits), 0, 0, _ptr(ref_logprobs), *clip, kl_coef, entropy_coef)
    if ref_logits is not None:
        (a.inner, a.outer_stride, a.inner_stride), (_, q.ref_outer_stride, q.ref_inner_stride) = _common_layout(logits, ref_logits)
    return a, q


def _policy_forward(coefs, d_logits, *tensors):
    logits = tensors[0]
    device, columns = logits.device, logits.shape[-1]
    loss, stats = torch.empty((), dtype=torch.float32, device=device), torch.empty(4, dtype=torch.float32, device=device)
    work = _bytes(_lib.rows_workspace(logits.numel() // columns, columns), device)
    a, q = _policy_args(coefs, work, *tensors)
    a.d_logits, q.loss, q.stats = _ptr(d_logits), loss.data_ptr(), stats.data_ptr()
    _run(_lib.policy_loss, "policy_loss", device, C.addressof(a), C.addressof(q))
    return loss, stats, work


def _capture(device):
    return _lib.capture_id(torch.cuda.current_stream(device).cuda_stream)


class _PolicyLoss(torch.autograd.Function):
    """The forward call writes the gradient too, from the row that it has in registers.  The first backward pass hands it out, after a kernel that goes
    over the rows again only where the loss's own gradient is not 1; each further one (retain_graph)
    computes its own, and so does a backward pass that is captured apart from its forward call."""

    @staticmethod
    def forward(ctx, coefs, *tensors):
        logits = tensors[0]
        d_logits = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        loss, stats, ctx.work = _policy_forward(coefs, d_logits, *tensors)
        ctx.coefs, ctx.d_logits, ctx.capture = coefs, d_logits, _capture(logits.device)
        ctx.save_for_backward(*tensors)
        ctx.mark_non_differentiable(stats)
        return loss, stats

    @staticmethod
    @once_differentiable
    def backward(ctx, d_loss, _):
        logits = ctx.saved_tensors[0]
        d_logits, ctx.d_logits = ctx.d_logits, None
        a, q = _policy_args(ctx.coefs, ctx.work, *ctx.saved_tensors)
        q.resume = 1
        if d_logits is not None and ctx.capture == _capture(logits.device) >= 0:
            q.resume = 3
        else:
            d_logits = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        a.d_logits, q.scale = d_logits.data_ptr(), d_loss.data_ptr()
        _run(_lib.policy_loss, "policy_loss", logits.device, C.addressof(a), C.addressof(q))
        return (None, d_logits) + (None,) * 6


def _common_layout(x, y):
    """the rows of two equally shaped tensors under one split of their leading dimensions, or ValueError"""
    lead = x.shape[:-1]
    for k in range(len(lead) + 1):
        got = []
        for z in (x, y):
            parts = []
            for lo, hi in ((0, k), (k, len(lead))):
                dims = [(n, s) for n, s in zip(lead[lo:hi], z.stride()[lo:hi]) if n != 1]
                if any(dims[i][1] != dims[i + 1][0] * dims[i + 1][1] for i in range(len(dims) - 1)):
                    break
                parts.append(dims[-1][1] if dims else 0)
            if len(parts) == 2:
                inner = 1
                for n in lead[k:]:
                    inner *= n
                got.append((max(1, inner), *parts))
        if len(got) == 2:
            return got
    raise ValueError("logits and ref_logits are strided in too different ways: make them contiguous")


def policy_loss(logits, actions, old_logprobs, advantages, *, clip=0.2, kl_coef=0.0, ref_logits=None, ref_logprobs=None, entropy_coef=0.0, valid=None):
    """The clipped policy loss with a KL term over rows of logits, as PolicyLoss(loss, stats):
    ratio = exp(logp - old_logprobs), objective = min(ratio * adv, clip(ratio, 1 - clip, 1 + clip) * adv),
    loss = mean over the valid rows of -objective + kl_coef * KL - entropy_coef * entropy.

    KL is KL(p | q) over all columns with q = softmax(ref_logits), or its estimator exp(d) - d - 1 with d = ref_logprobs - logp from the reference's
    log-probability of the action taken; at most one of the two is given, and the term is 0 without.  clip: a number, or (below, above).  logits as for
    action_logprobs; actions, old_logprobs, advantages, valid (uint8 or bool, None: all), ref_logprobs: [...]; ref_logits like logits.  Rows that are
    not valid are not looked at, whatever they hold, and get a zero gradient; without a valid row the loss is 0.  A valid row without any finite
    column counts, with nothing to add.  Only the logits get a gradient, once."""
    _check_rows(logits, actions)
    lead = logits.shape[:-1]
    for x, what in ((old_logprobs, "old_logprobs"), (advantages, "advantages"), (ref_logprobs, "ref_logprobs")):
        if x is not None or what != "ref_logprobs":
            _tensor(x, what, _F32, lead)
        _constant(x, what)
    if valid is not None:
        _tensor(valid, "valid", _FLAGS, lead)
    if ref_logits is not None:
        _tensor(ref_logits, "ref_logits", (logits.dtype,), logits.shape)
        _constant(ref_logits, "ref_logits")
        _need(ref_logprobs is None, "ref_logits or ref_logprobs, not both")
    low, high = clip if isinstance(clip, (tuple, list)) and len(clip) == 2 else (clip, clip)
    _number(low, "clip", 0.0, 1.0)
    _number(high, "clip", 0.0)
    _number(kl_coef, "kl_coef", 0.0)
    _number(entropy_coef, "entropy_coef")
    _need(kl_coef == 0.0 or ref_logits is not None or ref_logprobs is not None, "kl_coef without ref_logits or ref_logprobs")
    _on_gpu(logits, actions, old_logprobs, advantages, valid, ref_logits, ref_logprobs)
    _layout(logits, "logits")
    if ref_logits is not None:
        _layout(ref_logits, "ref_logits")
        _common_layout(logits, ref_logits)
    actions, old_logprobs, advantages, valid, ref_logprobs = (None if x is None else x.contiguous() for x in (actions, old_logprobs, advantages, valid, ref_logprobs))
    coefs = (float(low), float(high)), float(kl_coef), float(entropy_coef)
    tensors = logits, actions, old_logprobs, advantages, valid, ref_logits, ref_logprobs
    return PolicyLoss(*(_PolicyLoss.apply(coefs, *tensors) if _wants_grad(logits) else _policy_forward(coefs, None, *tensors)[:2]))
