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
import functools
import os
import struct
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from .env import DEFAULT_LIB_DIR

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}  # enum procgen_amd_dtype

# the C structs, packed field by field (native sizes and alignment; the closing 0P pads the end): a third of the time that filling a ctypes.Structure takes
_ARRAY3 = "Pqqq"  # struct procgen_amd_array3: data, t_stride, n_stride, d_stride
_RECURRENCE = struct.Struct("@4i" + 3 * _ARRAY3 + "Pqq4P" + 3 * _ARRAY3 + "2P" + "0P")
_ADVANTAGE = struct.Struct("@3iPqqPqqPqqff3P" + "0P")
_ROWS = struct.Struct("@iqqqPqqPiPP" + "0P")
_POLICY = struct.Struct("@4PqqP4f3Pi" + "0P")
_NO_ARRAY = (0, 0, 0, 0)


class _Library:
    """the entry points, loaded when an operator first runs"""

    def __init__(self):
        self.lib = None

    def __getattr__(self, name):
        if self.lib is None:
            lib = C.CDLL(os.path.join(DEFAULT_LIB_DIR, "libenv.so"))
            P, I, L = C.c_void_p, C.c_int, C.c_longlong
            S = C.c_char_p  # a packed struct
            for fn, res, args in (("recurrence_checkpoints", L, [I]), ("recurrence_workspace", L, [I, I, I]), ("recurrence_forward", I, [S, I, P]),
                                  ("recurrence_backward", I, [S, I, P]), ("advantages", I, [S, I, P]), ("rows_workspace", L, [L, L]),
                                  ("action_logprobs", I, [S, P, P, P, I, P]), ("action_logprobs_backward", I, [S, P, P, P, P, I, P]), ("policy_loss", I, [S, S, I, P]),
                                  ("capture_id", L, [P])):
                f = getattr(lib, "procgen_amd_" + fn)
                f.restype, f.argtypes = res, args
                setattr(self, fn, f)
            self.lib = lib
            return getattr(self, name)
        raise AttributeError(name)


_lib = _Library()
_stream = torch._C._cuda_getCurrentRawStream  # torch.cuda.current_stream(device).cuda_stream without the Stream object


@functools.lru_cache(maxsize=1024)
def _checkpoints(T):
    return _lib.recurrence_checkpoints(T)


@functools.lru_cache(maxsize=1024)
def _recurrence_workspace(T, N, D):
    return _lib.recurrence_workspace(T, N, D)


@functools.lru_cache(maxsize=1024)
def _rows_workspace(rows, columns):
    return _lib.rows_workspace(rows, columns)


def _run(fn, name, index, *args):
    rc = fn(*args, index, _stream(index))
    if rc:
        raise RuntimeError(f"{name}: " + ("the library refused the arguments" if rc < 0 else f"HIP error {rc}"))


def _need(ok, message, kind=ValueError):
    if not ok:
        raise kind(message)


def _tensor(x, what, dtypes, shape=None):
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{what} has to be a tensor")
    if x.dtype not in dtypes:
        raise TypeError(f"{what} has to be {' or '.join(str(d).replace('torch.', '') for d in dtypes)}, not {x.dtype}")
    if shape is not None and x.shape != shape:
        raise ValueError(f"{what} has to have the shape {tuple(shape)}, not {tuple(x.shape)}")


def _on_gpu(x, *others):
    """the one device all of them are on"""
    device = x.device
    if device.type != "cuda":
        raise ValueError(f"the learner operators run on the GPU only: a tensor is on {device}")
    for y in others:
        if y is not None and y.device != device:
            raise ValueError(f"the tensors are on different devices ({device} and {y.device})")
    return device


def _constant(x, what):
    if x is not None and x.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what} is a constant to this operator and gets no gradient: detach it")


def _number(x, what, low=float("-inf"), high=float("inf")):
    if not isinstance(x, (int, float)) or isinstance(x, bool):
        raise TypeError(f"{what} has to be a number")
    if not low <= x <= high:
        raise ValueError(f"{what} has to lie in [{low}, {high}], not {x}")


_FLAGS = (torch.uint8, torch.bool)
_F32 = (torch.float32,)
_INTS = (torch.int32, torch.int64)
_FLOATS = tuple(_DTYPES)


def _wants_grad(*tensors):
    if torch.is_grad_enabled():
        for x in tensors:
            if x is not None and x.requires_grad:
                return True
    return False


def _array3(x):
    return (x.data_ptr(), *x.stride())


def _bytes(n, device):
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


def _ptr(x):
    return 0 if x is None else x.data_ptr()


# ---- the memory of a policy ------------------------------------------------------------------------------------------------------------------


def _recurrence_args(gate, update, h, first, state, state_out, checkpoints, work, backward=3 * _NO_ARRAY + (0, 0)):
    flags = (first.data_ptr(), *first.stride()) if first is not None else (0, 0, 0)
    return _RECURRENCE.pack(_DTYPES[gate.dtype], *gate.shape, *_array3(gate), *_array3(update), *h, *flags, _ptr(state), _ptr(state_out), _ptr(checkpoints), _ptr(work), *backward)


def _recurrence_forward(gate, update, first, state, state_out, checkpoints=None):
    h = torch.empty_like(update)
    device = gate.device
    last = state_out if state_out is not None else torch.empty(gate.shape[1:], dtype=torch.float32, device=device)
    work = _bytes(_recurrence_workspace(*gate.shape), device)
    _run(_lib.recurrence_forward, "gated_recurrence", device.index, _recurrence_args(gate, update, _array3(h), first, state, last, checkpoints, work))
    return h, last


class _GatedRecurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, update, first, state):
        T, N, D = gate.shape
        checkpoints = torch.empty((_checkpoints(T), N, D), dtype=torch.float32, device=gate.device)
        h, last = _recurrence_forward(gate, update, first, state, None, checkpoints)
        ctx.save_for_backward(gate, update, first, state, checkpoints)
        ctx.set_materialize_grads(False)
        return h, last

    @staticmethod
    @once_differentiable
    def backward(ctx, d_h, d_last):
        gate, update, first, state, checkpoints = ctx.saved_tensors
        wanted = ctx.needs_input_grad
        d_gate = torch.empty_like(gate) if wanted[0] else None
        d_update = torch.empty_like(update) if wanted[1] else None
        d_state = torch.empty_like(state) if wanted[3] else None
        if d_last is not None:
            d_last = d_last.contiguous()
        work = _bytes(_recurrence_workspace(*gate.shape), gate.device)
        arrays = [_NO_ARRAY if x is None else _array3(x) for x in (d_h, d_gate, d_update)]
        a = _recurrence_args(gate, update, _NO_ARRAY, first, state, None, checkpoints, work, (*arrays[0], *arrays[1], *arrays[2], _ptr(d_last), _ptr(d_state)))
        _run(_lib.recurrence_backward, "gated_recurrence", gate.device.index, a)
        return d_gate, d_update, None, d_state


def gated_recurrence(gate, update, first=None, state=None, state_out=None):
    """h[t] = gate[t] * h[t-1] + update[t] along the steps of a window, each env and channel a chain of its own; where first[t] is set an episode
    begins and h[t] = update[t].  Returns (h, state): h [T, N, D] in the inputs' type, and the state behind the last step, float32 [N, D], to begin the
    next window or the next single step (T = 1) with.

    gate, update: [T, N, D] (or [T, N]) float32, float16 or bfloat16, any strides; first: [T, N] uint8 or bool, None: no episode begins; state:
    float32 [N, D] (or [N]), None: zeros.  state_out: a float32 buffer that takes the new state, `state` itself to move it on in place; only without
    gradients.  Differentiable in gate, update and state, once."""
    _tensor(gate, "gate", _FLOATS)
    shape = gate.shape
    if len(shape) not in (2, 3):
        raise ValueError(f"gate has to be [T, N, D] or [T, N], not {tuple(shape)}")
    _tensor(update, "update", (gate.dtype,), shape)
    if first is not None:
        _tensor(first, "first", _FLAGS, shape[:2])
    if state is not None:
        _tensor(state, "state", _F32, shape[1:])
    if state_out is not None:
        _tensor(state_out, "state_out", _F32, shape[1:])
        _need(state_out.is_contiguous(), "state_out has to be contiguous")
        _need(not _wants_grad(gate, update, state, state_out), "state_out overwrites a state: call under torch.no_grad(), or take the returned state")
    _on_gpu(gate, update, first, state, state_out)
    flat = len(shape) == 2
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
    _tensor(values, "values", _FLOATS, (T + 1, N))
    _tensor(first, "first", _FLAGS, (T + 1, N))
    _number(gamma, "gamma", 0.0, 1.0)
    _number(lam, "lam", 0.0, 1.0)
    _constant(rew, "rew")
    _constant(values, "values")
    device = _on_gpu(rew, values, first)
    adv = torch.empty((T, N), dtype=torch.float32, device=device)
    ret = torch.empty((T, N), dtype=torch.float32, device=device)
    if T and N:
        work = _bytes(_recurrence_workspace(T, N, 1), device)
        a = _ADVANTAGE.pack(_DTYPES[values.dtype], T, N, rew.data_ptr(), *rew.stride(), values.data_ptr(), *values.stride(), first.data_ptr(), *first.stride(), gamma, lam,
                            adv.data_ptr(), ret.data_ptr(), _ptr(work))
        _run(_lib.advantages, "advantages", device.index, a)
    return adv, ret


# ---- rows of logits --------------------------------------------------------------------------------------------------------------------------


def _layout(x, what):
    """(inner, outer stride, inner stride) of the rows of x [..., columns]: the leading dimensions as at most two strided ones"""
    if x.is_contiguous():
        return 1, x.shape[-1], 0
    *lead, columns = zip(x.shape, x.stride())
    if columns[0] != 1 and columns[1] != 1:
        raise ValueError(f"the columns of {what} have to be contiguous")
    dims = []
    for size, stride in lead:
        if size == 1:
            continue
        if dims and dims[-1][1] == stride * size:
            dims[-1] = (dims[-1][0] * size, stride)
        else:
            dims.append((size, stride))
    if len(dims) > 2:
        raise ValueError(f"the leading dimensions of {what} are strided in more than two ways: make it contiguous")
    if len(dims) == 2:
        return dims[1][0], dims[0][1], dims[1][1]
    return 1, dims[0][1] if dims else 0, 0


def _rows(logits, layout, actions, d_logits=None, work=None):
    inner, outer_stride, inner_stride = layout
    columns = logits.shape[-1]
    return _ROWS.pack(_DTYPES[logits.dtype], logits.numel() // columns, columns, inner or 1, logits.data_ptr(), outer_stride, inner_stride, actions.data_ptr(),
                      actions.dtype == torch.int64, _ptr(d_logits), _ptr(work))


def _check_rows(logits, actions):
    _tensor(logits, "logits", _FLOATS)
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError("logits have to be [..., columns] with one column at least")
    _tensor(actions, "actions", _INTS, logits.shape[:-1])


def _action_logprobs(logits, layout, actions, grad):
    device, lead = logits.device, logits.shape[:-1]
    logp = torch.empty(lead, dtype=torch.float32, device=device)
    entropy = torch.empty(lead, dtype=torch.float32, device=device)
    lse = torch.empty(lead, dtype=torch.float32, device=device) if grad else None
    _run(_lib.action_logprobs, "action_logprobs", device.index, _rows(logits, layout, actions), logp.data_ptr(), entropy.data_ptr(), _ptr(lse))
    return logp, entropy, lse


class _ActionLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, layout, actions):
        logp, entropy, lse = _action_logprobs(logits, layout, actions, True)
        ctx.save_for_backward(logits, actions, lse, entropy)
        ctx.set_materialize_grads(False)
        return logp, entropy

    @staticmethod
    @once_differentiable
    def backward(ctx, d_logp, d_entropy):
        logits, actions, lse, entropy = ctx.saved_tensors
        d_logits = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        d_logp = None if d_logp is None else d_logp.contiguous()
        d_entropy = None if d_entropy is None else d_entropy.contiguous()
        _run(_lib.action_logprobs_backward, "action_logprobs", logits.device.index, _rows(logits, _layout(logits, "logits"), actions, d_logits), lse.data_ptr(), entropy.data_ptr(),
             _ptr(d_logp), _ptr(d_entropy))
        return d_logits, None, None


def action_logprobs(logits, actions):
    """(logp, entropy), float32 [...]: the log-probability of actions[...] under softmax(logits[..., :]) and the entropy of that distribution.

    logits: [..., columns] float32, float16 or bfloat16, columns contiguous; actions: [...] int32 or int64.  A column of -inf is an action that
    cannot be taken; a row of nothing else has log-probability -inf, entropy 0 and a zero gradient.  An action outside [0, columns) -- the -1 of a forced
    reset -- has no log-probability: NaN, and a NaN gradient unless its gradients coming in are zero.  Differentiable in logits, once."""
    _check_rows(logits, actions)
    _on_gpu(logits, actions)
    layout = _layout(logits, "logits")
    if logits.numel() == 0:
        empty = logits.sum(-1, dtype=torch.float32)
        return empty, empty * 1
    actions = actions.contiguous()
    if _wants_grad(logits):
        return _ActionLogprobs.apply(logits, layout, actions)
    return _action_logprobs(logits, layout, actions, False)[:2]


class PolicyLoss(NamedTuple):
    loss: torch.Tensor   # float32, differentiable in the logits
    stats: torch.Tensor  # float32 [4]: the means of -objective, KL, entropy and of (ratio outside the clip range), constants


def _policy_args(coefs, work, d_logits, logits, actions, old, adv, valid, ref_logits, ref_logprobs, scale=None, loss=None, stats=None, resume=0):
    if ref_logits is None:
        layout, ref_strides = _layout(logits, "logits"), (0, 0)
    else:
        layout, (_, *ref_strides) = _common_layout(logits, ref_logits)
    return (_rows(logits, layout, actions, d_logits, work),
            _POLICY.pack(old.data_ptr(), adv.data_ptr(), _ptr(valid), _ptr(ref_logits), *ref_strides, _ptr(ref_logprobs), *coefs, _ptr(scale), _ptr(loss), _ptr(stats), resume))


def _policy_forward(coefs, d_logits, *tensors):
    logits = tensors[0]
    device, columns = logits.device, logits.shape[-1]
    loss, stats = torch.empty((), dtype=torch.float32, device=device), torch.empty(4, dtype=torch.float32, device=device)
    work = _bytes(_rows_workspace(logits.numel() // columns, columns), device)
    _run(_lib.policy_loss, "policy_loss", device.index, *_policy_args(coefs, work, d_logits, *tensors, loss=loss, stats=stats))
    return loss, stats, work


def _capture(device):
    return _lib.capture_id(_stream(device.index))


class _PolicyLoss(torch.autograd.Function):
    """The forward call writes the gradient too, from the row that it has in registers.  The first backward pass hands it out, after a kernel that goes
    over the rows again only where the loss's own gradient is not 1; each further one (retain_graph) computes its own, and so does a backward pass that
    is captured apart from its forward call."""

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
        tensors = ctx.saved_tensors
        logits = tensors[0]
        d_logits, ctx.d_logits, resume = ctx.d_logits, None, 3
        if d_logits is None or not ctx.capture == _capture(logits.device) >= 0:
            d_logits, resume = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device), 1
        _run(_lib.policy_loss, "policy_loss", logits.device.index, *_policy_args(ctx.coefs, ctx.work, d_logits, *tensors, scale=d_loss, resume=resume))
        return None, d_logits, None, None, None, None, None, None


def _common_layout(x, y):
    """the rows of two equally shaped tensors under one split of their leading dimensions, or ValueError"""
    if x.is_contiguous() and y.is_contiguous():
        return (1, x.shape[-1], 0), (1, x.shape[-1], 0)
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
    for x, what in ((old_logprobs, "old_logprobs"), (advantages, "advantages")):
        _tensor(x, what, _F32, lead)
        _constant(x, what)
    if ref_logprobs is not None:
        _tensor(ref_logprobs, "ref_logprobs", _F32, lead)
        _constant(ref_logprobs, "ref_logprobs")
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
    actions, old_logprobs, advantages, valid, ref_logprobs = (None if x is None else x.contiguous() for x in (actions, old_logprobs, advantages, valid, ref_logprobs))
    coefs = float(low), float(high), float(kl_coef), float(entropy_coef)
    tensors = logits, actions, old_logprobs, advantages, valid, ref_logits, ref_logprobs
    return PolicyLoss(*(_PolicyLoss.apply(coefs, *tensors) if _wants_grad(logits) else _policy_forward(coefs, None, *tensors)[:2]))
