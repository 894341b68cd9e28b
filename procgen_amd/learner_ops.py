"""
Learner operators over a rollout: what a policy gradient needs of a window of T steps of N envs, computed on the GPU where torch_view's tensors
already are.  Entry points of libenv.so (include/procgen_amd_learner.h), reached through csrc/learner_torch.cpp; hand-written kernels, no CPU path.

    views = torch_view.device_views(env)                         # rew, first, action of every step, on the GPU
    h, memory = gated_recurrence(gate, update, first, memory)    # the policy's memory over the window, cut where an episode begins
    logp, entropy = action_logprobs(logits, actions)             # what the rollout stores about its own actions
    adv, ret = advantages(rew, values, first, gamma=0.999, lam=0.95)
    out = policy_loss(logits, actions, logp, adv, entropy_coef=0.01)
    out.loss.backward()

Every operator runs on the current stream of its tensors' device, does not synchronise, keeps nothing between calls and can be captured into a graph.
Tensors may be strided (batch-major windows, slices, expanded dimensions); arguments that an operator does not take raise TypeError or ValueError
before anything runs.  Element types: float32, float16, bfloat16; sums, states and statistics are held in 32 bits or more.
Gradients are reverse-mode ones of the first order: a tensor with a forward-mode tangent and a call that is being traced are refused, too.
"""
import importlib.util
import os
import threading
from typing import NamedTuple

import torch

from .env import DEFAULT_LIB_DIR


class _Extension:
    """csrc/learner_torch.cpp, loaded when an operator first runs"""

    def __init__(self):
        self._loading = threading.Lock()  # several threads may be the first

    def __getattr__(self, name):
        with self._loading:
            if name not in self.__dict__:
                self._load()
        if name not in self.__dict__:
            raise AttributeError(name)
        return self.__dict__[name]

    def _load(self):
        path = os.path.join(DEFAULT_LIB_DIR, "learner_torch.so")
        if not os.path.exists(path):
            raise ImportError(f"{path} is not there: make in procgen_amd/csrc builds it, where a torch with ROCm's headers is installed")
        spec = importlib.util.spec_from_file_location("learner_torch", path)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        for fn in ("gated_recurrence", "advantages", "action_logprobs", "policy_loss"):
            setattr(self, fn, getattr(module, fn))


_ext = _Extension()


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
    if x.is_neg():
        raise ValueError(f"{what} is a view that torch negates when it reads it, and the kernels do not: resolve_neg() it")


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


_MOST = 0x7FFFFF00  # steps, chains, rows: counted in 32 bits


def _not_too_many(n, what):
    if n > _MOST:
        raise ValueError(f"{n} {what}: more than {_MOST} are not taken")


_FLAGS = (torch.uint8, torch.bool)
_F32 = (torch.float32,)
_INTS = (torch.int32, torch.int64)
_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


def _wants_grad(*tensors):
    if torch.is_grad_enabled():
        for x in tensors:
            if x is not None and x.requires_grad:
                return True
    return False


# ---- the memory of a policy ------------------------------------------------------------------------------------------------------------------


def _overlap(x, y):
    """whether the memory that two tensors span has a part in common"""
    spans = []
    for z in (x, y):
        if z.numel() == 0:
            return False
        spans.append((z.data_ptr(), z.data_ptr() + z.element_size() * (1 + sum((n - 1) * s for n, s in zip(z.shape, z.stride())))))
    return spans[0][0] < spans[1][1] and spans[1][0] < spans[0][1]


def gated_recurrence(gate, update, first=None, state=None, state_out=None):
    """h[t] = gate[t] * h[t-1] + update[t] along the steps of a window, each env and channel a chain of its own; where first[t] is set an episode
    begins and h[t] = update[t].  Returns (h, state): h [T, N, D] in the inputs' type, and the state behind the last step, float32 [N, D], to begin the
    next window or the next single step (T = 1) with.

    gate, update: [T, N, D] (or [T, N]) float32, float16 or bfloat16, any strides; first: [T, N] uint8 or bool, None: no episode begins; state:
    float32 [N, D] (or [N]), None: zeros.  state_out: a float32 buffer that takes the new state, `state` itself to move it on in place; only without
    gradients.  Differentiable in gate, update and state, once.

    Products of neighbouring gates are formed on the way (of 8 steps, and of up to the whole window where there are few chains): where such a product
    passes float32's range -- gates larger than one over a long stretch -- h behind it is not finite, unless h before it is zero or an episode begins in
    between; gradients alike, from the last step to the first."""
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
    _not_too_many(shape[0], "steps")
    _not_too_many(shape[1:].numel(), "chains")
    if state_out is not None:
        for x, what in ((gate, "gate"), (update, "update"), (first, "first"), (state, "state")):
            if x is not None and _overlap(x, state_out) and not (what == "state" and x.data_ptr() == state_out.data_ptr() and x.is_contiguous()):
                raise ValueError(f"state_out lies inside of the memory of {what}")
    flat = len(shape) == 2
    if flat:
        gate, update = gate.unsqueeze(2), update.unsqueeze(2)
        state = state.unsqueeze(1) if state is not None else None
        state_out = state_out.unsqueeze(1) if state_out is not None else None
    if gate.numel() == 0:  # no step or no chain: the state stays
        h = (update + gate) * 1
        last = state * 1 if state is not None else torch.zeros(gate.shape[1:], dtype=torch.float32, device=gate.device)
        if state_out is not None:
            last = state_out.copy_(last)
    else:
        h, last = _ext.gated_recurrence(gate, update, first, state, state_out)
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
    _not_too_many(T, "steps")
    _not_too_many(N, "envs")
    if T and N:
        return _ext.advantages(rew, values, first, gamma, lam)
    return tuple(torch.empty((T, N), dtype=torch.float32, device=device) for _ in range(2))


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


def _check_rows(logits, actions):
    _tensor(logits, "logits", _FLOATS)
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError("logits have to be [..., columns] with one column at least")
    _tensor(actions, "actions", _INTS, logits.shape[:-1])
    _not_too_many(actions.numel(), "rows")
    _not_too_many(logits.shape[-1] + (1 << 18), "columns")


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
    return _ext.action_logprobs(logits, actions, layout[0] or 1, layout[1], layout[2])


class PolicyLoss(NamedTuple):
    loss: torch.Tensor   # float32, differentiable in the logits
    stats: torch.Tensor  # float32 [4]: the means of -objective, KL, entropy and of (ratio outside the clip range), constants


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
    log-probability of the action taken; at most one of the two is given, and the term is 0 without.  With kl_coef = 0 a reference is only watched: it
    changes stats, and nothing else whatever it holds.  Where ref_logits excludes what the policy allows KL is infinite, or about as large as the numbers
    that exclude it (infinite, too, where their sum passes float32's range).  clip: a number, or (below, above).  logits as for
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
    layout, ref_strides = _layout(logits, "logits"), (0, 0)
    if ref_logits is not None:
        _layout(ref_logits, "ref_logits")
        layout, (_, *ref_strides) = _common_layout(logits, ref_logits)
    return PolicyLoss(*_ext.policy_loss(logits, actions, old_logprobs, advantages, valid, ref_logits, ref_logprobs, low, high, kl_coef, entropy_coef, layout[0] or 1, layout[1], layout[2],
                                        *ref_strides))
