"""CPU: the learner operators' refusals (before anything runs) and their C entry points."""
import ctypes as C
import os
import re
import struct
import subprocess
import sys

import pytest
import torch

from helpers import HIP_LIB, REPO
from procgen_amd import learner_ops as ops

F, U = torch.float32, torch.uint8


def z(*shape, dtype=F):
    return torch.zeros(shape, dtype=dtype)


def test_library_exports_every_declared_symbol():
    if not os.path.exists(HIP_LIB):
        pytest.skip("libenv.so not built (run __graft_entry__.build())")
    src = open(os.path.join(REPO, "include", "procgen_amd_learner.h")).read()
    syms = re.findall(r"^LIBENV_API\s+[\w\s\*]+?\b(\w+)\s*\(", src, re.M)
    assert len(syms) >= 8
    lib = C.CDLL(HIP_LIB)
    for s in syms:
        assert hasattr(lib, s), f"libenv.so does not export {s}"


def test_c_entries_refuse_what_they_cannot_run():
    """-1, nothing enqueued and no device touched: this runs where there is none"""
    if not os.path.exists(HIP_LIB):
        pytest.skip("libenv.so not built (run __graft_entry__.build())")
    lib = C.CDLL(HIP_LIB)
    zeros = bytes(1024)

    def recurrence(dtype, T):  # the struct's first fields; no arrays
        return struct.pack("@4i", dtype, T, 1, 1) + zeros

    assert lib.procgen_amd_recurrence_forward(recurrence(7, 1), 0, None) == -1
    for T in (0, 4):
        assert lib.procgen_amd_recurrence_forward(recurrence(0, T), 0, None) == -1 and lib.procgen_amd_recurrence_backward(recurrence(0, T), 0, None) == -1
    assert lib.procgen_amd_advantages(struct.pack("@3i", 0, 4, 4) + zeros, 0, None) == -1
    for columns in (0, 3):
        rows = struct.pack("@i3q", 0, 4, columns, 1) + zeros
        assert lib.procgen_amd_action_logprobs(rows, None, None, None, 0, None) == -1
        assert lib.procgen_amd_action_logprobs_backward(rows, None, None, None, None, 0, None) == -1
        assert lib.procgen_amd_policy_loss(rows, zeros, 0, None) == -1
    assert lib.procgen_amd_policy_loss(None, None, 0, None) == -1


@pytest.mark.parametrize("kind,call", [
    (ValueError, lambda: ops.gated_recurrence(z(4), z(4))),
    (ValueError, lambda: ops.gated_recurrence(z(4, 2, 3), z(4, 2, 2))),
    (TypeError, lambda: ops.gated_recurrence(z(4, 2, 3), z(4, 2, 3, dtype=torch.float16))),
    (TypeError, lambda: ops.gated_recurrence(z(4, 2, 3, dtype=torch.float64), z(4, 2, 3, dtype=torch.float64))),
    (TypeError, lambda: ops.gated_recurrence([0.5], z(4, 2, 3))),
    (ValueError, lambda: ops.gated_recurrence(z(4, 2, 3), z(4, 2, 3), first=z(4, 3, dtype=U))),
    (TypeError, lambda: ops.gated_recurrence(z(4, 2, 3), z(4, 2, 3), first=z(4, 2))),
    (TypeError, lambda: ops.gated_recurrence(z(4, 2, 3), z(4, 2, 3), state=z(2, 3, dtype=torch.bfloat16))),
    (ValueError, lambda: ops.gated_recurrence(z(4, 2, 3), z(4, 2, 3), state=z(3))),
    (ValueError, lambda: ops.gated_recurrence(z(4, 2, 3), z(4, 2, 3), state_out=z(3, 2).T)),
    (ValueError, lambda: ops.gated_recurrence(z(4, 2, 3).requires_grad_(), z(4, 2, 3), state_out=z(2, 3))),
    (ValueError, lambda: ops.gated_recurrence(z(4, 2, 3), z(4, 2, 3))),  # not on a GPU
    (ValueError, lambda: ops.advantages(z(4), z(5), z(5, dtype=U), gamma=0.9, lam=0.9)),
    (ValueError, lambda: ops.advantages(z(4, 2), z(4, 2), z(5, 2, dtype=U), gamma=0.9, lam=0.9)),
    (ValueError, lambda: ops.advantages(z(4, 2), z(5, 2), z(4, 2, dtype=U), gamma=0.9, lam=0.9)),
    (TypeError, lambda: ops.advantages(z(4, 2, dtype=torch.float16), z(5, 2), z(5, 2, dtype=U), gamma=0.9, lam=0.9)),
    (ValueError, lambda: ops.advantages(z(4, 2), z(5, 2), z(5, 2, dtype=U), gamma=1.1, lam=0.9)),
    (ValueError, lambda: ops.advantages(z(4, 2), z(5, 2), z(5, 2, dtype=U), gamma=float("nan"), lam=0.9)),
    (ValueError, lambda: ops.advantages(z(4, 2), z(5, 2).requires_grad_(), z(5, 2, dtype=U), gamma=0.9, lam=0.9)),
    (TypeError, lambda: ops.advantages(z(4, 2), z(5, 2), z(5, 2, dtype=U), gamma=z(1), lam=0.9)),
    (TypeError, lambda: ops.action_logprobs(z(4, 3), z(4))),
    (ValueError, lambda: ops.action_logprobs(z(4, 3), z(3, dtype=torch.int32))),
    (ValueError, lambda: ops.action_logprobs(z(4, 0), z(4, dtype=torch.int32))),
    (ValueError, lambda: ops.action_logprobs(z(4, 3), z(4, dtype=torch.int32))),  # not on a GPU
    (ValueError, lambda: ops.policy_loss(z(4, 3), z(4, dtype=torch.int32), z(3), z(4))),
    (TypeError, lambda: ops.policy_loss(z(4, 3), z(4, dtype=torch.int32), z(4), None)),
    (ValueError, lambda: ops.policy_loss(z(4, 3), z(4, dtype=torch.int32), z(4), z(4), ref_logits=z(4, 2))),
    (ValueError, lambda: ops.policy_loss(z(4, 3), z(4, dtype=torch.int32), z(4), z(4), ref_logits=z(4, 3), ref_logprobs=z(4))),
    (ValueError, lambda: ops.policy_loss(z(4, 3), z(4, dtype=torch.int32), z(4), z(4), kl_coef=0.1)),
    (ValueError, lambda: ops.policy_loss(z(4, 3), z(4, dtype=torch.int32), z(4), z(4), clip=-0.1)),
    (ValueError, lambda: ops.policy_loss(z(4, 3), z(4, dtype=torch.int32), z(4), z(4), clip=(1.5, 0.2))),
    (TypeError, lambda: ops.policy_loss(z(4, 3), z(4, dtype=torch.int32), z(4), z(4), clip="0.2")),
    (ValueError, lambda: ops.policy_loss(z(4, 3), z(4, dtype=torch.int32), z(4), z(4).requires_grad_())),
    (TypeError, lambda: ops.policy_loss(z(4, 3), z(4, dtype=torch.int32), z(4), z(4), valid=z(4))),
])
def test_refusals(kind, call):
    with pytest.raises(kind):
        call()


def test_more_than_32_bits_can_count_is_refused(monkeypatch):
    monkeypatch.setattr(ops, "_on_gpu", lambda x, *others: x.device)  # the shapes are checked behind the devices
    one = z(1)
    with pytest.raises(ValueError, match="steps"):
        ops.gated_recurrence(one.expand(1 << 31, 1), one.expand(1 << 31, 1))
    with pytest.raises(ValueError, match="chains"):
        ops.gated_recurrence(one.expand(1, 1 << 16, 1 << 16), one.expand(1, 1 << 16, 1 << 16))
    with pytest.raises(ValueError, match="envs"):
        ops.advantages(one.expand(1, 1 << 31), one.expand(2, 1 << 31), z(1, dtype=U).expand(2, 1 << 31), gamma=0.9, lam=0.9)
    with pytest.raises(ValueError, match="rows"):
        ops.action_logprobs(one.expand(1 << 31, 1), z(1, dtype=torch.int32).expand(1 << 31))
    with pytest.raises(ValueError, match="columns"):
        ops.action_logprobs(one.expand(1, 1 << 31), z(1, dtype=torch.int32))


def test_layouts():
    x = torch.zeros(6, 5, 4, 8)
    assert ops._layout(x, "x") == (1, 8, 0)  # (rows per inner group, stride of the groups, stride inside)
    assert ops._layout(x[:, :3], "x") == (12, 160, 8)
    assert ops._layout(x.transpose(0, 1)[0], "x") == (4, 160, 8)
    assert ops._layout(torch.zeros(7, 3)[:, :2], "x") == (1, 3, 0)
    assert ops._layout(torch.zeros(3), "x") == (1, 3, 0)
    assert ops._layout(torch.zeros(1, 3).expand(5, 3), "x") == (1, 0, 0)
    with pytest.raises(ValueError):
        ops._layout(x[:, :3, :2], "x")
    with pytest.raises(ValueError):
        ops._layout(torch.zeros(3, 4).T, "x")
    assert ops._common_layout(torch.zeros(6, 5, 8), torch.zeros(6, 7, 8)[:, :5]) == [(5, 40, 8), (5, 56, 8)]
    with pytest.raises(ValueError):
        ops._common_layout(torch.zeros(6, 5, 4, 8)[:, :4], torch.zeros(6, 4, 5, 8)[:, :, :4])


def test_package_import_does_not_touch_torch():
    code = "import sys; sys.path.insert(0, %r); import procgen_amd, procgen_amd.torch_view; assert 'torch' not in sys.modules" % REPO
    assert subprocess.run([sys.executable, "-c", code]).returncode == 0
