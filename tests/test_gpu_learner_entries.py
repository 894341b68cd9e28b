"""GPU: the learner operators' C entry points as a caller without torch's autograd uses them (include/procgen_amd_learner.h)."""
import ctypes as C

import pytest
import torch

from helpers import HIP_LIB
from test_gpu_learner_ops import TINY, check, gen, rand, recurrence_64, recurrence_inputs, rounding

pytestmark = pytest.mark.gpu


class Array3(C.Structure):
    _fields_ = [("data", C.c_void_p), ("t_stride", C.c_longlong), ("n_stride", C.c_longlong), ("d_stride", C.c_longlong)]


class Recurrence(C.Structure):
    _fields_ = [("dtype", C.c_int), ("T", C.c_int), ("N", C.c_int), ("D", C.c_int), ("gate", Array3), ("update", Array3), ("h", Array3), ("first", C.c_void_p),
                ("first_t_stride", C.c_longlong), ("first_n_stride", C.c_longlong), ("state", C.c_void_p), ("state_out", C.c_void_p), ("checkpoints", C.c_void_p),
                ("workspace", C.c_void_p), ("d_h", Array3), ("d_gate", Array3), ("d_update", Array3), ("d_state_out", C.c_void_p), ("d_state", C.c_void_p)]


def array3(x):
    return Array3(x.data_ptr(), *x.stride())


def library():
    lib = C.CDLL(HIP_LIB)
    lib.procgen_amd_recurrence_checkpoints.restype = lib.procgen_amd_recurrence_workspace.restype = C.c_longlong
    return lib


@pytest.mark.parametrize("T,N,D", [(1, 5, 8), (4, 3, 33), (5, 3, 8), (70, 2, 40), (5000, 1, 16)])
def test_a_state_moved_on_in_place_leaves_the_backward_pass_its_checkpoints(T, N, D):
    """state_out may be state; the backward call then finds the new state there, and begins from the checkpoints alone"""
    lib = library()
    gate, update, first, state, _ = recurrence_inputs(T, N, D, "f32", T)
    g = gen(T)
    d_h, d_last = rand((T, N, D), g), rand((N, D), g)
    want = recurrence_64(gate, update, first, state, d_h, d_last)
    gate, update, first, moved, d_h, d_last = (x.cuda() for x in (gate, update, first, state, d_h, d_last))
    h, d_gate, d_update = (torch.full_like(gate, float("nan")) for _ in range(3))
    d_state = torch.full_like(moved, float("nan"))
    checkpoints = torch.empty(lib.procgen_amd_recurrence_checkpoints(T) * N * D, device="cuda")
    work = torch.empty(max(1, lib.procgen_amd_recurrence_workspace(T, N, D)), dtype=torch.uint8, device="cuda")
    a = Recurrence(0, T, N, D, array3(gate), array3(update), array3(h), first.data_ptr(), N, 1, moved.data_ptr(), moved.data_ptr(), checkpoints.data_ptr(), work.data_ptr(),
                   array3(d_h), array3(d_gate), array3(d_update), d_last.data_ptr(), d_state.data_ptr())
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert lib.procgen_amd_recurrence_forward(C.byref(a), 0, stream) == 0
    assert lib.procgen_amd_recurrence_backward(C.byref(a), 0, stream) == 0
    f32 = torch.float32
    check(h, want["h"], want["E_h"] + rounding(want["h"], f32), "h")
    check(moved, want["last"], want["E_last"] + TINY[f32], "state")
    check(d_update, want["d_update"], want["E_d_update"] + rounding(want["d_update"], f32), "d_update")
    check(d_gate, want["d_gate"], want["E_d_gate"] + rounding(want["d_gate"], f32), "d_gate")
    check(d_state, want["d_state"], want["E_d_state"] + TINY[f32], "d_state")
