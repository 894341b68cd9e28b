"""CPU: sizes that the learner operators' C entry points refuse, before any device is touched."""
import ctypes as C
import os
import struct

import pytest

from helpers import HIP_LIB

pytestmark = pytest.mark.skipif(not os.path.exists(HIP_LIB), reason="libenv.so not built (run __graft_entry__.build())")
SOME = 4096  # a pointer that nothing may follow


def rows(count, columns, inner):
    return struct.pack("@i3qP2qPi2P", 0, count, columns, inner, SOME, columns, columns, SOME, 0, SOME, SOME)


@pytest.mark.parametrize("count,columns,inner", [(4, 3, 1 << 32), (4, 3, 1 << 40), (4, 3, (1 << 63) - 1), (4, 3, 0), (4, 3, -1), (1 << 31, 3, 1), (4, 1 << 31, 1), (-1, 3, 1)])
def test_rows_that_32_bits_cannot_count_are_refused(count, columns, inner):
    lib = C.CDLL(HIP_LIB)
    p = rows(count, columns, inner)
    one = C.c_void_p(SOME)
    assert lib.procgen_amd_action_logprobs(p, one, one, one, 0, None) == -1
    assert lib.procgen_amd_action_logprobs_backward(p, one, one, one, one, 0, None) == -1
    policy = struct.pack("@4P2qP4f3Pi4x", SOME, SOME, 0, 0, 0, 0, 0, 0.2, 0.2, 0.0, 0.0, 0, SOME, SOME, 0)
    assert lib.procgen_amd_policy_loss(p, policy, 0, None) == -1
