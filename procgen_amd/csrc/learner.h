// learner.h -- what the learner kernels (learner_scan.hip, learner_rows.hip) share: element types, wave reductions, launches at a C entry.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/procgen_amd_learner.h"

namespace pgamd {
namespace learner {

constexpr int WAVE = 64;

// ---- element types: 32 bits in registers whatever the memory holds ------------------------------------------------------------
struct F32 {
    typedef float T;
};
struct F16 {
    typedef _Float16 T;
};
struct BF16 {
    typedef __bf16 T;
};

// ---- reductions over a wave (every lane gets the result); `op` is taken in a fixed order, so results do not change from run to run ----
template <class T, class Op>
__device__ inline T wave_reduce(T v, Op op) {
    for (int d = WAVE / 2; d > 0; d >>= 1) v = op(v, __shfl_xor(v, d, WAVE));
    return v;
}
struct Sum {
    template <class T>
    __device__ T operator()(T a, T b) const { return a + b; }
};

// ---- a C entry's frame: the caller's current device is put back, whatever happens in between ------------------------------------------------
struct OnDevice {
    int old = -1;
    hipError_t err;
    explicit OnDevice(int device) {
        (void)hipGetLastError();  // what another call left behind (an event that was not ready, say) is not a launch's error
        err = hipGetDevice(&old);
        if (err == hipSuccess && old != device) err = hipSetDevice(device);
        else old = -1;
    }
    ~OnDevice() {
        if (old >= 0) (void)hipSetDevice(old);
    }
};
inline int launched() { return (int)hipGetLastError(); }  // the launch's own error: a C entry returns it and leaves none behind

inline bool known_dtype(int d) { return d >= PROCGEN_AMD_F32 && d <= PROCGEN_AMD_BF16; }
template <class Fn>
inline int by_dtype(int dtype, Fn fn) {
    switch (dtype) {
        case PROCGEN_AMD_F32: return fn(F32());
        case PROCGEN_AMD_F16: return fn(F16());
        default: return fn(BF16());
    }
}

}  // namespace learner
}  // namespace pgamd
