// learner_scan.hip -- recurrences along the steps of a rollout window: the gated linear recurrence of a policy's memory (forward, backward) and the
// advantages of its rewards, which are the same recurrence run from the last step to the first.
#include "learner.h"

namespace pgamd {
namespace learner {
namespace {

// one chain (n, d) per lane, all steps in order
template <class E>
__global__ void recurrence_forward(procgen_amd_recurrence p) {
    const long long c = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= (long long)p.N * p.D) return;
    const long long n = c / p.D, d = c % p.D;
    float h = p.state ? p.state[c] : 0.f;
    for (long long t = 0; t < p.T; t++) {
        const bool cut = p.first && p.first[t * p.first_t_stride + n * p.first_n_stride];
        const float b = load<E>(p.update.data, t * p.update.t_stride + n * p.update.n_stride + d * p.update.d_stride);
        const float a = load<E>(p.gate.data, t * p.gate.t_stride + n * p.gate.n_stride + d * p.gate.d_stride);
        h = cut ? b : fmaf(a, h, b);
        store<E>(p.h.data, t * p.h.t_stride + n * p.h.n_stride + d * p.h.d_stride, h);
    }
    if (p.state_out) p.state_out[c] = h;
}

template <class E>
__global__ void recurrence_backward(procgen_amd_recurrence p) {
    const long long c = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= (long long)p.N * p.D) return;
    const long long n = c / p.D, d = c % p.D;
    float g = p.d_state_out ? p.d_state_out[c] : 0.f;  // what reaches h[t] from the steps behind it
    for (long long t = p.T - 1; t >= 0; t--) {
        const bool cut = p.first && p.first[t * p.first_t_stride + n * p.first_n_stride];
        if (p.d_h.data) g += load<E>(p.d_h.data, t * p.d_h.t_stride + n * p.d_h.n_stride + d * p.d_h.d_stride);
        const float a = load<E>(p.gate.data, t * p.gate.t_stride + n * p.gate.n_stride + d * p.gate.d_stride);
        const float before = t > 0 ? load<E>(p.h.data, (t - 1) * p.h.t_stride + n * p.h.n_stride + d * p.h.d_stride) : p.state ? p.state[c] : 0.f;
        if (p.d_update.data) store<E>(p.d_update.data, t * p.d_update.t_stride + n * p.d_update.n_stride + d * p.d_update.d_stride, g);
        if (p.d_gate.data) store<E>(p.d_gate.data, t * p.d_gate.t_stride + n * p.d_gate.n_stride + d * p.d_gate.d_stride, cut ? 0.f : g * before);
        g = cut ? 0.f : a * g;
    }
    if (p.d_state) p.d_state[c] = g;
}

template <class E>
__global__ void advantages(procgen_amd_advantage p) {
    const long long n = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (n >= p.N) return;
    float next = 0.f, adv = 0.f;
    {
        const long long t = p.T;
        next = load<E>(p.values, t * p.values_t_stride + n * p.values_n_stride);
    }
    for (long long t = p.T - 1; t >= 0; t--) {
        const bool cut = p.first[(t + 1) * p.first_t_stride + n * p.first_n_stride];
        const float v = load<E>(p.values, t * p.values_t_stride + n * p.values_n_stride);
        const float r = p.rew[t * p.rew_t_stride + n * p.rew_n_stride];
        const float delta = (cut ? r : fmaf(p.gamma, next, r)) - v;
        adv = cut ? delta : fmaf(p.gamma * p.lam, adv, delta);
        if (p.adv) p.adv[t * p.N + n] = adv;
        if (p.ret) p.ret[t * p.N + n] = adv + v;
        next = v;
    }
}

bool shape_ok(int dtype, int T, int N, int D) { return known_dtype(dtype) && T >= 0 && N >= 0 && D >= 0 && (long long)N * D <= 0x7fffffffll; }
unsigned blocks_for(long long items) { return (unsigned)((items + 255) / 256); }

}  // namespace
}  // namespace learner
}  // namespace pgamd

using namespace pgamd::learner;

extern "C" {

LIBENV_API long long procgen_amd_recurrence_checkpoints(int T) { return 0; }
LIBENV_API long long procgen_amd_recurrence_workspace(int T, int N, int D) { return 0; }

LIBENV_API int procgen_amd_recurrence_forward(const struct procgen_amd_recurrence *a, int device, void *stream) {
    if (!a || !shape_ok(a->dtype, a->T, a->N, a->D) || a->T < 1) return -1;
    const long long chains = (long long)a->N * a->D;
    if (chains == 0) return 0;
    if (!a->gate.data || !a->update.data || !a->h.data) return -1;
    OnDevice on(device);
    if (on.err != hipSuccess) return (int)on.err;
    return by_dtype(a->dtype, [&](auto e) {
        recurrence_forward<decltype(e)><<<blocks_for(chains), 256, 0, (hipStream_t)stream>>>(*a);
        return launched();
    });
}

LIBENV_API int procgen_amd_recurrence_backward(const struct procgen_amd_recurrence *a, int device, void *stream) {
    if (!a || !shape_ok(a->dtype, a->T, a->N, a->D) || a->T < 1) return -1;
    const long long chains = (long long)a->N * a->D;
    if (chains == 0) return 0;
    if (!a->gate.data || !a->h.data) return -1;
    OnDevice on(device);
    if (on.err != hipSuccess) return (int)on.err;
    return by_dtype(a->dtype, [&](auto e) {
        recurrence_backward<decltype(e)><<<blocks_for(chains), 256, 0, (hipStream_t)stream>>>(*a);
        return launched();
    });
}

LIBENV_API int procgen_amd_advantages(const struct procgen_amd_advantage *a, int device, void *stream) {
    if (!a || !shape_ok(a->dtype, a->T, a->N, 1)) return -1;
    if (a->T == 0 || a->N == 0) return 0;
    if (!a->rew || !a->values || !a->first) return -1;
    OnDevice on(device);
    if (on.err != hipSuccess) return (int)on.err;
    return by_dtype(a->dtype, [&](auto e) {
        advantages<decltype(e)><<<blocks_for(a->N), 256, 0, (hipStream_t)stream>>>(*a);
        return launched();
    });
}

}  // extern "C"
