// learner_rows.hip -- rows of logits, one column per action: log-probabilities and entropy of the actions taken (forward, backward) and the clipped
// policy loss with its gradient.
//
// With m = max l, e[j] = exp(l[j] - m), s = sum e:  p[j] = e[j] / s,  log p[j] = (l[j] - m) - log s,  H = log s - (sum e (l - m)) / s, and against a
// reference row r (m', s' alike)  KL = (sum e ((l - m) - (r - m'))) / s + log(s' / s): every term is of the size of the differences, so nothing of
// the size of the logits cancels.  The gradients of all three operators have one form,
//     dl[j] = pick * (1[j = a] - p[j]) + p[j] * (kl * (log p[j] - log q[j] - KL) + ent * (log p[j] + H)).
#include "learner.h"

#include <algorithm>

namespace pgamd {
namespace learner {
namespace {

constexpr int ROWS_PER_BLOCK = 4;  // one wave per row
constexpr int MAX_COUNT_BLOCKS = 256;

__device__ inline long long action_of(const procgen_amd_rows &p, long long r) {
    return p.actions_are_64_bit ? ((const long long *)p.actions)[r] : (long long)((const int *)p.actions)[r];
}
__device__ inline long long row_offset(const procgen_amd_rows &p, long long r, long long outer, long long inner) { return (r / p.inner) * outer + (r % p.inner) * inner; }

struct Stats {
    float m, s, w;    // max, sum e, sum e (l - m)
    float m2, s2, u;  // of the reference row, and sum e ((l - m) - (r - m2))
};

template <class E, bool REF>
__device__ inline Stats row_stats(const typename E::T *l, const typename E::T *r, long long columns, int lane) {
    Stats x;
    x.m = x.m2 = -INFINITY;
    for (long long j = lane; j < columns; j += WAVE) {
        x.m = fmaxf(x.m, (float)l[j]);
        if (REF) x.m2 = fmaxf(x.m2, (float)r[j]);
    }
    x.m = wave_reduce(x.m, Max());
    if (REF) x.m2 = wave_reduce(x.m2, Max());
    x.s = x.w = x.s2 = x.u = 0.f;
    if (x.m > -INFINITY || x.m != x.m)
        for (long long j = lane; j < columns; j += WAVE) {
            const float d = (float)l[j] - x.m, e = __expf(d);
            x.s += e;
            if (e != 0.f) x.w += e * d;
            if (REF) {
                const float q = (float)r[j] - x.m2;
                x.s2 += __expf(q);
                if (e != 0.f) x.u += e * (d - q);
            }
        }
    x.s = wave_reduce(x.s, Sum());
    x.w = wave_reduce(x.w, Sum());
    if (REF) {
        x.s2 = wave_reduce(x.s2, Sum());
        x.u = wave_reduce(x.u, Sum());
    }
    return x;
}

template <class E>
__global__ void action_logprobs(procgen_amd_rows p, float *logp, float *entropy, float *lse) {
    const int lane = threadIdx.x % WAVE;
    const long long r = (long long)blockIdx.x * ROWS_PER_BLOCK + threadIdx.x / WAVE;
    if (r >= p.rows) return;
    const typename E::T *l = (const typename E::T *)p.logits + row_offset(p, r, p.outer_stride, p.inner_stride);
    const Stats x = row_stats<E, false>(l, nullptr, p.columns, lane);
    if (lane) return;
    const long long a = action_of(p, r);
    const bool empty = x.m == -INFINITY, known = a >= 0 && a < p.columns;
    const float log_s = logf(x.s);
    logp[r] = !known ? NAN : empty ? -INFINITY : ((float)l[a] - x.m) - log_s;
    entropy[r] = empty ? 0.f : log_s - x.w / x.s;
    if (lse) lse[r] = empty ? -INFINITY : x.m + log_s;
}

template <class E>
__global__ void action_logprobs_backward(procgen_amd_rows p, const float *lse, const float *entropy, const float *d_logp, const float *d_entropy) {
    const int lane = threadIdx.x % WAVE;
    const long long r = (long long)blockIdx.x * ROWS_PER_BLOCK + threadIdx.x / WAVE;
    if (r >= p.rows) return;
    const typename E::T *l = (const typename E::T *)p.logits + row_offset(p, r, p.outer_stride, p.inner_stride);
    typename E::T *d = (typename E::T *)p.d_logits + r * p.columns;
    const float pick = d_logp ? d_logp[r] : 0.f, ent = d_entropy ? d_entropy[r] : 0.f, z = lse[r], H = entropy[r];
    const long long a = action_of(p, r);
    const bool known = a >= 0 && a < p.columns;
    for (long long j = lane; j < p.columns; j += WAVE) {
        float g = 0.f;
        if (!(pick == 0.f && ent == 0.f) && z != -INFINITY) {
            const float log_p = (float)l[j] - z, q = __expf(log_p);
            g = (j == a ? pick : 0.f) - pick * q;
            if (q != 0.f) g -= ent * q * (log_p + H);
            if (!known) g = NAN;
        }
        d[j] = (typename E::T)g;
    }
}

// how many rows count: one partial sum per block, added up by every block that needs the number (whole numbers: any order gives the same)
__global__ void count_valid(const uint8_t *valid, long long rows, long long *counts) {
    long long n = 0;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < rows; i += (long long)gridDim.x * blockDim.x) n += valid[i] != 0;
    n = wave_reduce(n, Sum());
    __shared__ long long part[4];
    if (threadIdx.x % WAVE == 0) part[threadIdx.x / WAVE] = n;
    __syncthreads();
    if (threadIdx.x == 0) counts[blockIdx.x] = part[0] + part[1] + part[2] + part[3];
}

struct Coef {
    float pick, policy, kl, entropy, clipped;  // d loss / d logp of the action taken; the row's terms
};
template <bool REF>
__device__ inline Coef row_coef(const procgen_amd_policy &q, long long r, const Stats &x, float log_s, float logp) {
    Coef c;
    c.entropy = log_s - x.w / x.s;
    const float ratio = expf(logp - q.old_logprobs[r]), adv = q.adv[r], lo = 1.f - q.clip_low, hi = 1.f + q.clip_high;
    const float held = (ratio < lo ? lo : ratio > hi ? hi : ratio) * adv, plain = ratio * adv;
    const bool out = plain > held;  // the clipped side is the smaller one (and its gradient is zero); never where something is NaN
    c.policy = -(out ? held : plain);
    c.pick = out ? 0.f : -plain;
    c.clipped = ratio < lo || ratio > hi ? 1.f : 0.f;
    c.kl = 0.f;
    if (REF) c.kl = x.s2 > 0.f || x.s2 != x.s2 ? x.u / x.s + logf(x.s2 / x.s) : INFINITY;
    else if (q.ref_logprobs) {
        const float d = q.ref_logprobs[r] - logp;
        c.kl = expm1f(d) - d;
        c.pick -= q.kl_coef * expm1f(d);
    }
    return c;
}

template <class E, bool REF>
__global__ void policy_rows(procgen_amd_rows p, procgen_amd_policy q, const long long *counts, int count_blocks, double *partial) {
    const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
    long long n = p.rows;
    if (counts) {
        n = 0;
        for (int i = lane; i < count_blocks; i += WAVE) n += counts[i];
        n = wave_reduce(n, Sum());
    }
    const float scale = (q.scale ? *q.scale : 1.f) * (n > 0 ? (float)(1.0 / (double)n) : 0.f);
    double sum[4] = {0, 0, 0, 0};
    for (long long r = (long long)blockIdx.x * ROWS_PER_BLOCK + wave; r < p.rows; r += (long long)gridDim.x * ROWS_PER_BLOCK) {
        const typename E::T *l = (const typename E::T *)p.logits + row_offset(p, r, p.outer_stride, p.inner_stride);
        const typename E::T *l2 = REF ? (const typename E::T *)q.ref_logits + row_offset(p, r, q.ref_outer_stride, q.ref_inner_stride) : nullptr;
        typename E::T *d = p.d_logits ? (typename E::T *)p.d_logits + r * p.columns : nullptr;
        const bool used = !q.valid || q.valid[r];
        Stats x;
        if (used) x = row_stats<E, REF>(l, l2, p.columns, lane);
        if (!used || x.m == -INFINITY) {
            if (d)
                for (long long j = lane; j < p.columns; j += WAVE) d[j] = (typename E::T)0.f;
            continue;
        }
        const long long a = action_of(p, r);
        const bool known = a >= 0 && a < p.columns;
        const float log_s = logf(x.s), logp = known ? ((float)l[a] - x.m) - log_s : NAN;
        const Coef c = row_coef<REF>(q, r, x, log_s, logp);
        if (lane == 0) {
            sum[0] += c.policy;
            sum[1] += c.kl;
            sum[2] += c.entropy;
            sum[3] += c.clipped;
        }
        if (d) {
            const float inv_s = 1.f / x.s, log_s2 = REF ? logf(x.s2) : 0.f;
            for (long long j = lane; j < p.columns; j += WAVE) {
                const float dl = (float)l[j] - x.m, pj = __expf(dl) * inv_s, log_p = dl - log_s;
                float g = (j == a ? c.pick : 0.f) - c.pick * pj;
                if (pj != 0.f) {
                    float f = q.entropy_coef * (log_p + c.entropy);
                    if (REF) f += q.kl_coef * ((log_p - (((float)l2[j] - x.m2) - log_s2)) - c.kl);
                    g += pj * f;
                }
                d[j] = (typename E::T)(known ? g * scale : NAN);
            }
        }
    }
    if (!partial) return;
    __shared__ double part[ROWS_PER_BLOCK][4];
    if (lane == 0)
        for (int k = 0; k < 4; k++) part[wave][k] = sum[k];
    __syncthreads();
    if (threadIdx.x < 4) {
        double v = 0;
        for (int w = 0; w < ROWS_PER_BLOCK; w++) v += part[w][threadIdx.x];
        partial[(long long)blockIdx.x * 4 + threadIdx.x] = v;
    }
}

__global__ void policy_means(procgen_amd_policy q, long long rows, const long long *counts, int count_blocks, const double *partial, int blocks) {
    const int lane = threadIdx.x % WAVE, k = threadIdx.x / WAVE;  // wave k: the k-th mean
    long long n = rows;
    if (counts) {
        n = 0;
        for (int i = lane; i < count_blocks; i += WAVE) n += counts[i];
        n = wave_reduce(n, Sum());
    }
    double v = 0;
    for (int i = lane; i < blocks; i += WAVE) v += partial[(long long)i * 4 + k];
    v = wave_reduce(v, Sum());
    __shared__ double mean[4];
    if (lane == 0) mean[k] = n > 0 ? v / (double)n : 0.0;
    __syncthreads();
    if (threadIdx.x == 0) *q.loss = (float)(mean[0] + (q.kl_coef != 0.f ? (double)q.kl_coef * mean[1] : 0.0) - (q.entropy_coef != 0.f ? (double)q.entropy_coef * mean[2] : 0.0));
    if (lane == 0) q.stats[k] = (float)mean[k];
}

bool rows_ok(const procgen_amd_rows *p) { return p && known_dtype(p->dtype) && p->rows >= 0 && p->columns >= 1 && p->columns <= 0x7fffffffll && p->inner >= 1; }
constexpr int MAX_ROW_BLOCKS = 2048;
unsigned row_blocks(long long rows) { return (unsigned)((rows + ROWS_PER_BLOCK - 1) / ROWS_PER_BLOCK); }

}  // namespace
}  // namespace learner
}  // namespace pgamd

using namespace pgamd::learner;

extern "C" {

LIBENV_API long long procgen_amd_rows_workspace(long long rows, long long columns) { return MAX_COUNT_BLOCKS * (long long)sizeof(long long) + MAX_ROW_BLOCKS * 4ll * (long long)sizeof(double); }

LIBENV_API int procgen_amd_action_logprobs(const struct procgen_amd_rows *p, float *logp, float *entropy, float *lse, int device, void *stream) {
    if (!rows_ok(p) || p->rows > 0x7fffffffll) return -1;
    if (p->rows == 0) return 0;
    if (!p->logits || !p->actions || !logp || !entropy) return -1;
    OnDevice on(device);
    if (on.err != hipSuccess) return (int)on.err;
    return by_dtype(p->dtype, [&](auto e) {
        action_logprobs<decltype(e)><<<row_blocks(p->rows), 256, 0, (hipStream_t)stream>>>(*p, logp, entropy, lse);
        return launched();
    });
}

LIBENV_API int procgen_amd_action_logprobs_backward(const struct procgen_amd_rows *p, const float *lse, const float *entropy, const float *d_logp, const float *d_entropy, int device, void *stream) {
    if (!rows_ok(p) || p->rows > 0x7fffffffll) return -1;
    if (p->rows == 0) return 0;
    if (!p->logits || !p->actions || !p->d_logits || !lse || !entropy) return -1;
    OnDevice on(device);
    if (on.err != hipSuccess) return (int)on.err;
    return by_dtype(p->dtype, [&](auto e) {
        action_logprobs_backward<decltype(e)><<<row_blocks(p->rows), 256, 0, (hipStream_t)stream>>>(*p, lse, entropy, d_logp, d_entropy);
        return launched();
    });
}

LIBENV_API int procgen_amd_policy_loss(const struct procgen_amd_rows *p, const struct procgen_amd_policy *q, int device, void *stream) {
    if (!rows_ok(p) || !q || p->rows > 0x7fffffffll || (q->ref_logits && q->ref_logprobs) || !p->workspace || !q->loss != !q->stats) return -1;
    if (p->rows > 0 && (!p->logits || !p->actions || !q->old_logprobs || !q->adv)) return -1;
    OnDevice on(device);
    if (on.err != hipSuccess) return (int)on.err;
    long long *counts = q->valid ? (long long *)p->workspace : nullptr;
    double *partial = (double *)((long long *)p->workspace + MAX_COUNT_BLOCKS);
    int count_blocks = 0, blocks = 0, err = 0;
    if (p->rows > 0) {
        if (counts) {
            count_blocks = (int)std::min<long long>(MAX_COUNT_BLOCKS, (p->rows + 4095) / 4096);
            count_valid<<<count_blocks, 256, 0, (hipStream_t)stream>>>(q->valid, p->rows, counts);
            if ((err = launched())) return err;
        }
        blocks = (int)std::min<long long>(MAX_ROW_BLOCKS, row_blocks(p->rows));
        err = by_dtype(p->dtype, [&](auto e) {
            if (q->ref_logits) policy_rows<decltype(e), true><<<blocks, 256, 0, (hipStream_t)stream>>>(*p, *q, counts, count_blocks, q->loss ? partial : nullptr);
            else policy_rows<decltype(e), false><<<blocks, 256, 0, (hipStream_t)stream>>>(*p, *q, counts, count_blocks, q->loss ? partial : nullptr);
            return launched();
        });
        if (err) return err;
    }
    if (!q->loss) return 0;
    policy_means<<<1, 256, 0, (hipStream_t)stream>>>(*q, p->rows, counts, count_blocks, partial, blocks);
    return launched();
}

}  // extern "C"
