// learner_rows.hip -- rows of logits, one column per action: log-probabilities and entropy of the actions taken (forward, backward) and the clipped
// policy loss with its gradient.
//
// With m = max l, e[j] = exp(l[j] - m), s = sum e:  p[j] = e[j] / s,  log p[j] = (l[j] - m) - log s,  H = log s - (sum e (l - m)) / s, and against a
// reference row r (m', s' alike)  KL = (sum e ((l - m) - (r - m'))) / s + log(s' / s): every term is of the size of the differences, so nothing of
// the size of the logits cancels.  The gradients of all three operators have one form,
//     dl[j] = pick * (1[j = a] - p[j]) + p[j] * (kl * (log p[j] - log q[j] - KL) + ent * (log p[j] + H))
//           = e[j] * (cd * (l[j] - m) + cq * (r[j] - m') + c0)  (+ pick at a)
// with three coefficients of the row: an exponential, two FMAs and a product a column.
// Partial sums of a row are taken against the largest value their lane or wave has seen and rescaled when they meet (Stats::join), so a row is read once.
//
// Bound by memory: a column costs some 20 operations for 4 to 12 bytes.  Three kernels by the number of columns, each reading and writing a row once
// and 16 bytes a lane:
//   up to 64      a wave takes 64 rows through LDS, a lane per row: no reduction over lanes, coalesced although a row is no multiple of anything
//   more          a group of 16, 64, 256 or 1024 lanes per row keeps the row in its registers between the sums and the gradient
//   very long     the same group in batches; the gradient goes through them backwards, so the last is still in registers and the others in cache
#include "learner.h"

#include <algorithm>

namespace pgamd {
namespace learner {
namespace {

constexpr int BLOCK = 256;
constexpr int MAX_COUNT_BLOCKS = 256;
constexpr int CUS = 256;
constexpr int MAX_BLOCKS = 8 * CUS;

__device__ inline long long action_of(const procgen_amd_rows &p, long long r) {
    return p.actions_are_64_bit ? ((const long long *)p.actions)[r] : (long long)((const int *)p.actions)[r];
}
__device__ inline long long row_offset(const procgen_amd_rows &p, long long r, long long outer, long long inner) {
    return p.inner == 1 ? r * outer : (r / p.inner) * outer + (r % p.inner) * inner;
}

// a difference whose exponential is 0 in 32 bits, as a number that a zero can be multiplied with
__device__ inline float floor_of(float d) { return fmaxf(d, -1000.f); }

// sums over the columns seen so far.  m = -inf: none that is finite; s is then 0, or NaN where a NaN was among them
template <bool REF>
struct Stats {
    float m = -INFINITY, s = 0.f, w = 0.f;   // max, sum e, sum e (l - m)
    float m2 = -INFINITY, s2 = 0.f, u = 0.f; // of the reference row, and sum e ((l - m) - (r - m2))
    __device__ static float safe(float m) { return m == -INFINITY ? 0.f : m; }
    __device__ void put(float *to) const {
        to[0] = m, to[1] = s, to[2] = w;
        if (REF) to[3] = m2, to[4] = s2, to[5] = u;
    }
    __device__ void get(const float *from) {
        m = from[0], s = from[1], w = from[2];
        if (REF) m2 = from[3], s2 = from[4], u = from[5];
    }
    __device__ bool empty() const { return m == -INFINITY && s == 0.f; }
    // the same sums against larger maxima
    __device__ void rescale(float to, float to2) {
        const float d = m == -INFINITY ? 0.f : m - to, c = __expf(d), d2 = !REF || m2 == -INFINITY ? 0.f : m2 - to2;
        if (REF) {
            u = c == 0.f ? 0.f : c * (u + s * (d - d2));  // sums that vanish against the new maximum, far as it may be (s d overflows), are zero
            s2 *= __expf(d2);
            m2 = to2;
        }
        w = c == 0.f ? 0.f : c * (w + s * d);
        s *= c;
        m = to;
    }
    __device__ void add(float l, float r) {  // against maxima that cover them
        const float d = l - safe(m), e = __expf(d), f = floor_of(d);
        s += e;
        w = fmaf(e, f, w);
        if (REF) {
            const float q = r - safe(m2);
            s2 += __expf(q);
            u = fmaf(e, e == 0.f ? 0.f : f - q, u);
        }
    }
    // over `width` neighbouring lanes, all of which get the same bits
    template <int WIDTH>
    __device__ void join() {
        float to = m, to2 = m2;
        for (int d = WIDTH / 2; d > 0; d >>= 1) {
            to = fmaxf(to, __shfl_xor(to, d, WAVE));
            if (REF) to2 = fmaxf(to2, __shfl_xor(to2, d, WAVE));
        }
        rescale(to, to2);
        for (int d = WIDTH / 2; d > 0; d >>= 1) {
            s += __shfl_xor(s, d, WAVE);
            w += __shfl_xor(w, d, WAVE);
            if (REF) {
                s2 += __shfl_xor(s2, d, WAVE);
                u += __shfl_xor(u, d, WAVE);
            }
        }
    }
};

// what the rows add up to, and the gradient's coefficients of one row
struct Sums {
    double policy = 0, kl = 0, entropy = 0, clipped = 0;
};
struct Coef {
    float m, m2, cd, cq, c0, pick;
    // from the formula's numbers, all of them times `scale`; without a known action everything is NaN
    __device__ void set(bool known, float inv_s, float log_s, float log_s2, float H, float KL, float choice, float kl, float ent, float scale) {
        cd = (ent + kl) * inv_s * scale;
        cq = -kl * inv_s * scale;
        c0 = known ? (ent * (H - log_s) + (kl != 0.f ? kl * ((log_s2 - log_s) - KL) : 0.f) - choice) * inv_s * scale : NAN;
        pick = choice * scale;
    }
    template <bool REF>
    __device__ float gradient(float l, float r) const {
        const float d = l - m, e = __expf(d);
        float f = fmaf(cd, floor_of(d), c0);
        if (REF) f = fmaf(cq, e == 0.f ? 0.f : r - m2, f);
        return e * f;
    }
};

// Each operator's rows: what it fetches for a row besides its logits, whether it wants the row at all, what it makes of the row's sums.  finish() is
// called once per row by one lane at least, with `first` set in exactly one; it returns whether the row's gradient is anything but zero.
struct Logprobs {
    static constexpr bool GRADIENT = false, SUMS = false;
    __device__ bool done() const { return false; }
    float *logp, *entropy, *lse;
    struct In {};
    __device__ void begin(const procgen_amd_rows &) {}
    __device__ In fetch(long long) const { return In(); }
    __device__ bool wanted(const In &) const { return true; }
    template <bool REF>
    __device__ bool finish(long long r, const In &, const Stats<REF> &x, bool known, float l, bool first, Coef &, Sums &) const {
        if (!first) return false;
        const float log_s = logf(x.s), m = Stats<REF>::safe(x.m);
        logp[r] = !known ? NAN : x.empty() ? -INFINITY : (l - m) - log_s;
        entropy[r] = x.empty() ? 0.f : log_s - x.w / x.s;
        if (lse) lse[r] = x.empty() ? -INFINITY : m + log_s;
        return false;
    }
};

struct LogprobsBackward {  // of rows short enough to sum up again
    static constexpr bool GRADIENT = true, SUMS = false;
    __device__ bool done() const { return false; }
    const float *d_logp, *d_entropy;
    struct In {
        float d_logp, d_entropy;
    };
    __device__ void begin(const procgen_amd_rows &) {}
    __device__ In fetch(long long r) const { return {d_logp ? d_logp[r] : 0.f, d_entropy ? d_entropy[r] : 0.f}; }
    __device__ bool wanted(const In &in) const { return in.d_logp != 0.f || in.d_entropy != 0.f; }
    template <bool REF>
    __device__ bool finish(long long, const In &in, const Stats<REF> &x, bool known, float, bool, Coef &c, Sums &) const {
        if (x.empty()) return false;
        const float log_s = logf(x.s), inv_s = 1.f / x.s;
        c.m = Stats<REF>::safe(x.m);
        c.set(known, inv_s, log_s, 0.f, log_s - x.w * inv_s, 0.f, in.d_logp, 0.f, -in.d_entropy, 1.f);
        return true;
    }
};

struct Policy {
    static constexpr bool GRADIENT = true, SUMS = true;
    __device__ bool done() const { return (q.resume & 2) && *q.scale == 1.f; }  // the gradient that is there is the one that is wanted
    procgen_amd_policy q;
    const long long *counts;
    int count_blocks;
    long long n;
    float scale;
    __device__ void begin(const procgen_amd_rows &p) {
        n = p.rows;
        if (counts) {
            n = 0;
            for (int i = threadIdx.x % WAVE; i < count_blocks; i += WAVE) n += counts[i];
            n = wave_reduce(n, Sum());
        }
        scale = (q.scale ? *q.scale : 1.f) * (n > 0 ? (float)(1.0 / (double)n) : 0.f);
    }
    struct In {
        float old, adv, ref;
        uint8_t valid;
    };
    __device__ In fetch(long long r) const { return {q.old_logprobs[r], q.adv[r], q.ref_logprobs ? q.ref_logprobs[r] : 0.f, q.valid ? q.valid[r] : (uint8_t)1}; }
    __device__ bool wanted(const In &in) const { return in.valid; }
    template <bool REF>
    __device__ bool finish(long long, const In &in, const Stats<REF> &x, bool known, float l, bool first, Coef &c, Sums &sums) const {
        if (x.empty()) return false;
        c.m = Stats<REF>::safe(x.m);
        const float log_s = logf(x.s), inv_s = 1.f / x.s, H = log_s - x.w * inv_s, logp = known ? (l - c.m) - log_s : NAN;
        const float ratio = __expf(logp - in.old), adv = in.adv, lo = 1.f - q.clip_low, hi = 1.f + q.clip_high;
        const float held = (ratio < lo ? lo : ratio > hi ? hi : ratio) * adv, plain = ratio * adv;
        const bool out = plain > held;  // the clipped side is the smaller one and its gradient is zero; never where something is NaN
        float pick = out ? 0.f : -plain, KL = 0.f, log_s2 = 0.f;
        if (REF) {
            c.m2 = Stats<REF>::safe(x.m2);
            log_s2 = logf(x.s2);
            KL = x.s2 == 0.f ? INFINITY : x.u * inv_s + logf(x.s2 * inv_s);
        } else if (q.ref_logprobs) {
            const float d = in.ref - logp, f = expm1f(d);
            KL = f - d;
            pick -= q.kl_coef * f;
        }
        if (first) {
            sums.policy -= out ? held : plain;
            sums.kl += KL;
            sums.entropy += H;
            sums.clipped += ratio < lo || ratio > hi ? 1.0 : 0.0;
        }
        c.set(known, inv_s, log_s, log_s2, H, KL, pick, REF ? q.kl_coef : 0.f, q.entropy_coef, scale);
        return true;
    }
};

// the block's sums, in a fixed order
__device__ inline void put_sums(Sums x, double *partial) {
    __shared__ double part[BLOCK * 4 / WAVE][4];  // 1024 lanes at the most
    double v[4] = {x.policy, x.kl, x.entropy, x.clipped};
    for (int k = 0; k < 4; k++) v[k] = wave_reduce(v[k], Sum());
    __syncthreads();
    if (threadIdx.x % WAVE == 0)
        for (int k = 0; k < 4; k++) part[threadIdx.x / WAVE][k] = v[k];
    __syncthreads();
    if (threadIdx.x < 4) {
        double y = 0;
        for (unsigned w = 0; w < blockDim.x / WAVE; w++) y += part[w][threadIdx.x];
        partial[(long long)blockIdx.x * 4 + threadIdx.x] = y;
    }
}

template <class E>
struct Chunk {
    static constexpr int N = 16 / sizeof(typename E::T);
    typename E::T x[N];
    // forgets what the compiler has made of the values: they are widened again where they are used next, and not held in 32 bits in between
    __device__ void forget() {
        uint32_t w[4];
        __builtin_memcpy(w, x, 16);
        asm volatile("" : "+v"(w[0]), "+v"(w[1]), "+v"(w[2]), "+v"(w[3]));
        __builtin_memcpy(x, w, 16);
    }
    __device__ void load(const typename E::T *p) { __builtin_memcpy(x, p, 16); }  // from memory, whatever the alignment
    __device__ void store(typename E::T *p) const { __builtin_memcpy(p, x, 16); }
    __device__ void load_aligned(const typename E::T *p) { __builtin_memcpy(x, __builtin_assume_aligned(p, 16), 16); }  // from LDS
    __device__ void store_aligned(typename E::T *p) const { __builtin_memcpy(__builtin_assume_aligned(p, 16), x, 16); }
};

// ---- up to 64 columns: a lane per row -------------------------------------------------------------------------------------------------------------

// 64 rows on their way from memory to LDS (`rows` of them exist).  Contiguous rows go 16 bytes a lane and, where they are few registers, are fetched
// while the 64 before them are worked on; others go element by element.
template <class E, int MOST>
struct Tile {
    typedef typename E::T T;
    static constexpr int N = Chunk<E>::N, CHUNKS = MOST * (int)sizeof(T) / 16;  // 64 rows of MOST columns: so many 16 bytes a lane
    static constexpr bool AHEAD = CHUNKS <= 4;
    typedef uint32_t Bits __attribute__((ext_vector_type(4)));
    Bits c[AHEAD ? CHUNKS : 1];
    __device__ void fetch(const procgen_amd_rows &p, const void *from, long long outer, long long r0, int rows, int lane) {
        if (!AHEAD || p.inner != 1 || outer != p.columns) return;
        const int n = rows * (int)p.columns;
        const T *const src = (const T *)from + r0 * p.columns;
#pragma unroll
        for (int i = 0; i < (AHEAD ? CHUNKS : 0); i++) {
            const int at = (i * WAVE + lane) * N;
            if (at + N <= n) __builtin_memcpy(&c[i], src + at, 16);
        }
    }
    __device__ void put(T *lds, const procgen_amd_rows &p, const void *from, long long outer, long long inner, long long r0, int rows, int lane) const {
        const int columns = (int)p.columns, n = rows * columns;
        if (p.inner == 1 && outer == columns) {
            const T *const src = (const T *)from + r0 * columns;
            if (AHEAD) {
#pragma unroll
                for (int i = 0; i < (AHEAD ? CHUNKS : 0); i++) {
                    const int at = (i * WAVE + lane) * N;
                    if (at + N <= n) *(Bits *)(lds + at) = c[i];
                }
            } else {
                for (int at = lane * N; at + N <= n; at += WAVE * N) {
                    Chunk<E> k;
                    k.load(src + at);
                    k.store_aligned(lds + at);
                }
            }
            if (n / N * N + lane < n) lds[n / N * N + lane] = src[n / N * N + lane];
        } else {
            for (int i = lane; i < n; i += WAVE) {
                const int r = i / columns;
                lds[i] = ((const T *)from)[row_offset(p, r0 + r, outer, inner) + (i - r * columns)];
            }
        }
    }
};
__device__ inline void lds_settled() {  // a wave's own LDS is written and read in order; this holds the compiler to it
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// blocks of four waves that a compute unit holds: by registers (three, or four with a reference, for each of MOST columns) and by LDS
template <class E, int MOST, bool REF>
constexpr int short_residents() {
    return MOST <= 8 ? (REF ? 4 : 6) : MOST <= 16 ? (REF ? 3 : sizeof(typename E::T) == 4 ? 4 : 5) : MOST <= 32 ? (REF ? 2 : 3) : REF ? 1 : 2;
}

template <class E, int MOST, bool REF, class Op>
__global__ __launch_bounds__(BLOCK, (short_residents<E, MOST, REF>())) void short_rows(procgen_amd_rows p, Op op, const void *ref, long long ref_outer, long long ref_inner, double *partial) {
    typedef typename E::T T;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), columns = (int)p.columns;
    const int bytes = (WAVE * columns * (int)sizeof(T) + 15) & ~15;
    T *const tile = (T *)(lds + (size_t)wave * bytes * (REF ? 2 : 1)), *const tile2 = (T *)((char *)tile + bytes);
    if (op.done()) return;
    op.begin(p);
    Sums sums;
    const long long step = (long long)gridDim.x * (BLOCK / WAVE) * WAVE;
    Tile<E, MOST> next;
    Tile<E, REF ? MOST : 8> next2;
    typename Op::In next_in;
    long long next_a = 0;
    auto fetch = [&](long long r0) {
        const int rows = (int)min((long long)WAVE, p.rows - r0);
        const long long r = r0 + min(lane, rows - 1);
        next_in = op.fetch(r);
        next_a = action_of(p, r);
        next.fetch(p, p.logits, p.outer_stride, r0, rows, lane);
        if (REF) next2.fetch(p, ref, ref_outer, r0, rows, lane);
    };
    long long r0 = ((long long)blockIdx.x * (BLOCK / WAVE) + wave) * WAVE;
    if (r0 < p.rows) fetch(r0);
    for (; r0 < p.rows; r0 += step) {
        const int rows = (int)min((long long)WAVE, p.rows - r0);
        const bool mine = lane < rows;
        const long long r = mine ? r0 + lane : r0, a = next_a;
        const typename Op::In in = next_in;
        const bool wanted = mine && op.wanted(in);
        next.put(tile, p, p.logits, p.outer_stride, p.inner_stride, r0, rows, lane);
        if (REF) next2.put(tile2, p, ref, ref_outer, ref_inner, r0, rows, lane);
        lds_settled();
        if (r0 + step < p.rows) fetch(r0 + step);
        T *const row = tile + lane * columns;
        const T *const row2 = tile2 + lane * columns;
        bool some = false;
        Coef c;
        if (wanted) {
            // more than MOST / 2 columns, the others -inf; l and l2 become the differences to the maxima, e their exponentials
            float l[MOST], e[MOST], l2[REF ? MOST : 1];
            Stats<REF> x;
#pragma unroll
            for (int j = 0; j < MOST; j++) {
                const bool real = MOST > 8 && j <= MOST / 2 ? true : j < columns;
                l[j] = real ? (float)row[j] : -INFINITY;
                x.m = fmaxf(x.m, l[j]);
                if (REF) {
                    l2[j] = real ? (float)row2[j] : -INFINITY;
                    x.m2 = fmaxf(x.m2, l2[j]);
                }
            }
            const float m = Stats<REF>::safe(x.m), m2 = Stats<REF>::safe(x.m2);
#pragma unroll
            for (int j = 0; j < MOST; j++) {
                const float d = l[j] - m;
                e[j] = __expf(d);
                l[j] = floor_of(d);
                x.s += e[j];
                x.w = fmaf(e[j], l[j], x.w);
                if (REF) {
                    const float q = l2[j] - m2;
                    x.s2 += __expf(q);
                    l2[j] = e[j] == 0.f ? 0.f : q;
                    x.u = fmaf(e[j], l[j] - l2[j], x.u);
                }
            }
            const bool known = a >= 0 && a < columns;
            some = op.template finish<REF>(r, in, x, known, known ? (float)row[a] : 0.f, true, c, sums);
            if (Op::GRADIENT && some && p.d_logits) {
                const float taken = known ? (float)row[a] : 0.f, taken2 = REF && known ? (float)row2[a] : 0.f;
#pragma unroll
                for (int j = 0; j < MOST; j++) {
                    float f = fmaf(c.cd, l[j], c.c0);
                    if (REF) f = fmaf(c.cq, l2[j], f);
                    if ((MOST > 8 && j <= MOST / 2) || j < columns) row[j] = (T)(e[j] * f);
                }
                if (known) row[a] = (T)(c.gradient<REF>(taken, taken2) + c.pick);
            }
        }
        if (Op::GRADIENT && p.d_logits) {
            if (!some)
                for (int j = 0; j < columns; j++) row[j] = (T)0.f;
            lds_settled();
            T *const out = (T *)p.d_logits + r0 * columns;
            const int n = rows * columns;
            constexpr int N = Chunk<E>::N;
            for (int i = lane * N; i < n; i += WAVE * N) {
                if (i + N <= n) {
                    Chunk<E> k;
                    k.load_aligned(tile + i);
                    k.store(out + i);
                } else {
                    for (int k = i; k < n; k++) out[k] = tile[k];
                }
            }
            lds_settled();
        }
    }
    if (Op::SUMS && partial) put_sums(sums, partial);
}

// ---- more columns: a group of G lanes per row -----------------------------------------------------------------------------------------------------

template <class E, int G, int CH, bool REF, class Op>
__global__ __launch_bounds__(G > BLOCK ? G : BLOCK) void long_rows(procgen_amd_rows p, Op op, const void *ref, long long ref_outer, long long ref_inner, double *partial) {
    typedef typename E::T T;
    constexpr int N = Chunk<E>::N, THREADS = G > BLOCK ? G : BLOCK, PER_BLOCK = THREADS / G, SPAN = G * CH * N;  // columns of a batch
    const int g = threadIdx.x % G, lane = threadIdx.x % WAVE;
    __shared__ float wave_stats[2][G > WAVE ? G / WAVE : 1][6];
    if (op.done()) return;
    op.begin(p);
    Sums sums;
    const int columns = (int)p.columns, batches = (columns + SPAN - 1) / SPAN;
    int odd = 0;
    for (long long r = (long long)blockIdx.x * PER_BLOCK + threadIdx.x / G; r < p.rows; r += (long long)gridDim.x * PER_BLOCK) {
        const T *const row = (const T *)p.logits + row_offset(p, r, p.outer_stride, p.inner_stride);
        const T *const row2 = REF ? (const T *)ref + row_offset(p, r, ref_outer, ref_inner) : nullptr;
        T *const out = Op::GRADIENT && p.d_logits ? (T *)p.d_logits + r * p.columns : nullptr;
        bool some = false;
        Chunk<E> l[CH], l2[REF ? CH : 1];
        // Columns [at(b, i), + N) are chunk i of batch b.  The last one of a row reaches back so that it ends with the row: what it shares with its
        // neighbour counts as -inf here and is not written.  Chunks behind the row are all -inf.
        auto at = [&](int b, int i) { return b * SPAN + (i * G + g) * N; };
        auto load = [&](int b) {
#pragma unroll
            for (int i = 0; i < CH; i++) {
                const int j = min(at(b, i), columns - N);
                l[i].load(row + j);
                if (REF) l2[i].load(row2 + j);
            }
#pragma unroll
            for (int i = 0; i < CH; i++) {
                const int shared = at(b, i) - (columns - N);
                if (shared > 0)
                    for (int k = 0; k < N; k++)
                        if (k < shared) {
                            l[i].x[k] = (T)-INFINITY;
                            if (REF) l2[i].x[k] = (T)-INFINITY;
                        }
            }
        };
        auto forget = [&] {
            for (int i = 0; i < CH; i++) {
                l[i].forget();
                if (REF) l2[i].forget();
            }
        };
        Coef c;
        long long a = 0;
        const typename Op::In in = op.fetch(r);
        if (op.wanted(in)) {  // the same for the whole group
            a = action_of(p, r);
            const bool known = a >= 0 && a < columns;
            const float taken = (float)row[known ? a : 0];
            Stats<REF> x;
            for (int b = 0; b < batches; b++) {
                load(b);
                float to = x.m, to2 = x.m2;
#pragma unroll
                for (int i = 0; i < CH; i++)
                    for (int k = 0; k < N; k++) {
                        to = fmaxf(to, (float)l[i].x[k]);
                        if (REF) to2 = fmaxf(to2, (float)l2[i].x[k]);
                    }
                x.rescale(to, to2);
                forget();
#pragma unroll
                for (int i = 0; i < CH; i++)
                    for (int k = 0; k < N; k++) x.add((float)l[i].x[k], REF ? (float)l2[i].x[k] : 0.f);
            }
            x.template join<(G < WAVE ? G : WAVE)>();
            if (G > WAVE) {
                if (lane == 0) x.put(wave_stats[odd][threadIdx.x / WAVE]);
                __syncthreads();
                x = Stats<REF>();
                if (lane < G / WAVE) x.get(wave_stats[odd][lane]);
                x.template join<(G > WAVE ? G / WAVE : 1)>();
                // lanes beyond the first G / WAVE hold no wave's sums: they take the first one's
                x.m = __shfl(x.m, 0, WAVE), x.s = __shfl(x.s, 0, WAVE), x.w = __shfl(x.w, 0, WAVE);
                if (REF) x.m2 = __shfl(x.m2, 0, WAVE), x.s2 = __shfl(x.s2, 0, WAVE), x.u = __shfl(x.u, 0, WAVE);
                odd ^= 1;
            }
            some = op.template finish<REF>(r, in, x, known, taken, g == 0, c, sums);
            forget();
        }
        if (!Op::GRADIENT || !out) continue;
        for (int b = batches - 1; b >= 0; b--) {
            if (some && b < batches - 1) load(b);
#pragma unroll
            for (int i = 0; i < CH; i++) {
                const int j = min(at(b, i), columns - N), shared = at(b, i) - j;
                Chunk<E> d;
                for (int k = 0; k < N; k++) d.x[k] = some ? (T)c.gradient<REF>((float)l[i].x[k], REF ? (float)l2[i].x[k] : 0.f) : (T)0.f;
                if (shared == 0) {
                    d.store(out + j);
                } else {
                    for (int k = 0; k < N; k++)
                        if (k >= shared) out[j + k] = d.x[k];
                }
            }
        }
        if (some && a >= 0 && a < columns && (int)(a / N) % G == g)  // by the lane that wrote the column just now
            out[a] = (T)(c.gradient<REF>((float)row[a], REF ? (float)row2[a] : 0.f) + c.pick);
    }
    if (Op::SUMS && partial) put_sums(sums, partial);
}

// the gradient of long rows' log-probabilities: lse and entropy are known, so every column stands for itself
template <class E>
__global__ __launch_bounds__(BLOCK) void logprobs_gradient(procgen_amd_rows p, const float *lse, const float *entropy, const float *d_logp, const float *d_entropy) {
    typedef typename E::T T;
    constexpr int N = Chunk<E>::N;
    const int columns = (int)p.columns;
    const long long j = ((long long)blockIdx.x * BLOCK + threadIdx.x) * N;
    if (j >= columns) return;
    for (long long r = blockIdx.y; r < p.rows; r += gridDim.y) {
        const T *const row = (const T *)p.logits + row_offset(p, r, p.outer_stride, p.inner_stride);
        T *const out = (T *)p.d_logits + r * p.columns;
        const long long a = action_of(p, r);
        const float pick = d_logp ? d_logp[r] : 0.f, ent = d_entropy ? -d_entropy[r] : 0.f, z = lse[r];
        const bool known = a >= 0 && a < columns, some = !(pick == 0.f && ent == 0.f) && z != -INFINITY;
        Coef c;
        c.m = z;
        c.set(known, 1.f, 0.f, 0.f, entropy[r], 0.f, pick, 0.f, ent, 1.f);
        Chunk<E> x;
        const bool whole = j + N <= columns;
        if (whole) {
            x.load(row + j);
        } else {
            for (int k = 0; k < N; k++) x.x[k] = j + k < columns ? row[j + k] : (T)0.f;
        }
        for (int k = 0; k < N; k++) x.x[k] = some ? (T)(c.gradient<false>((float)x.x[k], 0.f) + (j + k == a ? pick : 0.f)) : (T)0.f;
        if (whole) {
            x.store(out + j);
        } else {
            for (int k = 0; k < N; k++)
                if (j + k < columns) out[j + k] = x.x[k];
        }
    }
}

// ---- the mean ------------------------------------------------------------------------------------------------------------------------------------

// how many rows count: one partial sum per block, added up by every wave that needs the number (whole numbers: any order gives the same)
__global__ __launch_bounds__(BLOCK) void count_valid(const uint8_t *valid, long long rows, long long *counts) {
    long long n = 0;
    const long long head = min(rows, (long long)(-(uintptr_t)valid & 15)), wide = (rows - head) / 16;  // bytes before the first aligned 16, and 16s
    const long long i = (long long)blockIdx.x * BLOCK + threadIdx.x, step = (long long)gridDim.x * BLOCK;
    for (long long k = i; k < wide; k += step) {
        const uint4 v = ((const uint4 *)(valid + head))[k];
        const unsigned x[4] = {v.x, v.y, v.z, v.w};
        for (int w = 0; w < 4; w++)
            for (int b = 0; b < 32; b += 8) n += (x[w] >> b & 0xff) != 0;
    }
    for (long long k = i; k < rows - wide * 16; k += step) n += valid[k < head ? k : k + wide * 16] != 0;
    n = wave_reduce(n, Sum());
    __shared__ long long part[BLOCK / WAVE];
    if (threadIdx.x % WAVE == 0) part[threadIdx.x / WAVE] = n;
    __syncthreads();
    if (threadIdx.x == 0) counts[blockIdx.x] = part[0] + part[1] + part[2] + part[3];
}

constexpr int MEANS = 1024;
__global__ __launch_bounds__(MEANS) void policy_means(procgen_amd_policy q, long long rows, const long long *counts, int count_blocks, const double *partial, int blocks) {
    const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE, k = lane % 4;  // four neighbouring lanes: a block's four sums
    double v = 0;
    for (int i = threadIdx.x / 4; i < blocks; i += MEANS / 4) v += partial[(long long)i * 4 + k];
    for (int d = WAVE / 2; d >= 4; d >>= 1) v += __shfl_xor(v, d, WAVE);
    __shared__ double part[MEANS / WAVE][4];
    if (lane < 4) part[wave][lane] = v;
    __syncthreads();
    if (wave) return;
    long long n = rows;
    if (counts) {
        n = 0;
        for (int i = lane; i < count_blocks; i += WAVE) n += counts[i];
        n = wave_reduce(n, Sum());
    }
    double mean[4] = {0, 0, 0, 0};
    for (int i = 0; i < 4 && n > 0; i++) {
        for (int w = 0; w < MEANS / WAVE; w++) mean[i] += part[w][i];
        mean[i] /= (double)n;
    }
    if (lane == 0) *q.loss = (float)(mean[0] + (q.kl_coef != 0.f ? (double)q.kl_coef * mean[1] : 0.0) - (q.entropy_coef != 0.f ? (double)q.entropy_coef * mean[2] : 0.0));
    if (lane < 4) q.stats[lane] = (float)mean[lane];
}

// ---- launches ------------------------------------------------------------------------------------------------------------------------------------

bool rows_ok(const procgen_amd_rows *p) {
    return p && known_dtype(p->dtype) && p->rows >= 0 && p->rows <= 0x7fffff00ll && p->columns >= 1 && p->columns <= 0x7ffffff0ll - (1 << 18) && p->inner >= 1;
}

// one kernel over all rows; returns the blocks it was launched with (the partial sums), or -1 - error
template <class E, bool REF, class Op>
int launch_rows(const procgen_amd_rows &p, const Op &op, const void *ref, long long ref_outer, long long ref_inner, double *partial, hipStream_t stream) {
    int blocks = 0;
    auto grid = [&](int per_block, int most) { return blocks = (int)std::min<long long>(most, (p.rows + per_block - 1) / per_block); };
    constexpr int N = Chunk<E>::N;
    if (p.columns <= 64) {
        const size_t lds = ((WAVE * p.columns * sizeof(typename E::T) + 15) & ~15ull) * (BLOCK / WAVE) * (REF ? 2 : 1);
        if (p.columns <= 8) short_rows<E, 8, REF, Op><<<grid(BLOCK, CUS * short_residents<E, 8, REF>()), BLOCK, lds, stream>>>(p, op, ref, ref_outer, ref_inner, partial);
        else if (p.columns <= 16) short_rows<E, 16, REF, Op><<<grid(BLOCK, CUS * short_residents<E, 16, REF>()), BLOCK, lds, stream>>>(p, op, ref, ref_outer, ref_inner, partial);
        else if (p.columns <= 32) short_rows<E, 32, REF, Op><<<grid(BLOCK, CUS * short_residents<E, 32, REF>()), BLOCK, lds, stream>>>(p, op, ref, ref_outer, ref_inner, partial);
        else short_rows<E, 64, REF, Op><<<grid(BLOCK, CUS * short_residents<E, 64, REF>()), BLOCK, lds, stream>>>(p, op, ref, ref_outer, ref_inner, partial);
    } else if (p.columns <= 16 * 2 * N) {
        long_rows<E, 16, 2, REF, Op><<<grid(BLOCK / 16, MAX_BLOCKS), BLOCK, 0, stream>>>(p, op, ref, ref_outer, ref_inner, partial);
    } else if (p.columns <= 64 * 2 * N) {
        long_rows<E, 64, 2, REF, Op><<<grid(BLOCK / 64, MAX_BLOCKS), BLOCK, 0, stream>>>(p, op, ref, ref_outer, ref_inner, partial);
    } else if (p.columns <= 256 * 4 * N) {
        long_rows<E, 256, 4, REF, Op><<<grid(1, MAX_BLOCKS), BLOCK, 0, stream>>>(p, op, ref, ref_outer, ref_inner, partial);
    } else {
        long_rows<E, 1024, 4, REF, Op><<<grid(1, MAX_BLOCKS / 4), 1024, 0, stream>>>(p, op, ref, ref_outer, ref_inner, partial);
    }
    const int err = launched();
    return err ? -1 - err : blocks;
}

}  // namespace
}  // namespace learner
}  // namespace pgamd

using namespace pgamd::learner;

extern "C" {

LIBENV_API long long procgen_amd_rows_workspace(long long rows, long long columns) { return MAX_COUNT_BLOCKS * (long long)sizeof(long long) + MAX_BLOCKS * 4ll * (long long)sizeof(double); }

LIBENV_API int procgen_amd_action_logprobs(const struct procgen_amd_rows *p, float *logp, float *entropy, float *lse, int device, void *stream) {
    if (!rows_ok(p)) return -1;
    if (p->rows == 0) return 0;
    if (!p->logits || !p->actions || !logp || !entropy) return -1;
    OnDevice on(device);
    if (on.err != hipSuccess) return (int)on.err;
    const int got = by_dtype(p->dtype, [&](auto e) { return launch_rows<decltype(e), false>(*p, Logprobs{logp, entropy, lse}, nullptr, 0, 0, nullptr, (hipStream_t)stream); });
    return got < 0 ? -1 - got : 0;
}

LIBENV_API int procgen_amd_action_logprobs_backward(const struct procgen_amd_rows *p, const float *lse, const float *entropy, const float *d_logp, const float *d_entropy, int device, void *stream) {
    if (!rows_ok(p)) return -1;
    if (p->rows == 0) return 0;
    if (!p->logits || !p->actions || !p->d_logits || !lse || !entropy) return -1;
    OnDevice on(device);
    if (on.err != hipSuccess) return (int)on.err;
    return by_dtype(p->dtype, [&](auto e) {
        typedef decltype(e) E;
        if (p->columns <= 64) {
            const int got = launch_rows<E, false>(*p, LogprobsBackward{d_logp, d_entropy}, nullptr, 0, 0, nullptr, (hipStream_t)stream);
            return got < 0 ? -1 - got : 0;
        }
        const long long chunks = (p->columns + Chunk<E>::N - 1) / Chunk<E>::N;
        const dim3 grid((unsigned)((chunks + BLOCK - 1) / BLOCK), (unsigned)std::min<long long>(p->rows, 65535));
        logprobs_gradient<E><<<grid, BLOCK, 0, (hipStream_t)stream>>>(*p, lse, entropy, d_logp, d_entropy);
        return launched();
    });
}

LIBENV_API long long procgen_amd_capture_id(void *stream) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    unsigned long long id = 0;
    if (hipStreamGetCaptureInfo((hipStream_t)stream, &status, &id) != hipSuccess) {
        (void)hipGetLastError();
        return -1;
    }
    return status == hipStreamCaptureStatusActive ? (long long)id : 0;
}

LIBENV_API int procgen_amd_policy_loss(const struct procgen_amd_rows *p, const struct procgen_amd_policy *q, int device, void *stream) {
    if (!rows_ok(p) || !q || (q->ref_logits && q->ref_logprobs) || !p->workspace || !q->loss != !q->stats || (q->resume && (q->loss || !q->scale || (p->rows > 0 && !p->d_logits)))) return -1;
    if (p->rows > 0 && (!p->logits || !p->actions || !q->old_logprobs || !q->adv)) return -1;
    OnDevice on(device);
    if (on.err != hipSuccess) return (int)on.err;
    long long *counts = q->valid ? (long long *)p->workspace : nullptr;
    double *partial = (double *)((long long *)p->workspace + MAX_COUNT_BLOCKS);
    int count_blocks = 0, blocks = 0;
    if (p->rows > 0) {
        if (counts) {
            count_blocks = (int)std::min<long long>(MAX_COUNT_BLOCKS, (p->rows + 16 * BLOCK - 1) / (16 * BLOCK));
            if (!q->resume) {
                count_valid<<<count_blocks, BLOCK, 0, (hipStream_t)stream>>>(q->valid, p->rows, counts);
                if (int err = launched()) return err;
            }
        }
        blocks = by_dtype(p->dtype, [&](auto e) {
            typedef decltype(e) E;
            const Policy op{*q, counts, count_blocks, 0, 0.f};
            double *to = q->loss ? partial : nullptr;
            if (q->ref_logits) return launch_rows<E, true>(*p, op, q->ref_logits, q->ref_outer_stride, q->ref_inner_stride, to, (hipStream_t)stream);
            return launch_rows<E, false>(*p, op, nullptr, 0, 0, to, (hipStream_t)stream);
        });
        if (blocks < 0) return -1 - blocks;
    }
    if (!q->loss) return 0;
    policy_means<<<1, MEANS, 0, (hipStream_t)stream>>>(*q, p->rows, counts, count_blocks, partial, blocks);
    return launched();
}

}  // extern "C"
