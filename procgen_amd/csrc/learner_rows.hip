// learner_rows.hip -- rows of logits, one column per action: log-probabilities and entropy of the actions taken (forward, backward) and the clipped
// policy loss with its gradient.
//
// With m = max l, x[j] = l[j] - m, e[j] = exp(x[j]), s = sum e:
//     p[j] = e[j] / s,   log p[j] = x[j] - log s,   H = log s - sum e x / s,
// and against a reference row r (y[j] = r[j] - max r, s' alike)  KL = sum e (x - y) / s + log s' - log s: every term is of the size of the differences, so
// nothing of the size of the logits cancels.  The gradients of all three operators have one form,
//     dl[j] = pick * (1[j = a] - p[j]) + p[j] * (kl * (log p[j] - log q[j] - KL) + ent * (log p[j] + H))
//           = e[j] * (cd x[j] + cq y[j] + c0)  (+ pick at a)
// with three coefficients of the row.  The difference comes first and is rounded by itself, at any size of l.  (Taken as one FMA, l log2 e - m log2 e, it
// would be off by half a step of m log2 e, which from |m| of 2^30 on is more than float32's exponents reach.)  A column that is -inf (or too far below
// the maximum) has e = 0 and counts as 0 whatever it is multiplied with: product() is the hardware's multiplication in which zero times anything is zero.
// Partial sums of a row are taken against the largest value their lane or wave has seen and rescaled when they meet (Stats::join), so a row is read once.
//
// Bound by memory: by the counters a bf16 column costs 12 vector instructions for 2 bytes without a gradient, 22 for 4 with one, 41 for 6 beside a reference,
// everything about its row included (a 1 GiB copy reaches 5.1 TB/s on the same card).  By the number of columns:
//   up to 32      a wave takes 64 rows through LDS, a lane per row: no reduction over lanes, coalesced although a row is no multiple of anything
//                 (16 bits without a reference up to 63)
//   up to 10240   a group of 4 to 256 lanes per row, the whole row in their registers between the sums and the gradient (5120 in float32; 4096 and 2048
//                 where the rows are too few to fill the card one a block)
//   more          a block per row, in batches; the gradient goes through them backwards: the last is still in registers, those before it in LDS, and
//                 only what is left is read from memory again
#include "learner.h"

#include <algorithm>
#include <type_traits>

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
    if (p.inner == 1) return r * outer;
    const uint32_t per = (uint32_t)p.inner, group = (uint32_t)r / per;  // rows fit 32 bits
    return group * outer + ((uint32_t)r - group * per) * inner;
}

constexpr float LOG2E = 1.44269504088896340736f;
__device__ inline float exp2_of(float t) { return __builtin_amdgcn_exp2f(t); }
__device__ float multiply_legacy(float, float) __asm("llvm.amdgcn.fmul.legacy");  // v_mul_legacy_f32, which has no builtin function
__device__ inline float product(float e, float x) { return multiply_legacy(e, x); }

__device__ inline float exp_of(float x) { return exp2_of(x * LOG2E); }
// what a row's columns are taken against: its maximum, or 0 where no column is finite
__device__ inline float level_of(float m) { return m == -INFINITY ? 0.f : m; }

// sums over the columns seen so far.  m = -inf: none that is finite; s is then 0, or NaN where a NaN was among them
template <bool REF>
struct Stats {
    float m = -INFINITY, s = 0.f, w = 0.f;   // max, sum e, sum e x
    float m2 = -INFINITY, s2 = 0.f, u = 0.f; // of the reference row, and sum e (x - y)
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
        const float d = m == -INFINITY ? 0.f : m - to, c = exp_of(d), d2 = !REF || m2 == -INFINITY ? 0.f : m2 - to2;
        if (REF) {
            u = product(c, product(s, d - d2) + u);
            s2 *= exp_of(d2);  // a NaN stays one
            m2 = to2;
        }
        w = product(c, product(s, d) + w);
        s *= c;
        m = to;
    }
    // columns against levels that cover them
    __device__ void add(float level, float level2, float l, float r) {
        const float x = l - level, e = exp_of(x);
        s += e;
        w += product(e, x);
        if (REF) {
            const float y = r - level2;
            s2 += exp_of(y);
            u += product(e, x - y);
        }
    }
    // lanes that hold no wave's sums take the first one's
    __device__ void from_first() {
        m = __shfl(m, 0, WAVE), s = __shfl(s, 0, WAVE), w = __shfl(w, 0, WAVE);
        if (REF) m2 = __shfl(m2, 0, WAVE), s2 = __shfl(s2, 0, WAVE), u = __shfl(u, 0, WAVE);
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
// a row's own numbers
template <bool REF>
struct Row {
    float m, log_s, inv_s, H, log_s2, KL;
    __device__ explicit Row(const Stats<REF> &x) {
        m = level_of(x.m);
        inv_s = 1.f / x.s;
        log_s = logf(x.s);
        H = log_s - x.w * inv_s;
        log_s2 = KL = 0.f;
        if (REF) {
            log_s2 = logf(x.s2);
            KL = x.s2 == 0.f ? INFINITY : fmaf(x.u, inv_s, logf(x.s2 * inv_s));
        }
    }
    __device__ float logp(float l) const { return (l - m) - log_s; }
};

// what the rows add up to, and the gradient's coefficients of one row
struct Sums {
    double policy = 0, kl = 0, entropy = 0, clipped = 0;
};
struct Coef {
    float level, level2, cd, cq, c0, pick;
    // from the formula's numbers, all of them times `scale`.  Without a known action, or with a NaN among the logits, everything is NaN.
    template <bool REF>
    __device__ void set(bool known, const Stats<REF> &x, const Row<REF> &row, float choice, float kl, float ent, float scale) {
        level = known && x.s == x.s ? row.m : NAN, level2 = level_of(x.m2);
        const float by = row.inv_s * scale;
        cd = (ent + kl) * by;
        cq = -kl * by;
        c0 = (ent * (row.H - row.log_s) + (REF && kl != 0.f ? kl * ((row.log_s2 - row.log_s) - row.KL) : 0.f) - choice) * by;
        pick = choice * scale;
    }
    __device__ bool nan() const { return level != level; }
    template <bool REF>
    __device__ float gradient(float l, float r) const {
        const float x = l - level;
        float f = fmaf(cd, x, c0);
        if (REF) f += product(cq, r - level2);  // a reference without weight may hold anything
        return product(exp_of(x), f);
    }
};

// Each operator's rows: what it fetches for a row besides its logits, whether it wants the row at all, what it makes of the row's sums.  finish() is
// called once per row by one lane at least, with `first` set in exactly one; it returns whether the row's gradient is anything but zero.
struct Logprobs {
    static constexpr bool GRADIENT = false, LONG = true;
    __device__ bool done() const { return false; }
    float *logp, *entropy;
    procgen_amd_lse *lse;
    struct In {};
    __device__ void begin(const procgen_amd_rows &) {}
    __device__ In fetch(long long) const { return In(); }
    __device__ bool wanted(const In &) const { return true; }
    template <bool REF>
    __device__ bool finish(long long r, const In &, const Stats<REF> &x, bool known, float l, bool first, Coef &, Sums &) const {
        if (!first) return false;
        const Row<REF> row(x);
        logp[r] = !known ? NAN : x.empty() ? -INFINITY : row.logp(l);
        entropy[r] = x.empty() ? 0.f : row.H;
        if (lse) lse[r] = x.empty() ? procgen_amd_lse{-INFINITY, 0.f} : procgen_amd_lse{row.m, row.log_s};
        return false;
    }
};

struct LogprobsBackward {  // of rows short enough to sum up again: 256 chunks, which the 64 lanes of a wave hold
    static constexpr bool GRADIENT = true, LONG = false;
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
        c.set(known, x, Row<REF>(x), in.d_logp, 0.f, -in.d_entropy, 1.f);
        return true;
    }
};

struct Policy {
    static constexpr bool GRADIENT = true, LONG = true;
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
        const Row<REF> row(x);
        const float logp = known ? row.logp(l) : NAN, ratio = __expf(logp - in.old), adv = in.adv, lo = 1.f - q.clip_low, hi = 1.f + q.clip_high;
        const float held = (ratio < lo ? lo : ratio > hi ? hi : ratio) * adv, plain = ratio * adv;
        const bool out = plain > held;  // the clipped side is the smaller one and its gradient is zero; never where something is NaN
        float pick = out ? 0.f : -plain, KL = row.KL;
        if (!REF && q.ref_logprobs) {
            const float d = in.ref - logp, f = expm1f(d);
            KL = f - d;
            pick -= product(q.kl_coef, f);  // without weight it may be infinite
        }
        if (first) {
            sums.policy -= out ? held : plain;
            sums.kl += KL;
            sums.entropy += row.H;
            sums.clipped += ratio < lo || ratio > hi ? 1.0 : 0.0;
        }
        c.set(known, x, row, pick, REF ? q.kl_coef : 0.f, q.entropy_coef, scale);
        return true;
    }
};

// lane 4 w + k of the first wave takes wave w's k-th sum; lanes 0 to 3 (and every fourth after them) return the totals
__device__ inline double sum_of_waves(const double (*part)[4], int waves) {
    const int lane = threadIdx.x;
    double v = lane / 4 < waves ? part[lane / 4][lane % 4] : 0.0;
    for (int d = WAVE / 2; d >= 4; d >>= 1) v += __shfl_xor(v, d, WAVE);
    return v;
}

// the loss and the four means, by one thread
__device__ inline void put_means(const procgen_amd_policy &q, long long n, double *sum) {
    for (int k = 0; k < 4; k++) sum[k] = n > 0 ? sum[k] / (double)n : 0.0;
    *q.loss = (float)(sum[0] + (q.kl_coef != 0.f ? (double)q.kl_coef * sum[1] : 0.0) - (q.entropy_coef != 0.f ? (double)q.entropy_coef * sum[2] : 0.0));
    for (int k = 0; k < 4; k++) q.stats[k] = (float)sum[k];
}

// the block's sums, in a fixed order; the only block of a launch makes the means of them
__device__ inline void put_sums(Sums x, const Policy &op, double *partial) {
    __shared__ double part[BLOCK * 4 / WAVE][4];  // 1024 lanes at the most
    double v[4] = {x.policy, x.kl, x.entropy, x.clipped};
    for (int k = 0; k < 4; k++) v[k] = wave_reduce(v[k], Sum());
    __syncthreads();
    if (threadIdx.x % WAVE == 0)
        for (int k = 0; k < 4; k++) part[threadIdx.x / WAVE][k] = v[k];
    __syncthreads();
    if (threadIdx.x >= WAVE) return;
    const double mine = sum_of_waves(part, blockDim.x / WAVE);
    for (int k = 0; k < 4; k++) v[k] = __shfl(mine, k, WAVE);
    if (threadIdx.x) return;
    if (gridDim.x == 1) put_means(op.q, op.n, v);
    else
        for (int k = 0; k < 4; k++) partial[(long long)blockIdx.x * 4 + k] = v[k];
}
__device__ inline void put_sums(Sums, const Logprobs &, double *) {}
__device__ inline void put_sums(Sums, const LogprobsBackward &, double *) {}

// 16 bytes of a row in registers, as memory holds them
typedef uint32_t Bits __attribute__((ext_vector_type(4)));
template <class E>
struct Chunk {
    typedef typename E::T T;
    static constexpr int N = 16 / sizeof(T);
    Bits w;
    __device__ void load(const T *p) { __builtin_memcpy(&w, p, 16); }  // whatever the alignment
    __device__ void store(T *p) const { __builtin_memcpy(p, &w, 16); }
    __device__ float operator[](int k) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[k]);
        else if constexpr (__is_same(T, __bf16)) return __builtin_bit_cast(float, k % 2 ? w[k / 2] & 0xffff0000u : w[k / 2] << 16);
        else return (float)__builtin_bit_cast(T, (uint16_t)(w[k / 2] >> k % 2 * 16));
    }
    __device__ void set(int d, float x, float y) {  // word d: value d, or values 2 d and 2 d + 1
        if constexpr (sizeof(T) == 4) {
            w[d] = __float_as_uint(x);
        } else {
            typedef T Two __attribute__((ext_vector_type(2)));
            typedef float TwoF __attribute__((ext_vector_type(2)));
            const Two two = __builtin_convertvector((TwoF{x, y}), Two);
            w[d] = __builtin_bit_cast(uint32_t, two);
        }
    }
    __device__ T piece(int k) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[k]);
        else return __builtin_bit_cast(T, (uint16_t)(w[k / 2] >> k % 2 * 16));
    }
    // -inf for the first n values, or the last -n
    __device__ void drop(int n) {
        constexpr uint32_t INF = sizeof(T) == 4 ? 0xff800000u : __is_same(T, __bf16) ? 0xff80u : 0xfc00u;
        auto out = [&](int k) { return n > 0 ? k < n : k >= N + n; };
        for (int d = 0; d < 4; d++) {
            if constexpr (sizeof(T) == 4) {
                if (out(d)) w[d] = INF;
            } else {
                if (out(2 * d)) w[d] = (w[d] & 0xffff0000u) | INF;
                if (out(2 * d + 1)) w[d] = (w[d] & 0xffffu) | INF << 16;
            }
        }
    }
    // forgets what the compiler has made of the values: they are widened again where they are used next, and not held in 32 bits in between
    __device__ void forget() { asm volatile("" : "+v"(w)); }
};

// ---- up to 32 columns, or 63: a lane per row -------------------------------------------------------------------------------------------------------------

// 64 rows on their way from memory to LDS (`rows` of them exist), fetched while the 64 before them are worked on.  Contiguous rows are one array of 16
// bytes a lane.  Rows apart from each other (APART, kernels of their own: one for both would spill registers) are cut into such pieces each, the last moved
// back to end with its row; rows under 16 bytes go element by element.  Loss and gradient of 2 097 152 x 15
// out of rows of 16: bf16 51 us (element by element 73), with a reference 68 (171), float32 52 (105); of 31 out of 32 bf16 90 (214), float32 108 (367).
//
// Rows of 16 or 32 float32 are 64 or 128 bytes: lanes that all read one column of theirs would meet in four or two of the 64 banks.  With TURN a row's
// chunks are swapped by the row's place, and 16 lanes that read a chunk each go over every bank once.  Loss and gradient of 4 194 304 x 16 float32: 107
// us instead of 150, with a reference 160 instead of 204, of the log-probabilities 103 instead of 143.
template <class E, int MOST, bool TURN>
__device__ inline int place(int i) {  // in LDS, of element i of the 64 rows
    return TURN ? i ^ (i / MOST * MOST / 64 % (MOST / Chunk<E>::N) * Chunk<E>::N) : i;
}
template <class E, int MOST, bool TURN, bool APART>
struct Tile {
    typedef typename E::T T;
    static constexpr int N = Chunk<E>::N, CHUNKS = MOST * (int)sizeof(T) / 16;  // 64 rows of MOST columns: so many 16 bytes a lane
    Chunk<E> c[CHUNKS];
    struct Piece {  // of a row that is not followed by the next
        int row, column;
        __device__ Piece(int i, int lane, int columns) {
            const uint32_t pieces = (columns + N - 1) / N, at = i * WAVE + lane;
            row = at * (65536 / pieces + 1) >> 16;  // at / pieces: at < 512, pieces <= 8
            column = min((int)(at - row * pieces) * N, columns - N);
        }
    };
    __device__ void fetch(const procgen_amd_rows &p, const void *from, long long outer, long long inner, long long r0, int rows, int lane) {
        const int columns = (int)p.columns, n = rows * columns;
        const T *const src = (const T *)from + r0 * columns;
        if (APART && columns < N) return;
#pragma unroll
        for (int i = 0; i < CHUNKS; i++) {
            if constexpr (APART) {
                const Piece q(i, lane, columns);
                if (q.row < rows) c[i].load((const T *)from + row_offset(p, r0 + q.row, outer, inner) + q.column);
            } else {
                const int at = (i * WAVE + lane) * N;
                if (at + N <= n) c[i].load(src + at);
            }
        }
    }
    __device__ void put(T *lds, const procgen_amd_rows &p, const void *from, long long outer, long long inner, long long r0, int rows, int lane) const {
        const int columns = (int)p.columns, n = rows * columns;
        if (APART && columns < N) {
            for (int i = lane; i < n; i += WAVE) {
                const int r = i / columns;
                lds[place<E, MOST, TURN>(i)] = ((const T *)from)[row_offset(p, r0 + r, outer, inner) + (i - r * columns)];
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < CHUNKS; i++) {
            if constexpr (APART) {
                const Piece q(i, lane, columns);
                if (q.row < rows)
                    for (int k = 0; k < N; k++) lds[place<E, MOST, TURN>(q.row * columns + q.column + k)] = c[i].piece(k);
            } else {
                const int at = (i * WAVE + lane) * N;
                if (at + N <= n) *(Bits *)(lds + place<E, MOST, TURN>(at)) = c[i].w;
            }
        }
        if (!APART && n / N * N + lane < n) lds[place<E, MOST, TURN>(n / N * N + lane)] = ((const T *)from)[r0 * columns + n / N * N + lane];
    }
};
__device__ inline void lds_settled() {  // a wave's own LDS is written and read in order; this holds the compiler to it
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// bytes of LDS that 64 rows take, with slack for the columns that the last row does not have
template <class E, int MOST>
__host__ __device__ constexpr int short_tile(int columns) {
    return ((WAVE * columns * (int)sizeof(typename E::T) + 15) & ~15) + MOST * (int)sizeof(typename E::T);
}
// blocks of four waves that a compute unit holds: by registers (three, or four with a reference, for each of MOST columns) and by LDS.  Loss of 64 M bf16 (32 M float32)
// logits in us with one block less : these : one more, which spills:
//   columns          4                8               15               24               31              48              63
//   bf16       155:143:140       87:83:83       89:77:124        76:63:124        92:74:114      113:73:111      115:76:142
//     reference 256:225:205   140:124:114     149:120:166      181:110:124      176:114:203
//   float32      93:87:84         69:67:69        66:57:85         71:61:77         88:62:65
//     reference 145:122:119      101:92:94       93:85:152       125:94:156      113:88:278
// (16 float32 with a reference, two blocks: 134:89:86.)  The gradient of log-probabilities alone would take one more up to 16 columns (15 bf16 67:62, 31 float32 54:50).
template <class E, int MOST, bool REF, bool TURN = false>
constexpr int short_residents() {
    return MOST <= 8 ? (REF ? 4 : 6) : MOST <= 16 ? (REF ? (TURN ? 2 : 3) : sizeof(typename E::T) == 4 ? 4 : 5) : MOST <= 24 ? (REF ? 2 : sizeof(typename E::T) == 4 ? 3 : 4) : MOST > 32 || REF || sizeof(typename E::T) == 4 ? 2 : 3;
}

// Loss and gradient of 4 194 304 x 15 bf16: 65 to 74 us, 306 MB, 4.1 to 4.7 TB/s; without fetching ahead 98, with the register limit of six blocks (and
// spills) 93, of four 78.  What is left is the issue of instructions: some 340 vector and 190 scalar ones for 64 rows.
template <class E, int MOST, bool REF, class Op, bool TURN, bool APART>
__global__ __launch_bounds__(BLOCK, (short_residents<E, MOST, REF, TURN>())) void short_rows(procgen_amd_rows p, Op op, const void *ref, long long ref_outer, long long ref_inner, double *partial) {
    typedef typename E::T T;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), columns = (int)p.columns;
    const int bytes = short_tile<E, MOST>(columns);
    T *const tile = (T *)(lds + (size_t)wave * bytes * (REF ? 2 : 1)), *const tile2 = (T *)((char *)tile + bytes);
    if (op.done()) return;
    op.begin(p);
    Sums sums;
    const long long step = (long long)gridDim.x * (BLOCK / WAVE) * WAVE;
    Tile<E, MOST, TURN, APART> next;
    Tile<E, REF ? MOST : 8, REF && TURN, APART> next2;
    typename Op::In next_in;
    int next_a = -1;  // -1: not one of the columns
    auto fetch = [&](long long r0) {
        const int rows = (int)min((long long)WAVE, p.rows - r0);
        const long long r = r0 + min(lane, rows - 1);
        next_in = op.fetch(r);
        const long long a = action_of(p, r);
        next_a = a >= 0 && a < columns ? (int)a : -1;
        next.fetch(p, p.logits, p.outer_stride, p.inner_stride, r0, rows, lane);
        if (REF) next2.fetch(p, ref, ref_outer, ref_inner, r0, rows, lane);
    };
    long long r0 = ((long long)blockIdx.x * (BLOCK / WAVE) + wave) * WAVE;
    if (r0 < p.rows) fetch(r0);
    for (; r0 < p.rows; r0 += step) {
        const int rows = (int)min((long long)WAVE, p.rows - r0);
        const bool mine = lane < rows;
        const long long r = mine ? r0 + lane : r0;
        const int a = next_a;
        const typename Op::In in = next_in;
        const bool wanted = mine && op.wanted(in);
        next.put(tile, p, p.logits, p.outer_stride, p.inner_stride, r0, rows, lane);
        if (REF) next2.put(tile2, p, ref, ref_outer, ref_inner, r0, rows, lane);
        lds_settled();
        if (r0 + step < p.rows) fetch(r0 + step);
        const int turn = TURN ? place<E, MOST, TURN>(lane * MOST) % MOST : 0;
        T *const row = tile + lane * columns;
        const T *const row2 = tile2 + lane * columns;
        bool some = false;
        Coef c;
        if (wanted) {
            // the columns that a row has not are -inf; l and l2 become x and y
            // reads what a row has not and drops it, which keeps the reads together: loss of 64 M bf16 logits at 9, 15, 16, 24, 32, 63 columns 105, 76, 70, 63, 68, 76 us, with
            // a branch around each of those reads 104, 77, 74, 66, 77, 85
            constexpr bool AGAIN = MOST > 48 || (REF && MOST > 24 && sizeof(T) == 4);  // exponentials are taken again for the gradient: registers for all of them would be spilled
            constexpr int surely = TURN ? MOST : MOST > 32 ? MOST - 16 : MOST > 16 ? MOST - 8 : MOST > 8 ? MOST / 2 : 0;
            float l[MOST], e[MOST], l2[REF ? MOST : 1];
            Stats<REF> x;
#pragma unroll
            for (int j = 0; j < MOST; j++) {
                l[j] = (float)row[j ^ turn];  // of the row behind, or of the tile's slack, where there is no such column
                if (REF) l2[j] = (float)row2[j ^ turn];
            }
#pragma unroll
            for (int j = 0; j < MOST; j++) {
                if (j > surely && j >= columns) l[j] = l2[REF ? j : 0] = -INFINITY;
                x.m = fmaxf(x.m, l[j]);
                if (REF) x.m2 = fmaxf(x.m2, l2[j]);
            }
            const float level = level_of(x.m), level2 = level_of(x.m2);
#pragma unroll
            for (int j = 0; j < MOST; j++) {
                l[j] -= level;
                e[j] = exp_of(l[j]);
                x.s += e[j];
                x.w += product(e[j], l[j]);
                if (REF) {
                    l2[j] -= level2;
                    x.s2 += exp_of(l2[j]);
                    x.u += product(e[j], l[j] - l2[j]);
                }
            }
            const bool known = a >= 0;
            const float taken = known ? (float)row[a ^ turn] : 0.f, taken2 = REF && known ? (float)row2[a ^ turn] : 0.f;
            some = op.template finish<REF>(r, in, x, known, taken, true, c, sums);
            if (Op::GRADIENT && some && p.d_logits) {
#pragma unroll
                for (int j = 0; j < MOST; j++) {
                    if (AGAIN) {
                        asm volatile("" : "+v"(l[j]));
                        e[j] = exp_of(l[j]);
                    }
                    float f = fmaf(c.cd, l[j], c.c0);
                    if (REF) f += product(c.cq, l2[j]);
                    if (j <= surely || j < columns) row[j ^ turn] = (T)product(e[j], f);
                }
                if (known) row[a ^ turn] = (T)(c.gradient<REF>(taken, taken2) + c.pick);
                if (c.nan())
                    for (int j = 0; j < columns; j++) row[j] = (T)NAN;
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
                    k.w = *(const Bits *)(tile + place<E, MOST, TURN>(i));
                    k.store(out + i);
                } else {
                    for (int k = i; k < n; k++) out[k] = tile[place<E, MOST, TURN>(k)];
                }
            }
            lds_settled();
        }
    }
    if (partial) put_sums(sums, op, partial);
}

// ---- more columns: a group of G lanes per row -----------------------------------------------------------------------------------------------------

// Where a row's columns are among the lanes of a group.  Chunk c is the 16 aligned bytes of columns [c N - ahead, + N), whatever the row's own alignment
// (a row at an odd address costs an eighth more time otherwise); lane g has the chunks g, g + G, ...  The first and the last chunk of a row are moved so
// that they end in it: what they share with their neighbour counts as -inf and is not written.  Chunks behind the row are all -inf.
template <class E>
struct Place {
    typedef typename E::T T;
    static constexpr int N = Chunk<E>::N;
    int columns, ahead;
    __device__ Place(const T *row, int columns_) : columns(columns_), ahead((int)((uintptr_t)row / sizeof(T) % N)) {}
    __device__ int wanted(int chunk) const { return chunk * N - ahead; }
    __device__ int column(int chunk) const { return max(0, min(wanted(chunk), columns - N)); }
    __device__ void drop(Chunk<E> &x, int chunk) const {
        const int moved = wanted(chunk) - column(chunk);
        if (moved) x.drop(moved);
    }
    __device__ void put(T *out, int chunk, const Chunk<E> &x) const {
        const int j = wanted(chunk), from = column(chunk);
        if (j >= columns) return;
        if (from == j) {
            x.store(out + j);
        } else {
            for (int k = 0; k < N; k++)
                if (from + k >= j && from + k < j + N) out[from + k] = x.piece(k);
        }
    }
    __device__ int chunk_of(int column) const { return (column + ahead) / N; }
};

// Rows that fit the registers of a group, of lanes inside of a wave or of two or four waves: the next rows are on their way while these are worked on.
// Loss and gradient of 64 M bf16 logits at 64, 512, 1024, 2000 columns: 70, 54, 54, 56 us (3.9 to 5.0 TB/s), with a reference 106, 96, 97, 102.  Three, four
// or five chunks a lane leave at most a quarter of the lanes without columns: at 127, 255, 300, 511, 2047 columns 92, 79, 66, 74, 69 us; with four alone, and
// so up to half of them without, 127, 123, 97, 121, 106.  A group of two or four waves holds 4100, 5000, 8200 columns: 67, 56, 65 us, in batches of a block 113,
// 90, 77; with a reference 123, 107, 122, in batches 232, 188, 148.
template <class E, int G, int CH, bool REF, class Op>
__global__ __launch_bounds__(BLOCK) void group_rows(procgen_amd_rows p, Op op, const void *ref, long long ref_outer, long long ref_inner, double *partial) {
    typedef typename E::T T;
    constexpr int N = Chunk<E>::N, PER = N / 4, PER_BLOCK = BLOCK / G, WAVES = G / WAVE, LANES = WAVES ? WAVE : G;
    const int g = threadIdx.x % G, columns = (int)p.columns;
    __shared__ float wave_stats[2][WAVES > 1 ? BLOCK / WAVE : 1][6];
    int odd = 0;
    if (op.done()) return;
    op.begin(p);
    Sums sums;
    Bits next[CH], next2[REF ? CH : 1];
    typename Op::In next_in;
    int next_a = -1;
    auto row_of = [&](long long r) { return (const T *)p.logits + row_offset(p, r, p.outer_stride, p.inner_stride); };
    auto row2_of = [&](long long r) { return (const T *)ref + row_offset(p, r, ref_outer, ref_inner); };
    auto fetch = [&](long long r) {
        r = min(r, p.rows - 1);
        const T *const row = row_of(r), *const row2 = REF ? row2_of(r) : nullptr;
        const Place<E> at(row, columns);
#pragma unroll
        for (int i = 0; i < CH; i++) {
            const int j = at.column(i * G + g);
            __builtin_memcpy(&next[i], row + j, 16);
            if (REF) __builtin_memcpy(&next2[i], row2 + j, 16);
        }
        next_in = op.fetch(r);
        const long long a = action_of(p, r);
        next_a = a >= 0 && a < columns ? (int)a : -1;
    };
    const long long step = (long long)gridDim.x * PER_BLOCK;
    long long r = (long long)blockIdx.x * PER_BLOCK + threadIdx.x / G;
    fetch(r);
    for (long long first = (long long)blockIdx.x * PER_BLOCK; first < p.rows; first += step, r += step) {
        const bool mine = r < p.rows;
        const long long here = mine ? r : p.rows - 1;
        const T *const row = row_of(here), *const row2 = REF ? row2_of(here) : nullptr;
        const Place<E> at(row, columns);
        Chunk<E> l[CH], l2[REF ? CH : 1];
        const typename Op::In in = next_in;
        const int a = next_a;
        const float taken = (float)row[max(a, 0)], taken2 = REF ? (float)row2[max(a, 0)] : 0.f;
#pragma unroll
        for (int i = 0; i < CH; i++) {
            l[i].w = next[i];
            at.drop(l[i], i * G + g);
            if (REF) {
                l2[i].w = next2[i];
                at.drop(l2[i], i * G + g);
            }
        }
        if (first + step < p.rows) fetch(r + step);
        Stats<REF> x;
        float to = -INFINITY, to2 = -INFINITY;
#pragma unroll
        for (int i = 0; i < CH; i++)
#pragma unroll
            for (int k = 0; k < N; k++) {
                to = fmaxf(to, l[i][k]);
                if (REF) to2 = fmaxf(to2, l2[i][k]);
            }
        for (int d = LANES / 2; d > 0; d >>= 1) {
            to = fmaxf(to, __shfl_xor(to, d, WAVE));
            if (REF) to2 = fmaxf(to2, __shfl_xor(to2, d, WAVE));
        }
        x.m = to, x.m2 = to2;
        const float level = level_of(to), level2 = level_of(to2);
#pragma unroll
        for (int i = 0; i < CH; i++) {
            l[i].forget();
            if (REF) l2[i].forget();
#pragma unroll
            for (int k = 0; k < N; k++) x.add(level, level2, l[i][k], REF ? l2[i][k] : 0.f);
        }
        for (int d = LANES / 2; d > 0; d >>= 1) {
            x.s += __shfl_xor(x.s, d, WAVE);
            x.w += __shfl_xor(x.w, d, WAVE);
            if (REF) {
                x.s2 += __shfl_xor(x.s2, d, WAVE);
                x.u += __shfl_xor(x.u, d, WAVE);
            }
        }
        if constexpr (WAVES > 1) {
            const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
            if (lane == 0) x.put(wave_stats[odd][wave]);
            __syncthreads();
            x = Stats<REF>();
            if (lane < WAVES) x.get(wave_stats[odd][wave / WAVES * WAVES + lane]);
            x.template join<WAVES>();
            x.from_first();
            odd ^= 1;
        }
        Coef c;
        const bool some = mine && op.wanted(in) && op.template finish<REF>(here, in, x, a >= 0, taken, g == 0, c, sums);
        if (!Op::GRADIENT || !p.d_logits || !mine) continue;
        T *const out = (T *)p.d_logits + r * p.columns;
#pragma unroll
        for (int i = 0; i < CH; i++) {
            l[i].forget();
            if (REF) l2[i].forget();
            Chunk<E> d;
            d.w = Bits{0, 0, 0, 0};
            if (some) {
#pragma unroll
                for (int k = 0; k < N; k += PER)
                    d.set(k / PER, c.gradient<REF>(l[i][k], REF ? l2[i][k] : 0.f), PER > 1 ? c.gradient<REF>(l[i][k + PER - 1], REF ? l2[i][k + PER - 1] : 0.f) : 0.f);
            }
            at.put(out, i * G + g, d);
        }
        if (some && a >= 0 && at.chunk_of(a) % G == g) out[a] = (T)(c.gradient<REF>(taken, taken2) + c.pick);  // by the lane that wrote the column just now
    }
    if (partial) put_sums(sums, op, partial);
}

// A block per row, in batches of G lanes times CH chunks; the next batch is on its way while one is summed up.
// Loss and gradient of 2048 x 50021 bf16 with a reference, a tenth of the rows left out: 154 us for 574 MB, 3.7 TB/s; some 240 MB are read twice, so that memory sees 5.3.  With rows at
// their own alignment 204, without columns kept in LDS 173.  Log-probabilities of 1000 x 32001: 16 us, 4.0 TB/s.
template <class E, int G, int CH, bool REF, class Op>
__global__ __launch_bounds__(G, 4) void long_rows(procgen_amd_rows p, Op op, const void *ref, long long ref_outer, long long ref_inner, double *partial) {
    typedef typename E::T T;
    constexpr int N = Chunk<E>::N, SPAN = G * CH * N;  // columns of a batch
    const int g = threadIdx.x, lane = threadIdx.x % WAVE;
    __shared__ float wave_stats[2][G / WAVE][6];
    // a lane's own columns of the last batches but one stay in LDS, 128 bytes of it a lane, and are not read from memory again for the gradient
    constexpr int KEPT = Op::GRADIENT ? 8 / (CH * (REF ? 2 : 1)) : 0;
    __shared__ Bits kept[KEPT ? KEPT : 1][REF ? 2 : 1][KEPT ? CH : 1][KEPT ? G : 1];
    if (op.done()) return;
    op.begin(p);
    Sums sums;
    const int columns = (int)p.columns;
    int odd = 0;
    for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const T *const row = (const T *)p.logits + row_offset(p, r, p.outer_stride, p.inner_stride);
        const T *const row2 = REF ? (const T *)ref + row_offset(p, r, ref_outer, ref_inner) : nullptr;
        T *const out = Op::GRADIENT && p.d_logits ? (T *)p.d_logits + r * p.columns : nullptr;
        bool some = false;
        const Place<E> at(row, columns);
        const int batches = (columns + at.ahead + SPAN - 1) / SPAN;
        auto chunk = [&](int b, int i) { return (b * CH + i) * G + g; };
        Chunk<E> l[CH], l2[REF ? CH : 1], next[CH], next2[REF ? CH : 1];  // the batch that is worked on, and the one on its way
        auto load = [&](int b) {
#pragma unroll
            for (int i = 0; i < CH; i++) {
                const int j = at.column(chunk(b, i));
                next[i].load(row + j);
                if (REF) next2[i].load(row2 + j);
            }
        };
        auto take = [&](int b) {
#pragma unroll
            for (int i = 0; i < CH; i++) {
                l[i] = next[i];
                if (REF) l2[i] = next2[i];
                at.drop(l[i], chunk(b, i));
                if (REF) at.drop(l2[i], chunk(b, i));
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
            float level = 0.f, level2 = 0.f;
            load(0);
            for (int b = 0; b < batches; b++) {
                take(b);
                if (b + 1 < batches) load(b + 1);
                if constexpr (KEPT > 0) {
                    if (out && b < batches - 1 && b >= batches - 1 - KEPT) {
#pragma unroll
                        for (int i = 0; i < CH; i++) {
                            kept[batches - 2 - b][0][i][g] = l[i].w;
                            if constexpr (REF) kept[batches - 2 - b][1][i][g] = l2[i].w;
                        }
                    }
                }
                float to = x.m, to2 = x.m2;
#pragma unroll
                for (int i = 0; i < CH; i++)
                    for (int k = 0; k < N; k++) {
                        to = fmaxf(to, l[i][k]);
                        if (REF) to2 = fmaxf(to2, l2[i][k]);
                    }
                // m need not be the largest value, only near it: it is moved where it is left behind by more than 8, which after the first batches is rare
                if (!(to <= x.m + 8.f) || (REF && !(to2 <= x.m2 + 8.f))) {
                    x.rescale(to, to2);
                    level = level_of(to);
                    level2 = level_of(to2);
                }
                forget();
#pragma unroll
                for (int i = 0; i < CH; i++)
                    for (int k = 0; k < N; k++) x.add(level, level2, l[i][k], REF ? l2[i][k] : 0.f);
            }
            x.template join<WAVE>();
            if (lane == 0) x.put(wave_stats[odd][threadIdx.x / WAVE]);
            __syncthreads();
            x = Stats<REF>();
            if (lane < G / WAVE) x.get(wave_stats[odd][lane]);
            x.template join<G / WAVE>();
            x.from_first();
            odd ^= 1;
            if (Op::GRADIENT && out && batches > 1 + KEPT) load(batches - 2 - KEPT);  // the first batch that has to be read again
            some = op.template finish<REF>(r, in, x, known, taken, g == 0, c, sums);
            forget();
        }
        if (!Op::GRADIENT || !out) continue;
        if (!some) {
            for (int i = 0; i < batches * CH; i++) {
                Chunk<E> zero;
                zero.w = Bits{0, 0, 0, 0};
                at.put(out, chunk(0, i), zero);
            }
            continue;
        }
        for (int b = batches - 1; b >= 0; b--) {
            if (KEPT && b < batches - 1 && b >= batches - 1 - KEPT) {
                if constexpr (KEPT > 0) {
#pragma unroll
                    for (int i = 0; i < CH; i++) {
                        l[i].w = kept[batches - 2 - b][0][i][g];
                        if constexpr (REF) l2[i].w = kept[batches - 2 - b][1][i][g];
                    }
                }
            } else if (b < batches - 1) {
                take(b);
                if (b > 0) load(b - 1);
            }
#pragma unroll
            for (int i = 0; i < CH; i++) {
                Chunk<E> d;
                constexpr int PER = N / 4;  // values of a word
#pragma unroll
                for (int k = 0; k < N; k += PER)
                    d.set(k / PER, c.gradient<REF>(l[i][k], REF ? l2[i][k] : 0.f), PER > 1 ? c.gradient<REF>(l[i][k + PER - 1], REF ? l2[i][k + PER - 1] : 0.f) : 0.f);
                at.put(out, chunk(b, i), d);
            }
        }
        if (a >= 0 && a < columns && at.chunk_of((int)a) % G == g)  // by the lane that wrote the column just now
            out[a] = (T)(c.gradient<REF>((float)row[a], REF ? (float)row2[a] : 0.f) + c.pick);
    }
    if (partial) put_sums(sums, op, partial);
}

// The gradient of long rows' log-probabilities: the largest value, the log of the sum and the entropy are known, so every column stands for itself.
// 1000 x 32001 bf16: 25 us, 5.1 TB/s.
template <class E>
__global__ __launch_bounds__(BLOCK) void logprobs_gradient(procgen_amd_rows p, const procgen_amd_lse *lse, const float *entropy, const float *d_logp, const float *d_entropy) {
    typedef typename E::T T;
    constexpr int N = Chunk<E>::N;
    const int columns = (int)p.columns;
    for (long long r = blockIdx.y; r < p.rows; r += gridDim.y) {
        const T *const row = (const T *)p.logits + row_offset(p, r, p.outer_stride, p.inner_stride);
        T *const out = (T *)p.d_logits + r * p.columns;
        const int ahead = (int)((uintptr_t)row / sizeof(T) % N), j = (int)(((long long)blockIdx.x * BLOCK + threadIdx.x) * N) - ahead;
        if (j >= columns) continue;
        const long long a = action_of(p, r);
        const float pick = d_logp ? d_logp[r] : 0.f, ent = d_entropy ? -d_entropy[r] : 0.f;
        const procgen_amd_lse z = lse[r];
        const bool known = a >= 0 && a < columns, some = !(pick == 0.f && ent == 0.f) && z.largest != -INFINITY;
        Chunk<E> x;
        const int at = max(0, min(j, columns - N));  // aligned 16 bytes but for the first and the last, which write only their own
        x.load(row + at);
        const float H = entropy[r];
        constexpr int PER = N / 4;
        auto gradient = [&](int k) {
            const float log_p = (x[k] - z.largest) - z.log_sum, p = __expf(log_p);
            return product(p, ent * (log_p + H) - pick) + (at + k == a ? pick : 0.f) + (known ? 0.f : NAN);
        };
        for (int k = 0; k < N; k += PER) {
            const float y = some ? gradient(k) : 0.f, z1 = some && PER > 1 ? gradient(k + PER - 1) : 0.f;
            x.set(k / PER, y, z1);
        }
        if (at == j) {
            x.store(out + j);
        } else {
            for (int k = 0; k < N; k++)
                if (at + k >= j && at + k < j + N) out[at + k] = x.piece(k);
        }
    }
}

// ---- the mean ------------------------------------------------------------------------------------------------------------------------------------

// 4 194 304 flags in 5 us, most of it the launch's own.
// How many rows count: one partial sum per block, added up by every wave that needs the number (whole numbers: any order gives the same)
__global__ __launch_bounds__(BLOCK) void count_valid(const uint8_t *valid, long long rows, long long *counts) {
    long long n = 0;
    const long long head = min(rows, (long long)(-(uintptr_t)valid & 15)), wide = (rows - head) / 16;  // bytes before the first aligned 16, and 16s
    const long long i = (long long)blockIdx.x * BLOCK + threadIdx.x, step = (long long)gridDim.x * BLOCK;
#pragma unroll 4
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
#pragma unroll 4
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
    const double mine = sum_of_waves(part, MEANS / WAVE);
    double sum[4];
    for (int i = 0; i < 4; i++) sum[i] = __shfl(mine, i, WAVE);
    if (lane == 0) put_means(q, n, sum);
}

// ---- launches ------------------------------------------------------------------------------------------------------------------------------------

bool rows_ok(const procgen_amd_rows *p) {
    return p && known_dtype(p->dtype) && p->rows >= 0 && p->rows <= 0x7fffff00ll && p->columns >= 1 && p->columns <= 0x7ffffff0ll - (1 << 18) && p->inner >= 1 && p->inner <= 0x7fffff00ll;  // rows are divided by inner in 32 bits
}

template <int I>
using Const = std::integral_constant<int, I>;

// one kernel over all rows; returns the blocks it was launched with (the partial sums), or -1 - error
template <class E, bool REF, class Op>
int launch_rows(const procgen_amd_rows &p, const Op &op, const void *ref, long long ref_outer, long long ref_inner, double *partial, hipStream_t stream) {
    int blocks = 0;
    auto grid = [&](int per_block, int most) { return blocks = (int)std::min<long long>(most, (p.rows + per_block - 1) / per_block); };
    // two rounds of one block, which ends with the means, cost less than a launch for them
    auto short_grid = [&](int most) { return partial && p.rows <= 2 * BLOCK ? blocks = 1 : grid(BLOCK, most); };
    constexpr int N = Chunk<E>::N;
    constexpr long long SIZE = sizeof(typename E::T);
    // as many columns as a row can span in aligned chunks
    const bool aligned = ((uintptr_t)p.logits | (uintptr_t)(p.outer_stride * SIZE) | (uintptr_t)(p.inner_stride * SIZE)) % 16 == 0;
    const long long padded = p.columns + (aligned ? 0 : N - 1);
    // A lane per row, where its registers leave enough waves.  Over 64 M columns in all, against the groups: 16-bit 17 columns 81 : 190 us, 32 60 : 96,
    // 33 83 : 160, 48 62 : 86, 63 68 : 113, but 64 152 : 68, with a reference 32 98 : 150, but 33 291 : 225; float32 16 107 : 171, 24 110 : 143, 31 109 : 189,
    // 32 107 : 127, with a reference 16 160 : 203, 24 156 : 168, 25 169 : 203, 31 149 : 201, but 32 314 : 141.
    constexpr int LANE_A_ROW = SIZE == 2 ? (REF ? 32 : 63) : REF ? 31 : 32;
    // with a gradient, float32 goes in chunks of as many values as 16 bits do: loss of 16000 columns 133 -> 122 us, with a reference 153 -> 119
    constexpr int MORE = Op::GRADIENT && SIZE == 4 ? 2 : 1;
    auto group = [&](auto lanes, auto chunks) {  // whether a row fits, and if so the launch
        constexpr int G = decltype(lanes)::value, CH = decltype(chunks)::value;
        if constexpr (G * CH * N > LANE_A_ROW) {
            if (padded <= G * CH * N) {
                group_rows<E, G, CH, REF, Op><<<grid(BLOCK / G, CUS * 4), BLOCK, 0, stream>>>(p, op, ref, ref_outer, ref_inner, partial);
                return true;
            }
        }
        return false;
    };
    auto groups = [&](auto lanes) { return group(lanes, Const<3>()) || group(lanes, Const<4>()) || group(lanes, Const<5>()); };
    const bool apart = p.inner != 1 || p.outer_stride != p.columns || (REF && ref_outer != p.columns);
    auto lanes = [&](auto most, auto turn) {
        constexpr int MOST = decltype(most)::value;
        constexpr bool TURN = decltype(turn)::value;
        const int n = short_grid(CUS * short_residents<E, MOST, REF, TURN>());
        const size_t lds = (size_t)short_tile<E, MOST>((int)p.columns) * (BLOCK / WAVE) * (REF ? 2 : 1);
        if (apart) short_rows<E, MOST, REF, Op, TURN, true><<<n, BLOCK, lds, stream>>>(p, op, ref, ref_outer, ref_inner, partial);
        else short_rows<E, MOST, REF, Op, TURN, false><<<n, BLOCK, lds, stream>>>(p, op, ref, ref_outer, ref_inner, partial);
    };
    if (p.columns <= LANE_A_ROW) {
        const std::integral_constant<bool, false> straight;
        const std::integral_constant<bool, SIZE == 4> turned;
        if (p.columns <= 8) lanes(Const<8>(), straight);
        else if (SIZE == 4 && p.columns == 16) lanes(Const<16>(), turned);
        else if (p.columns <= 16) lanes(Const<16>(), straight);
        else if (p.columns <= 24) lanes(Const<24>(), straight);
        else if (p.columns < 32) lanes(Const<32>(), straight);
        else if (p.columns == 32) {
            if constexpr (SIZE == 2 || !REF) lanes(Const<32>(), turned);
        } else if constexpr (SIZE == 2 && !REF) {
            if (p.columns <= 48) lanes(Const<48>(), straight);
            else lanes(Const<64>(), straight);
        }
    } else if (group(Const<4>(), Const<2>()) || groups(Const<4>()) || groups(Const<8>()) || groups(Const<16>()) || groups(Const<32>()) || groups(Const<64>())) {
    } else if constexpr (!Op::LONG) {
        return -1 - (int)hipErrorInvalidValue;
    } else if (group(Const<128>(), Const<3>()) || group(Const<64>(), Const<8>()) || (p.rows >= 2 * CUS && (group(Const<128>(), Const<5>()) || groups(Const<256>())))) {
    } else if (p.columns <= 256 * 2 * N || (p.rows >= 2 * CUS && !(REF && p.d_logits))) {
        long_rows<E, 256, 2 * MORE, REF, Op><<<grid(1, CUS * 4), BLOCK, 0, stream>>>(p, op, ref, ref_outer, ref_inner, partial);
    } else if (REF && p.rows >= 2 * CUS) {  // 2048 x 50021 bf16 with a reference: 154 us, against 173 with 256 lanes and two chunks, 179 with 1024
        if constexpr (REF) long_rows<E, 512, MORE, REF, Op><<<grid(1, CUS * 2), 512, 0, stream>>>(p, op, ref, ref_outer, ref_inner, partial);
    } else {  // too few rows to fill the card: more lanes for each
        long_rows<E, 1024, 2, REF, Op><<<grid(1, CUS), 1024, 0, stream>>>(p, op, ref, ref_outer, ref_inner, partial);
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

LIBENV_API int procgen_amd_action_logprobs(const struct procgen_amd_rows *p, float *logp, float *entropy, struct procgen_amd_lse *lse, int device, void *stream) {
    if (!rows_ok(p)) return -1;
    if (p->rows == 0) return 0;
    if (!p->logits || !p->actions || !logp || !entropy) return -1;
    OnDevice on(device);
    if (on.err != hipSuccess) return (int)on.err;
    const int got = by_dtype(p->dtype, [&](auto e) { return launch_rows<decltype(e), false>(*p, Logprobs{logp, entropy, lse}, nullptr, 0, 0, nullptr, (hipStream_t)stream); });
    return got < 0 ? -1 - got : 0;
}

LIBENV_API int procgen_amd_action_logprobs_backward(const struct procgen_amd_rows *p, const struct procgen_amd_lse *lse, const float *entropy, const float *d_logp, const float *d_entropy, int device, void *stream) {
    if (!rows_ok(p)) return -1;
    if (p->rows == 0) return 0;
    if (!p->logits || !p->actions || !p->d_logits || !lse || !entropy) return -1;
    OnDevice on(device);
    if (on.err != hipSuccess) return (int)on.err;
    return by_dtype(p->dtype, [&](auto e) {
        typedef decltype(e) E;
        if (p->columns <= 256 * Chunk<E>::N) {
            const int got = launch_rows<E, false>(*p, LogprobsBackward{d_logp, d_entropy}, nullptr, 0, 0, nullptr, (hipStream_t)stream);
            return got < 0 ? -1 - got : 0;
        }
        const long long chunks = (p->columns + Chunk<E>::N - 1) / Chunk<E>::N + 1;  // one more for rows that begin inside of 16 bytes
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
    if (!q->loss || blocks == 1) return 0;
    policy_means<<<1, MEANS, 0, (hipStream_t)stream>>>(*q, p->rows, counts, count_blocks, partial, blocks);
    return launched();
}

}  // extern "C"
