// learner_scan.hip -- recurrences along the steps of a rollout window: the gated linear recurrence of a policy's memory (forward, backward) and the
// advantages of its rewards, which are the same recurrence run from the last step to the first.
//
// A step is the affine map x -> a x + b, or x -> b where an episode begins (`cut`: a select, so that nothing of the other episode, NaN or infinite,
// passes).  Maps compose to maps of the same kind, so a chain is cut into pieces that are summed up at the same time and joined afterwards:
//   wave     8 consecutive steps in registers (4 backwards), their composition (A, B, cut) by an FMA each
//   block    four waves (eight or sixteen where chains are few) take consecutive pieces of a tile; the pieces' maps meet in LDS, every wave runs its value
//            at the tile's start through the pieces before its own, and does its steps again from there: one read and one write of the data, one barrier
//            a tile
//   segment  where there are too few chains to fill the card, the window is cut into segments for blocks of their own: a first kernel composes each
//            segment's map, the second begins each segment with the maps of those before it (the data is read twice)
// Lanes are chains (VEC neighbouring channels each), so that every load of a step is one coalesced row piece.
//
// Bound by memory: two to five operations an element.  A 1 GiB copy reaches 5.1 TB/s on the same card, a read alone 3.9; times below are of kernels whose
// inputs come from HBM.
#include "learner.h"

#include <algorithm>
#include <type_traits>

namespace pgamd {
namespace learner {
namespace {

constexpr int W1 = 4, WS = 8;     // waves of a block: where there are chains enough, and where there are few or a window is cut into segments
constexpr int KF = 8, KB = 4;     // steps of a wave in a tile: forwards (and advantages), backwards
constexpr int UNIT = KF * WS;     // a segment is a whole number of these: of the tiles of either direction
constexpr int CHECK = KB * W1;    // steps from one checkpoint to the next: a tile of the backward pass, or half of one

// VEC neighbouring channels of a step, as memory holds them.  Loads are unconditional (addresses are clamped into the arrays and values selected
// afterwards): a load behind a branch of its own would be waited for before the next is issued.
template <class E, int VEC>
struct Raw {
    typename E::T x[VEC];
    __device__ void load(const typename E::T *p) { __builtin_memcpy(x, p, sizeof x); }  // one wide load, whatever the alignment
};

template <int VEC>
struct Map {
    float A[VEC], B[VEC];
    bool cut;
    __device__ void identity() {
        cut = false;
        for (int v = 0; v < VEC; v++) A[v] = 1.f, B[v] = 0.f;
    }
    // FAR: A may have passed float's range, which no step of it has: zero times it is zero
    template <bool FAR>
    __device__ float at(float x, int v) const {
        return cut || (FAR && x == 0.f) ? B[v] : fmaf(A[v], x, B[v]);
    }
    __device__ void then(const Map &m) {  // this map first, m behind it
        for (int v = 0; v < VEC; v++) {
            B[v] = m.template at<true>(B[v], v);
            A[v] = A[v] * m.A[v];
        }
        cut = cut || m.cut;
    }
};

template <int VEC>
__device__ inline bool any_nan(const float (&x)[VEC], const float (&y)[VEC], const float (&z)[VEC]) {  // in any lane of the wave
    bool any = false;
    for (int v = 0; v < VEC; v++) any = any || __builtin_isunordered(x[v], y[v]) || __builtin_isunordered(x[v], z[v]);
    return __builtin_expect(__any(any), 0);
}

// the pieces' maps of a tile, by wave and lane
template <int VEC, int WAVES>
struct Pieces {
    struct alignas(4 * VEC) Vec {
        float x[VEC];
    };
    Vec A[WAVES][WAVE], B[WAVES][WAVE];
    int cut[WAVES][WAVE];
    __device__ void put(int w, int lane, const Map<VEC> &m) {
        Vec a, b;
        for (int v = 0; v < VEC; v++) a.x[v] = m.A[v], b.x[v] = m.B[v];
        A[w][lane] = a, B[w][lane] = b;
        cut[w][lane] = m.cut;
    }
    __device__ Map<VEC> get(int w, int lane) const {
        Map<VEC> m;
        const Vec a = A[w][lane], b = B[w][lane];
        for (int v = 0; v < VEC; v++) m.A[v] = a.x[v], m.B[v] = b.x[v];
        m.cut = cut[w][lane];
        return m;
    }
};

// where a lane's chains are: env n, channels d .. d + VEC - 1.  The last lane of an env reaches back over its neighbour's channels where VEC does not
// divide D, and writes only those from `skip` on; lanes behind the last chain double the last one and write nothing (skip = VEC).
template <int VEC>
struct Chain {
    int n, d, skip;
    long long c;  // index of the first one in [N][D]
    __device__ Chain(unsigned unit, int N, int D) {
        const unsigned lanes = ((unsigned)D + VEC - 1) / VEC, units = (unsigned)N * lanes, u = min(unit, units - 1);
        n = (int)(u / lanes);
        const int wanted = (int)(u - (unsigned)n * lanes) * VEC;
        d = min(wanted, D - VEC);
        skip = unit < units ? wanted - d : VEC;
        c = (long long)n * D + d;
    }
    __device__ bool mine(int v) const { return v >= skip; }
};

// segments of a window: `tiles` tiles each, maps[segment][A, B][chain], cuts[segment][chain], and a copy of the state that the window begins in
// (state_out may be the same memory, and its block does not wait for the first segment's)
struct Segments {
    int count, tiles;
    float *maps, *state;
    uint8_t *cuts;
    __device__ long long at(int s, int which, long long chains, long long c) const { return ((long long)s * 2 + which) * chains + c; }
};
template <int VEC>
__device__ inline void put_segment(const Segments &g, int s, long long chains, const Chain<VEC> &ch, const Map<VEC> &m) {
    for (int v = 0; v < VEC; v++)
        if (ch.mine(v)) {
            g.maps[g.at(s, 0, chains, ch.c + v)] = m.A[v];
            g.maps[g.at(s, 1, chains, ch.c + v)] = m.B[v];
            g.cuts[s * chains + ch.c + v] = m.cut;
        }
}
template <int VEC>
__device__ inline Map<VEC> get_segment(const Segments &g, int s, long long chains, const Chain<VEC> &ch) {
    Map<VEC> m;
    for (int v = 0; v < VEC; v++) m.A[v] = g.maps[g.at(s, 0, chains, ch.c + v)], m.B[v] = g.maps[g.at(s, 1, chains, ch.c + v)];
    m.cut = g.cuts[s * chains + ch.c];
    return m;
}

// x[] run through the segments [from, to) in order (to < from: downwards): the waves take a part each and join in LDS
template <int VEC, int WAVES>
__device__ inline void run_segments(float *x, const Segments &g, int from, int to, long long chains, const Chain<VEC> &ch, Pieces<VEC, WAVES> &pieces, int w, int W, int lane) {
    const int n = abs(to - from), way = to < from ? -1 : 1, first = (int)((long long)n * w / W), last = (int)((long long)n * (w + 1) / W);
    Map<VEC> m;
    m.identity();
    for (int i = first; i < last; i++) m.then(get_segment<VEC>(g, from + way * i - (way < 0), chains, ch));
    pieces.put(w, lane, m);
    __syncthreads();
    for (int k = 0; k < W; k++) {
        const Map<VEC> q = pieces.get(k, lane);
        for (int v = 0; v < VEC; v++) x[v] = q.template at<true>(x[v], v);
    }
    __syncthreads();
}

// a lane's view of one array: the rows of its channels
template <class E, int VEC, int K>
struct Column {
    typename E::T *base;
    long long stride;
    __device__ Column(const procgen_amd_array3 &a, const Chain<VEC> &ch) : base((typename E::T *)a.data + ch.n * a.n_stride + ch.d * a.d_stride), stride(a.t_stride) {}
    __device__ void load(Raw<E, VEC> *to, int t, int last) const {  // steps t .. t + K - 1, none behind `last`
#pragma unroll
        for (int k = 0; k < K; k++) to[k].load(base + min(t + k, last) * stride);
    }
    __device__ void store(int t, const float *x, const Chain<VEC> &ch) const {
        typename E::T raw[VEC], *p = base + t * stride;
        for (int v = 0; v < VEC; v++) raw[v] = (typename E::T)x[v];
        if (ch.skip == 0) {
            __builtin_memcpy(p, raw, sizeof raw);
        } else {
            for (int v = 0; v < VEC; v++)
                if (ch.mine(v)) p[v] = raw[v];
        }
    }
};
// the flags of a lane's env; without any, some bytes of the gates are read and masked
struct Flags {
    const uint8_t *base;
    long long stride;
    uint8_t mask;
    __device__ Flags(const uint8_t *first, long long t_stride, long long n_stride, int n, const void *otherwise)
        : base(first ? first + n * n_stride : (const uint8_t *)otherwise), stride(first ? t_stride : 0), mask(first ? 0xff : 0) {}
    template <int K>
    __device__ void load(uint8_t (&to)[K], int t, int last) const {
#pragma unroll
        for (int k = 0; k < K; k++) to[k] = base[min(t + k, last) * stride];
    }
};

template <int VEC>
__device__ inline void load_state(float *x, const float *state, const Chain<VEC> &ch) {
    if (state) {
        __builtin_memcpy(x, state + ch.c, VEC * sizeof(float));
    } else {
        for (int v = 0; v < VEC; v++) x[v] = 0.f;
    }
}
template <int VEC>
__device__ inline void store_state(float *state, const float *x, const Chain<VEC> &ch) {
    if (ch.skip == 0) {
        __builtin_memcpy(state + ch.c, x, VEC * sizeof(float));
    } else {
        for (int v = 0; v < VEC; v++)
            if (ch.mine(v)) state[ch.c + v] = x[v];
    }
}

// the composition of K steps: x -> gate x + update forwards; backwards the gradient y of a step's h from behind it becomes gate (d + y) before it
template <int VEC, bool REVERSE, int K>
__device__ inline Map<VEC> compose(const float (&a)[K][VEC], const float (&b)[K][VEC], const bool (&cut)[K]) {
    Map<VEC> m;
    m.identity();
#pragma unroll
    for (int i = 0; i < K; i++) {
        const int k = REVERSE ? K - 1 - i : i;
        for (int v = 0; v < VEC; v++) {
            m.B[v] = REVERSE ? (cut[k] ? 0.f : a[k][v] * (b[k][v] + m.B[v])) : (cut[k] ? b[k][v] : fmaf(a[k][v], m.B[v], b[k][v]));
            m.A[v] *= a[k][v];
        }
        m.cut = m.cut || cut[k];
    }
    return m;
}
// K loaded steps in 32 bits; those at `end` and behind it become the identity
template <class E, int VEC, int K>
__device__ inline void convert(float (&x)[K][VEC], const Raw<E, VEC> (&raw)[K], int t, int end, float otherwise) {
#pragma unroll
    for (int k = 0; k < K; k++)
        for (int v = 0; v < VEC; v++) x[k][v] = t + k < end ? (float)raw[k].x[v] : otherwise;
}
template <int K>
__device__ inline void convert(bool (&cut)[K], const uint8_t (&raw)[K], uint8_t mask, int t, int end) {
#pragma unroll
    for (int k = 0; k < K; k++) cut[k] = t + k < end && (raw[k] & mask);
}

// 32768 x 512 float32: 37 us forwards (134 MB read, 3.6 TB/s: the rate of a read), 25 backwards (the gates still in the Infinity Cache).
// The map of every segment (blockIdx.y): forwards of gate and update, backwards of gate and d_h.  The waves take a part of the segment each.
template <class E, int VEC, int WAVES, bool REVERSE>
__global__ __launch_bounds__(WAVES *WAVE) void recurrence_segments(procgen_amd_recurrence p, Segments g) {
    constexpr int K = KF;
    __shared__ Pieces<VEC, WAVES> pieces;
    const int lane = threadIdx.x, w = __builtin_amdgcn_readfirstlane(threadIdx.y), W = blockDim.y, s = blockIdx.y;
    const Chain<VEC> ch(blockIdx.x * WAVE + lane, p.N, p.D);
    const long long chains = (long long)p.N * p.D;
    const int begin = s * g.tiles * UNIT, end = min((long long)p.T, (long long)begin + (long long)g.tiles * UNIT);
    const int part = (g.tiles * UNIT + W * K - 1) / (W * K) * K;  // steps of a wave
    const int from = min((long long)end, (long long)begin + (long long)w * part), to = min((long long)end, (long long)from + part);
    const bool any = !REVERSE || p.d_h.data;
    const Column<E, VEC, K> gate(p.gate, ch), other(REVERSE ? (any ? p.d_h : p.gate) : p.update, ch);
    const Flags first(p.first, p.first_t_stride, p.first_n_stride, ch.n, gate.base);
    Map<VEC> m;
    m.identity();
    for (int i = 0; i < to - from; i += K) {
        const int t = REVERSE ? from + (to - from - 1) / K * K - i : from + i;
        Raw<E, VEC> ra[K], rb[K];
        uint8_t rf[K];
        gate.load(ra, t, end - 1);
        other.load(rb, t, end - 1);
        first.load(rf, t, end - 1);
        float a[K][VEC], b[K][VEC];
        bool cut[K];
        convert<E, VEC, K>(a, ra, t, to, 1.f);
        convert<E, VEC, K>(b, rb, t, any ? to : 0, 0.f);
        convert(cut, rf, first.mask, t, to);
        m.then(compose<VEC, REVERSE, K>(a, b, cut));
    }
    pieces.put(w, lane, m);
    __syncthreads();
    if (w) return;
    m.identity();
    for (int k = 0; k < W; k++) m.then(pieces.get(REVERSE ? W - 1 - k : k, lane));
    put_segment<VEC>(g, s, chains, ch, m);
    if (!REVERSE && s == 0 && p.state) {
        float x[VEC];
        load_state<VEC>(x, p.state, ch);
        store_state<VEC>(g.state, x, ch);
    }
}

// 256 x 512 x 256 bf16: 46 us, 210 MB with the checkpoints, 4.6 TB/s (eight waves a block 49, two channels a lane 49).  32768 x 512 float32 behind its
// segments: 39 us, 5.2 TB/s.  What is left: the last tiles of a block have nothing on its way, and 2048 blocks of four waves end at different times.
template <class E, int VEC, int WAVES>
__global__ __launch_bounds__(WAVES *WAVE) void recurrence_forward(procgen_amd_recurrence p, Segments g) {
    constexpr int K = KF, TILE = K * WAVES;
    __shared__ Pieces<VEC, WAVES> pieces[2];
    const int lane = threadIdx.x, w = __builtin_amdgcn_readfirstlane(threadIdx.y), W = blockDim.y, s = blockIdx.y;
    const Chain<VEC> ch(blockIdx.x * WAVE + lane, p.N, p.D);
    const long long chains = (long long)p.N * p.D;
    const int begin = s * g.tiles * UNIT, end = min((long long)p.T, (long long)begin + (long long)g.tiles * UNIT), last = end - 1;
    const Column<E, VEC, K> gate(p.gate, ch), update(p.update, ch), out(p.h, ch);
    const Flags first(p.first, p.first_t_stride, p.first_n_stride, ch.n, gate.base);
    Raw<E, VEC> ra[K], rb[K];
    uint8_t rf[K];
    auto load = [&](int t) {
        gate.load(ra, t, last);
        update.load(rb, t, last);
        first.load(rf, t, last);
    };
    load(begin + w * K);
    float x[VEC];
    load_state<VEC>(x, p.state && g.count > 1 ? g.state : p.state, ch);
    if (s) run_segments(x, g, 0, s, chains, ch, pieces[0], w, W, lane);
    for (int t0 = begin, odd = 0; t0 < end; t0 += TILE, odd ^= 1) {
        const int t = t0 + w * K;
        float a[K][VEC], b[K][VEC];
        bool cut[K];
        convert<E, VEC, K>(a, ra, t, end, 1.f);
        convert<E, VEC, K>(b, rb, t, end, 0.f);
        convert(cut, rf, first.mask, t, end);
        if (t0 + TILE < end) load(t + TILE);  // the next tile is on its way while this one is joined
        pieces[odd].put(w, lane, compose<VEC, false, K>(a, b, cut));
        __syncthreads();
        float y[VEC], start[VEC];
        for (int v = 0; v < VEC; v++) start[v] = y[v] = x[v];
        auto join = [&](auto far) {
            for (int k = 0; k < W; k++) {
                const Map<VEC> q = pieces[odd].get(k, lane);
                for (int v = 0; v < VEC; v++) {
                    if (k == w) y[v] = x[v];
                    x[v] = q.template at<decltype(far)::value>(x[v], v);
                }
            }
        };
        join(std::false_type());
        if (any_nan(x, y, y)) {  // it may be an infinite product times zero: once more, with a question at every piece, which at once would cost up to a tenth of the time
            for (int v = 0; v < VEC; v++) x[v] = y[v] = start[v];
            join(std::true_type());
        }
        if (p.checkpoints && w * K % CHECK == 0 && t < end) store_state<VEC>(p.checkpoints + (long long)(t / CHECK) * chains, y, ch);
#pragma unroll
        for (int k = 0; k < K; k++) {
            for (int v = 0; v < VEC; v++) y[v] = cut[k] ? b[k][v] : fmaf(a[k][v], y[v], b[k][v]);
            if (t + k < end) out.store(t + k, y, ch);
        }
    }
    if (p.state_out && w == 0 && s == g.count - 1) store_state<VEC>(p.state_out, x, ch);
}

// Backwards over the tiles.  h is not read: its 32-bit value before every step comes from the checkpoint at the tile's start and the same joins as in
// the forward pass (update is read in its place, so the bytes are the same and 16-bit rounding of h does not reach d_gate).
// 256 x 512 x 256 bf16: 74 us, 344 MB, 4.6 TB/s; tiles of 64 steps over eight waves took 96 (158 registers, one block on a compute unit), of 32 steps 78.
// 32768 x 512 float32: 63 us, 5.4 TB/s.
template <class E, int VEC, int WAVES>
__global__ __launch_bounds__(WAVES *WAVE) void recurrence_backward(procgen_amd_recurrence p, Segments g) {
    constexpr int K = KB, TILE = K * WAVES;
    __shared__ Pieces<VEC, WAVES> fore[2], back[2];
    const int lane = threadIdx.x, w = __builtin_amdgcn_readfirstlane(threadIdx.y), W = blockDim.y, s = blockIdx.y;
    const Chain<VEC> ch(blockIdx.x * WAVE + lane, p.N, p.D);
    const long long chains = (long long)p.N * p.D;
    const int begin = s * g.tiles * UNIT, end = min((long long)p.T, (long long)begin + (long long)g.tiles * UNIT), last = end - 1;
    const bool any = p.d_h.data;
    const Column<E, VEC, K> gate(p.gate, ch), update(p.update, ch), d_h(any ? p.d_h : p.gate, ch), d_gate(p.d_gate, ch), d_update(p.d_update, ch);
    const Flags first(p.first, p.first_t_stride, p.first_n_stride, ch.n, gate.base);
    Raw<E, VEC> ra[K], rb[K], rd[K];
    uint8_t rf[K];
    float start[VEC];
    auto load = [&](int t0) {
        const int t = t0 + w * K;
        gate.load(ra, t, last);
        d_h.load(rd, t, last);
        update.load(rb, t, last);
        first.load(rf, t, last);
        load_state<VEC>(start, p.checkpoints + (long long)(t0 / CHECK) * chains, ch);
    };
    const int top = begin + (end - begin - 1) / TILE * TILE;
    load(top);
    float y[VEC];  // what reaches h from the steps behind the tile
    load_state<VEC>(y, p.d_state_out, ch);
    if (s < g.count - 1) run_segments(y, g, g.count, s + 1, chains, ch, fore[0], w, W, lane);
    for (int t0 = top, odd = 0; t0 >= begin; t0 -= TILE, odd ^= 1) {
        const int t = t0 + w * K;
        float a[K][VEC], b[K][VEC], d[K][VEC], x[VEC], before[VEC], behind[VEC];
        bool cut[K];
        convert<E, VEC, K>(a, ra, t, end, 1.f);
        convert<E, VEC, K>(b, rb, t, end, 0.f);
        convert<E, VEC, K>(d, rd, t, any ? end : 0, 0.f);
        convert(cut, rf, first.mask, t, end);
        for (int v = 0; v < VEC; v++) x[v] = start[v];
        if (t0 > begin) load(t0 - TILE);
        fore[odd].put(w, lane, compose<VEC, false, K>(a, b, cut));
        back[odd].put(w, lane, compose<VEC, true, K>(a, d, cut));
        __syncthreads();
        float first_x[VEC], first_y[VEC];
        for (int v = 0; v < VEC; v++) before[v] = first_x[v] = x[v], behind[v] = first_y[v] = y[v];
        auto join = [&](auto far) {
            constexpr bool FAR = decltype(far)::value;
#pragma clang loop unroll_count(FAR ? 1 : 4)
            for (int k = 0; k < W; k++) {
                const Map<VEC> f = fore[odd].get(k, lane), q = back[odd].get(W - 1 - k, lane);
                for (int v = 0; v < VEC; v++) {
                    if (k == w) before[v] = x[v];
                    x[v] = f.template at<FAR>(x[v], v);
                    if (W - 1 - k == w) behind[v] = y[v];
                    y[v] = q.template at<FAR>(y[v], v);
                }
            }
        };
        join(std::false_type());
        if (any_nan(y, before, behind)) {
            for (int v = 0; v < VEC; v++) before[v] = x[v] = first_x[v], behind[v] = y[v] = first_y[v];
            join(std::true_type());
        }
#pragma unroll
        for (int k = 0; k < K; k++)  // b becomes the value before the step
            for (int v = 0; v < VEC; v++) {
                const float h = cut[k] ? b[k][v] : fmaf(a[k][v], before[v], b[k][v]);
                b[k][v] = before[v];
                before[v] = h;
            }
#pragma unroll
        for (int k = K - 1; k >= 0; k--) {
            for (int v = 0; v < VEC; v++) {
                const float gr = d[k][v] + behind[v];
                d[k][v] = gr;
                b[k][v] = cut[k] ? 0.f : gr * b[k][v];
                behind[v] = cut[k] ? 0.f : a[k][v] * gr;
            }
            if (t + k < end) {
                if (p.d_update.data) d_update.store(t + k, d[k], ch);
                if (p.d_gate.data) d_gate.store(t + k, b[k], ch);
            }
        }
    }
    if (p.d_state && w == 0 && s == 0) store_state<VEC>(p.d_state, y, ch);
}

// ---- a few steps, as acting takes them: a lane goes through them by itself, 16 bytes of channels at a time ----------------------------------------------

constexpr int FEW = 4;
template <class E, int VEC>
struct FewSteps {
    const Chain<VEC> ch;
    float a[FEW][VEC], b[FEW][VEC], x[VEC];
    bool cut[FEW];
    __device__ FewSteps(const procgen_amd_recurrence &p, const float *state) : ch(blockIdx.x * blockDim.x + threadIdx.x, p.N, p.D) {
        const Column<E, VEC, FEW> gate(p.gate, ch), update(p.update, ch);
        const Flags first(p.first, p.first_t_stride, p.first_n_stride, ch.n, gate.base);
        Raw<E, VEC> ra[FEW], rb[FEW];
        uint8_t rf[FEW];
        gate.load(ra, 0, p.T - 1);
        update.load(rb, 0, p.T - 1);
        first.load(rf, 0, p.T - 1);
        load_state<VEC>(x, state, ch);
        convert<E, VEC, FEW>(a, ra, 0, p.T, 1.f);
        convert<E, VEC, FEW>(b, rb, 0, p.T, 0.f);
        convert(cut, rf, first.mask, 0, p.T);
    }
};
template <class E, int VEC>
__global__ __launch_bounds__(256) void recurrence_few_forward(procgen_amd_recurrence p) {
    FewSteps<E, VEC> s(p, p.state);
    const Column<E, VEC, FEW> out(p.h, s.ch);
    if (p.checkpoints) store_state<VEC>(p.checkpoints, s.x, s.ch);
#pragma unroll
    for (int k = 0; k < FEW; k++) {
        for (int v = 0; v < VEC; v++) s.x[v] = s.cut[k] ? s.b[k][v] : fmaf(s.a[k][v], s.x[v], s.b[k][v]);
        if (k < p.T) out.store(k, s.x, s.ch);
    }
    if (p.state_out) store_state<VEC>(p.state_out, s.x, s.ch);
}
template <class E, int VEC>
__global__ __launch_bounds__(256) void recurrence_few_backward(procgen_amd_recurrence p) {
    FewSteps<E, VEC> s(p, p.checkpoints);  // the only one: the state that the window began in
    const bool any = p.d_h.data;
    const Column<E, VEC, FEW> d_h(any ? p.d_h : p.gate, s.ch), d_gate(p.d_gate, s.ch), d_update(p.d_update, s.ch);
    Raw<E, VEC> rd[FEW];
    d_h.load(rd, 0, p.T - 1);
    float d[FEW][VEC], y[VEC];
    load_state<VEC>(y, p.d_state_out, s.ch);
    convert<E, VEC, FEW>(d, rd, 0, any ? p.T : 0, 0.f);
#pragma unroll
    for (int k = 0; k < FEW; k++)  // b becomes the value before the step
        for (int v = 0; v < VEC; v++) {
            const float h = s.cut[k] ? s.b[k][v] : fmaf(s.a[k][v], s.x[v], s.b[k][v]);
            s.b[k][v] = s.x[v];
            s.x[v] = h;
        }
#pragma unroll
    for (int k = FEW - 1; k >= 0; k--) {
        for (int v = 0; v < VEC; v++) {
            const float gr = d[k][v] + y[v];
            d[k][v] = gr;
            s.b[k][v] = s.cut[k] ? 0.f : gr * s.b[k][v];
            y[v] = s.cut[k] ? 0.f : s.a[k][v] * gr;
        }
        if (k < p.T) {
            if (p.d_update.data) d_update.store(k, d[k], s.ch);
            if (p.d_gate.data) d_gate.store(k, s.b[k], s.ch);
        }
    }
    if (p.d_state) store_state<VEC>(p.d_state, y, s.ch);
}

// ---- advantages: the recurrence adv[t] = (gamma lam) adv[t+1] + delta[t], from the last step to the first, a chain per env -----------------------------

template <class E>
struct Advantage {
    static constexpr int K = KF;
    const procgen_amd_advantage &p;
    const Chain<1> ch;
    const float decay;
    const uint8_t *first;
    const typename E::T *values;
    const float *rew;
    // steps t .. t + K - 1 as loaded: flags and values of the step behind each, the value of the first, rewards
    uint8_t rf[K];
    typename E::T rv[K + 1];
    float rr[K];
    __device__ Advantage(const procgen_amd_advantage &args)
        : p(args), ch(blockIdx.x * WAVE + threadIdx.x, args.N, 1), decay(args.gamma * args.lam), first(args.first + ch.n * args.first_n_stride),
          values((const typename E::T *)args.values + ch.n * args.values_n_stride), rew(args.rew + ch.n * args.rew_n_stride) {}
    __device__ void load(int t, int last) {
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int at = min(t + k, last);
            rf[k] = first[(at + 1) * p.first_t_stride];
            rr[k] = rew[at * p.rew_t_stride];
            rv[k] = values[at * p.values_t_stride];
        }
        rv[K] = values[(min(t + K - 1, last) + 1) * p.values_t_stride];
    }
    // cut[k], a[k] (1 where there is no step), b[k] = delta, v[k] = the value before the step
    __device__ void convert(int t, int end, bool *cut, float *a, float *b, float *v) const {
        const int n = min(K, end - t);
#pragma unroll
        for (int k = 0; k < K; k++) {
            const bool real = k < n;
            cut[k] = real && rf[k];
            v[k] = (float)rv[k];
            const float after = k + 1 < n ? (float)rv[k + 1] : (float)rv[K];
            a[k] = real ? decay : 1.f;
            b[k] = real ? (cut[k] ? rr[k] : fmaf(p.gamma, after, rr[k])) - v[k] : 0.f;
        }
    }
};
template <int K>
__device__ inline Map<1> compose_back(const bool (&cut)[K], const float (&a)[K], const float (&b)[K]) {
    Map<1> m;
    m.identity();
#pragma unroll
    for (int k = K - 1; k >= 0; k--) {
        m.B[0] = cut[k] ? b[k] : fmaf(a[k], m.B[0], b[k]);
        m.A[0] *= a[k];
        m.cut = m.cut || cut[k];
    }
    return m;
}

template <class E, int WAVES>
__global__ __launch_bounds__(WAVES *WAVE) void advantage_segments(procgen_amd_advantage p, Segments g) {
    constexpr int K = KF;
    __shared__ Pieces<1, WAVES> pieces;
    const int lane = threadIdx.x, w = __builtin_amdgcn_readfirstlane(threadIdx.y), W = blockDim.y, s = blockIdx.y;
    Advantage<E> r(p);
    const int begin = s * g.tiles * UNIT, end = min((long long)p.T, (long long)begin + (long long)g.tiles * UNIT);
    const int part = (g.tiles * UNIT + W * K - 1) / (W * K) * K;
    const int from = min((long long)end, (long long)begin + (long long)w * part), to = min((long long)end, (long long)from + part);
    Map<1> m;
    m.identity();
    for (int t = from + (to - from - 1) / K * K; t >= from && t < to; t -= K) {
        bool cut[K];
        float a[K], b[K], v[K];
        r.load(t, to - 1);
        r.convert(t, to, cut, a, b, v);
        m.then(compose_back(cut, a, b));
    }
    pieces.put(w, lane, m);
    __syncthreads();
    if (w) return;
    m.identity();
    for (int k = W - 1; k >= 0; k--) m.then(pieces.get(k, lane));
    put_segment<1>(g, s, p.N, r.ch, m);
}

// 256 x 65536, values in float32: 55 us, 286 MB, 5.2 TB/s: the rate of a copy.
template <class E, int WAVES>
__global__ __launch_bounds__(WAVES *WAVE) void advantages(procgen_amd_advantage p, Segments g) {
    constexpr int K = KF, TILE = K * WAVES;
    __shared__ Pieces<1, WAVES> pieces[2];
    const int lane = threadIdx.x, w = __builtin_amdgcn_readfirstlane(threadIdx.y), W = blockDim.y, s = blockIdx.y;
    Advantage<E> r(p);
    const int begin = s * g.tiles * UNIT, end = min((long long)p.T, (long long)begin + (long long)g.tiles * UNIT);
    const int top = begin + (end - begin - 1) / TILE * TILE;
    r.load(top + w * K, end - 1);
    float y = 0.f;
    if (s < g.count - 1) run_segments(&y, g, g.count, s + 1, p.N, r.ch, pieces[0], w, W, lane);
    for (int t0 = top, odd = 0; t0 >= begin; t0 -= TILE, odd ^= 1) {
        const int t = t0 + w * K;
        bool cut[K];
        float a[K], b[K], v[K];
        r.convert(t, end, cut, a, b, v);
        if (t0 > begin) r.load(t - TILE, end - 1);
        pieces[odd].put(w, lane, compose_back(cut, a, b));
        __syncthreads();
        float adv = y;
        for (int k = W - 1; k >= 0; k--) {
            if (k == w) adv = y;
            y = pieces[odd].get(k, lane).template at<false>(y, 0);  // gamma lam is one at the most
        }
#pragma unroll
        for (int k = K - 1; k >= 0; k--) {
            adv = cut[k] ? b[k] : fmaf(a[k], adv, b[k]);
            if (r.ch.mine(0) && t + k < end) {
                if (p.adv) p.adv[(long long)(t + k) * p.N + r.ch.n] = adv;
                if (p.ret) p.ret[(long long)(t + k) * p.N + r.ch.n] = adv + v[k];
            }
        }
    }
}

// ---- launches ----------------------------------------------------------------------------------------------------------------------------------

bool shape_ok(int dtype, int T, int N, int D) { return known_dtype(dtype) && T >= 0 && T <= 0x7fffff00 && N >= 0 && D >= 0 && (long long)N * D <= 0x7fffff00ll; }

constexpr int FULL = 512;  // blocks that fill the card: two on each of the 256 compute units
// Blocks from which on a window stays whole.  256 blocks of eight waves read the inputs once in less time than 512 blocks of segments read them twice: 2048
// x 32 x 512 float32 forward 78 : 122 us, backward 153 : 186; at 192 blocks 4000 x 24 x 512 bf16 does not, 276 : 232 backwards.  Advantages, one kernel
// with little to keep, go on to 128 blocks of sixteen waves: 1000 x 10000 float32 36 : 55.
constexpr int ENOUGH = FULL / 2, ENOUGH_ADVANTAGES = FULL / 4, WA = 16;
int units_of(int T) { return (T + UNIT - 1) / UNIT; }
// How many segments a window of so many chains is cut into: by its sizes alone, so that the workspace does not depend on strides.  Not more than 256, since
// every segment begins with the maps of all before it (100 000 x 16 float32: forward and backward 125 us with 128, 87 with 256, 85 with 512).
int segments_of(int T, long long chains, int enough = ENOUGH) {
    const long long blocks = (chains + WAVE - 1) / WAVE;
    if (blocks >= enough) return 1;
    return (int)std::max(1ll, std::min({(FULL + blocks - 1) / blocks, units_of(T) / 2ll, 256ll}));
}
Segments segments(int T, long long chains, void *workspace, int enough = ENOUGH) {
    Segments g;
    const int wanted = segments_of(T, chains, enough);
    g.tiles = (units_of(T) + wanted - 1) / wanted;
    g.count = (units_of(T) + g.tiles - 1) / g.tiles;
    g.maps = (float *)workspace;
    g.state = g.maps + 2ll * g.count * chains;
    g.cuts = (uint8_t *)(g.state + chains);
    return g;
}
long long segment_bytes(int T, long long chains) {
    const long long s = segments_of(T, chains);
    return s > 1 ? s * chains * 9 + chains * 4 : 0;
}

// neighbouring channels of a lane, where the arrays have them next to each other: as many as still leave half a card's blocks, up to 8 bytes; two
// backwards, whose three arrays would take 190 registers with four
bool channels_adjoin(const procgen_amd_recurrence *a, bool backward) {
    const procgen_amd_array3 *all[] = {&a->gate, &a->update, &a->h, &a->d_h, &a->d_gate, &a->d_update};
    for (int i = 0; i < (backward ? 6 : 3); i++)
        if (all[i]->data && all[i]->d_stride != 1) return false;
    return true;
}
int vec_for(const procgen_amd_recurrence *a, bool backward) {
    if (!channels_adjoin(a, backward)) return 1;
    for (int vec = backward || a->dtype == PROCGEN_AMD_F32 ? 2 : 4; vec > 1; vec /= 2)
        if (a->D >= vec && (long long)a->N * ((a->D + vec - 1) / vec) >= FULL * (long long)WAVE) return vec;
    return 1;
}
// fn(VEC, WAVES): a window in segments has few chains, and goes with one a lane: float32 32768 x 512 forward 57 us, backward 91, 4096 x 16 x 256 55 and 88, with two
// 57 and 98, 58 and 98.  (Of 16 bits two a lane with twice the segments would take less: bf16 53 : 42 and 80 : 61, 49 : 36 and 73 : 54.)  With one a lane eight waves:
// 1024 x 64 x 512 bf16 forward 53 us, backward 109, with four 66 and 126
template <int MOST, class Fn>
int by_shape(const Segments &g, int vec, Fn fn) {
    typedef std::integral_constant<int, 1> One;
    const std::integral_constant<int, W1> waves;
    switch (g.count > 1 ? 1 : vec) {
        case 4:
            if constexpr (MOST == 4) return fn(std::integral_constant<int, 4>(), waves);
        case 2: return fn(std::integral_constant<int, 2>(), waves);
        default: return fn(One(), std::integral_constant<int, WS>());
    }
}
// fn(VEC) for a few steps: up to 16 bytes a lane, where that leaves a block for every compute unit.  65 536 x 256 bf16, one step: forward 31 us
// against 115 with the tiles, backward 34 against 143
template <class E, class Fn>
int by_few(const procgen_amd_recurrence *a, bool backward, Fn fn) {
    int vec = channels_adjoin(a, backward) ? 16 / (int)sizeof(typename E::T) : 1;
    while (vec > 1 && (a->D < vec || (long long)a->N * ((a->D + vec - 1) / vec) < 256 * 256)) vec /= 2;
    const unsigned blocks = (unsigned)(((long long)a->N * ((a->D + vec - 1) / vec) + 255) / 256);
    switch (vec) {
        case 8:
            if constexpr (sizeof(typename E::T) == 2) return fn(std::integral_constant<int, 8>(), blocks);
        case 4: return fn(std::integral_constant<int, 4>(), blocks);
        case 2: return fn(std::integral_constant<int, 2>(), blocks);
        default: return fn(std::integral_constant<int, 1>(), blocks);
    }
}
unsigned chain_blocks(const procgen_amd_recurrence *a, int vec) { return (unsigned)(((long long)a->N * ((a->D + vec - 1) / vec) + WAVE - 1) / WAVE); }

}  // namespace
}  // namespace learner
}  // namespace pgamd

using namespace pgamd::learner;

extern "C" {

LIBENV_API long long procgen_amd_recurrence_checkpoints(int T) { return T > 0 ? ((long long)T + CHECK - 1) / CHECK : 0; }
LIBENV_API long long procgen_amd_recurrence_workspace(int T, int N, int D) { return T > 0 && N > 0 && D > 0 ? segment_bytes(T, (long long)N * D) : 0; }

LIBENV_API int procgen_amd_recurrence_forward(const struct procgen_amd_recurrence *a, int device, void *stream) {
    if (!a || !shape_ok(a->dtype, a->T, a->N, a->D) || a->T < 1) return -1;
    const long long chains = (long long)a->N * a->D;
    if (chains == 0) return 0;
    const Segments g = segments(a->T, chains, a->workspace);
    if (!a->gate.data || !a->update.data || !a->h.data || (g.count > 1 && !a->workspace)) return -1;
    OnDevice on(device);
    if (on.err != hipSuccess) return (int)on.err;
    return by_dtype(a->dtype, [&](auto e) {
        typedef decltype(e) E;
        if (a->T <= FEW)
            return by_few<E>(a, false, [&](auto vec, unsigned blocks) {
                recurrence_few_forward<E, decltype(vec)::value><<<blocks, 256, 0, (hipStream_t)stream>>>(*a);
                return launched();
            });
        return by_shape<sizeof(typename E::T) == 2 ? 4 : 2>(g, vec_for(a, false), [&](auto vec, auto waves) {
            constexpr int VEC = decltype(vec)::value, WAVES = decltype(waves)::value;
            const dim3 grid(chain_blocks(a, VEC), g.count), block(WAVE, std::min(WAVES, (a->T + KF - 1) / KF));
            if constexpr (VEC == 1) {
                if (g.count > 1) {
                    recurrence_segments<E, VEC, WAVES, false><<<grid, block, 0, (hipStream_t)stream>>>(*a, g);
                    if (int err = launched()) return err;
                }
            }
            recurrence_forward<E, VEC, WAVES><<<grid, block, 0, (hipStream_t)stream>>>(*a, g);
            return launched();
        });
    });
}

LIBENV_API int procgen_amd_recurrence_backward(const struct procgen_amd_recurrence *a, int device, void *stream) {
    if (!a || !shape_ok(a->dtype, a->T, a->N, a->D) || a->T < 1) return -1;
    const long long chains = (long long)a->N * a->D;
    if (chains == 0) return 0;
    const Segments g = segments(a->T, chains, a->workspace);
    if (!a->gate.data || !a->update.data || !a->checkpoints || (g.count > 1 && !a->workspace)) return -1;
    OnDevice on(device);
    if (on.err != hipSuccess) return (int)on.err;
    return by_dtype(a->dtype, [&](auto e) {
        typedef decltype(e) E;
        if (a->T <= FEW)
            return by_few<E>(a, true, [&](auto vec, unsigned blocks) {
                recurrence_few_backward<E, decltype(vec)::value><<<blocks, 256, 0, (hipStream_t)stream>>>(*a);
                return launched();
            });
        return by_shape<2>(g, vec_for(a, true), [&](auto vec, auto waves) {
            constexpr int VEC = decltype(vec)::value, WAVES = decltype(waves)::value;
            const dim3 grid(chain_blocks(a, VEC), g.count), block(WAVE, std::min(WAVES, (a->T + KB - 1) / KB));
            if constexpr (VEC == 1) {
                if (g.count > 1) {
                    recurrence_segments<E, VEC, WAVES, true><<<grid, block, 0, (hipStream_t)stream>>>(*a, g);
                    if (int err = launched()) return err;
                }
            }
            recurrence_backward<E, VEC, WAVES><<<grid, block, 0, (hipStream_t)stream>>>(*a, g);
            return launched();
        });
    });
}

LIBENV_API int procgen_amd_advantages(const struct procgen_amd_advantage *a, int device, void *stream) {
    if (!a || !shape_ok(a->dtype, a->T, a->N, 1)) return -1;
    if (a->T == 0 || a->N == 0) return 0;
    const Segments g = segments(a->T, a->N, a->workspace, ENOUGH_ADVANTAGES);
    if (!a->rew || !a->values || !a->first || (g.count > 1 && !a->workspace)) return -1;
    OnDevice on(device);
    if (on.err != hipSuccess) return (int)on.err;
    return by_dtype(a->dtype, [&](auto e) {
        typedef decltype(e) E;
        const unsigned blocks = (a->N + WAVE - 1) / WAVE;
        if (g.count > 1) {
            const dim3 grid(blocks, g.count), block(WAVE, WS);
            advantage_segments<E, WS><<<grid, block, 0, (hipStream_t)stream>>>(*a, g);
            if (int err = launched()) return err;
            advantages<E, WS><<<grid, block, 0, (hipStream_t)stream>>>(*a, g);
        } else if (blocks < FULL) {  // 256 x 16384 float32: 15 us, with four waves 21
            advantages<E, WA><<<blocks, dim3(WAVE, std::min(WA, (a->T + KF - 1) / KF)), 0, (hipStream_t)stream>>>(*a, g);
        } else {
            advantages<E, W1><<<blocks, dim3(WAVE, std::min(W1, (a->T + KF - 1) / KF)), 0, (hipStream_t)stream>>>(*a, g);
        }
        return launched();
    });
}

}  // extern "C"
