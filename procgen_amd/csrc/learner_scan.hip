// learner_scan.hip -- recurrences along the steps of a rollout window: the gated linear recurrence of a policy's memory (forward, backward) and the
// advantages of its rewards, which are the same recurrence run from the last step to the first.
//
// A step is the affine map x -> a x + b, or x -> b where an episode begins (`cut`: a select, so that nothing of the other episode, NaN or infinite,
// passes).  Maps compose to maps of the same kind, so a chain is cut into pieces that are summed up at the same time and joined afterwards:
//   wave     K = 8 consecutive steps in registers, their composition (A, B, cut) by 8 FMAs
//   block    W <= 8 waves take consecutive pieces of a tile of 64 steps; the pieces' maps meet in LDS, every wave runs its value at the tile's start
//            through the pieces before its own, and does its steps again from there: one read and one write of the data, one barrier a tile
//   segment  where there are too few chains to fill the card, the window is cut into segments for blocks of their own: a first kernel composes each
//            segment's map, the second begins each segment with the maps of those before it (the data is read twice)
// Lanes are chains (VEC neighbouring channels each), so that every load of a step is one coalesced row piece.
#include "learner.h"

#include <algorithm>

namespace pgamd {
namespace learner {
namespace {

constexpr int K = 8, MAX_W = 8, TILE = K * MAX_W;

// the element types' rows of VEC neighbouring channels; `count` of them exist (the last lane of an env may hold fewer)
template <class E, int VEC>
struct Row {
    float x[VEC];
};
template <class E, int VEC>
__device__ inline Row<E, VEC> load_row(const typename E::T *p, int count) {
    Row<E, VEC> r;
    typename E::T raw[VEC];
    if (count == VEC) {
        __builtin_memcpy(raw, p, sizeof raw);  // one wide load, whatever the alignment
    } else {
        for (int v = 0; v < VEC; v++) raw[v] = v < count ? p[v] : (typename E::T)0.f;
    }
    for (int v = 0; v < VEC; v++) r.x[v] = (float)raw[v];
    return r;
}
template <class E, int VEC>
__device__ inline void store_row(typename E::T *p, int count, const Row<E, VEC> &r) {
    typename E::T raw[VEC];
    for (int v = 0; v < VEC; v++) raw[v] = (typename E::T)r.x[v];
    if (count == VEC) {
        __builtin_memcpy(p, raw, sizeof raw);
    } else {
        for (int v = 0; v < VEC; v++)
            if (v < count) p[v] = raw[v];
    }
}

template <int VEC>
struct Map {
    float A[VEC], B[VEC];
    bool cut;
    __device__ void identity() {
        cut = false;
        for (int v = 0; v < VEC; v++) A[v] = 1.f, B[v] = 0.f;
    }
    __device__ float at(float x, int v) const { return cut ? B[v] : fmaf(A[v], x, B[v]); }
    __device__ void then(const Map &m) {  // this map first, m behind it
        for (int v = 0; v < VEC; v++) {
            B[v] = m.at(B[v], v);
            A[v] = A[v] * m.A[v];
        }
        cut = cut || m.cut;
    }
};

// the pieces' maps of a tile, by wave and lane
template <int VEC>
struct Pieces {
    float A[MAX_W][VEC][WAVE], B[MAX_W][VEC][WAVE];
    int cut[MAX_W][WAVE];
    __device__ void put(int w, int lane, const Map<VEC> &m) {
        for (int v = 0; v < VEC; v++) A[w][v][lane] = m.A[v], B[w][v][lane] = m.B[v];
        cut[w][lane] = m.cut;
    }
    __device__ Map<VEC> get(int w, int lane) const {
        Map<VEC> m;
        for (int v = 0; v < VEC; v++) m.A[v] = A[w][v][lane], m.B[v] = B[w][v][lane];
        m.cut = cut[w][lane];
        return m;
    }
};

// where a lane's chains are: env n, channels d .. d + count - 1
template <int VEC>
struct Chain {
    int n, d, count;
    long long c;  // index of the first one in [N][D]
    __device__ Chain(long long unit, int N, int D) {
        const int lanes = (D + VEC - 1) / VEC;
        n = (int)(unit / lanes);
        d = (int)(unit - (long long)n * lanes) * VEC;
        count = n < N ? min(VEC, D - d) : 0;
        c = (long long)n * D + d;
    }
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
        if (v < ch.count) {
            g.maps[g.at(s, 0, chains, ch.c + v)] = m.A[v];
            g.maps[g.at(s, 1, chains, ch.c + v)] = m.B[v];
            g.cuts[s * chains + ch.c + v] = m.cut;
        }
}
template <int VEC>
__device__ inline Map<VEC> get_segment(const Segments &g, int s, long long chains, const Chain<VEC> &ch) {
    Map<VEC> m;
    m.identity();
    for (int v = 0; v < VEC; v++)
        if (v < ch.count) {
            m.A[v] = g.maps[g.at(s, 0, chains, ch.c + v)];
            m.B[v] = g.maps[g.at(s, 1, chains, ch.c + v)];
        }
    if (ch.count) m.cut = g.cuts[s * chains + ch.c];
    return m;
}

// x[] run through the segments [from, to) in order (to < from: downwards): the waves take a part each and join in LDS
template <int VEC>
__device__ inline void run_segments(float *x, const Segments &g, int from, int to, long long chains, const Chain<VEC> &ch, Pieces<VEC> &pieces, int w, int W, int lane) {
    const int n = abs(to - from), way = to < from ? -1 : 1, first = (int)((long long)n * w / W), last = (int)((long long)n * (w + 1) / W);
    Map<VEC> m;
    m.identity();
    for (int i = first; i < last; i++) m.then(get_segment<VEC>(g, from + way * i - (way < 0), chains, ch));
    pieces.put(w, lane, m);
    __syncthreads();
    for (int k = 0; k < W; k++) {
        const Map<VEC> q = pieces.get(k, lane);
        for (int v = 0; v < VEC; v++) x[v] = q.at(x[v], v);
    }
    __syncthreads();
}

template <class E, int VEC>
struct Recurrence {  // a lane's view of the arrays
    const procgen_amd_recurrence &p;
    const Chain<VEC> ch;
    const uint8_t *first;
    __device__ Recurrence(const procgen_amd_recurrence &args, long long unit)
        : p(args), ch(unit, args.N, args.D), first(args.first ? args.first + ch.n * args.first_n_stride : nullptr) {}
    __device__ typename E::T *at(const procgen_amd_array3 &a, int t) const {
        return (typename E::T *)a.data + t * a.t_stride + ch.n * a.n_stride + ch.d * a.d_stride;
    }
    __device__ Row<E, VEC> load(const procgen_amd_array3 &a, int t, bool real, float otherwise) const {
        if (real) return load_row<E, VEC>(at(a, t), ch.count);
        Row<E, VEC> r;
        for (int v = 0; v < VEC; v++) r.x[v] = otherwise;
        return r;
    }
    __device__ bool cut(int t, bool real) const { return real && first && first[t * p.first_t_stride]; }
};

// K steps of a wave, t .. t + K - 1 (those at `end` and behind it are the identity)
template <class E, int VEC, bool REVERSE>
__device__ inline Map<VEC> compose(const Row<E, VEC> *a, const Row<E, VEC> *b, const bool *cut) {
    Map<VEC> m;
    m.identity();
    for (int i = 0; i < K; i++) {
        const int k = REVERSE ? K - 1 - i : i;
        for (int v = 0; v < VEC; v++) {
            // backwards a step takes the gradient y of its h from behind to a (d + y) before it
            m.B[v] = REVERSE ? (cut[k] ? 0.f : a[k].x[v] * (b[k].x[v] + m.B[v])) : (cut[k] ? b[k].x[v] : fmaf(a[k].x[v], m.B[v], b[k].x[v]));
            m.A[v] *= a[k].x[v];
        }
        m.cut = m.cut || cut[k];
    }
    return m;
}

// the map of every segment (blockIdx.y): forwards of gate and update, backwards of gate and d_h.  The waves take a part of the segment each.
template <class E, int VEC, bool REVERSE>
__global__ __launch_bounds__(MAX_W *WAVE) void recurrence_segments(procgen_amd_recurrence p, Segments g) {
    __shared__ Pieces<VEC> pieces;
    const int lane = threadIdx.x, w = threadIdx.y, W = blockDim.y, s = blockIdx.y;
    const Recurrence<E, VEC> r(p, (long long)blockIdx.x * WAVE + lane);
    const long long chains = (long long)p.N * p.D;
    const int begin = s * g.tiles * TILE, end = min((long long)p.T, (long long)begin + (long long)g.tiles * TILE);
    const int part = (g.tiles * TILE + W * K - 1) / (W * K) * K;  // steps of a wave
    const int from = begin + w * part, to = min(end, from + part);
    Map<VEC> m;
    m.identity();
    for (int i = 0; i < part; i += K) {
        const int t = REVERSE ? from + part - K - i : from + i;
        Row<E, VEC> a[K], b[K];
        bool cut[K];
#pragma unroll
        for (int k = 0; k < K; k++) {
            const bool real = r.ch.count && t + k < to;
            a[k] = r.load(p.gate, t + k, real, 1.f);
            b[k] = r.load(REVERSE ? p.d_h : p.update, t + k, real && (!REVERSE || p.d_h.data), 0.f);
            cut[k] = r.cut(t + k, real);
        }
        m.then(compose<E, VEC, REVERSE>(a, b, cut));
    }
    pieces.put(w, lane, m);
    __syncthreads();
    if (w) return;
    m.identity();
    for (int k = 0; k < W; k++) m.then(pieces.get(REVERSE ? W - 1 - k : k, lane));
    put_segment<VEC>(g, s, chains, r.ch, m);
    if (!REVERSE && s == 0 && p.state)
        for (int v = 0; v < r.ch.count; v++) g.state[r.ch.c + v] = p.state[r.ch.c + v];
}

template <class E, int VEC>
__global__ __launch_bounds__(MAX_W *WAVE) void recurrence_forward(procgen_amd_recurrence p, Segments g) {
    __shared__ Pieces<VEC> pieces[2];
    const int lane = threadIdx.x, w = threadIdx.y, W = blockDim.y, s = blockIdx.y;
    const Recurrence<E, VEC> r(p, (long long)blockIdx.x * WAVE + lane);
    const long long chains = (long long)p.N * p.D;
    float x[VEC];
    for (int v = 0; v < VEC; v++) x[v] = p.state && v < r.ch.count ? (g.count > 1 ? g.state : p.state)[r.ch.c + v] : 0.f;
    if (s) run_segments<VEC>(x, g, 0, s, chains, r.ch, pieces[0], w, W, lane);
    const int begin = s * g.tiles * TILE, end = min((long long)p.T, (long long)begin + (long long)g.tiles * TILE);
    for (int t0 = begin, odd = 0; t0 < end; t0 += TILE, odd ^= 1) {
        const int t = t0 + w * K;
        Row<E, VEC> a[K], b[K];
        bool cut[K];
#pragma unroll
        for (int k = 0; k < K; k++) {
            const bool real = r.ch.count && t + k < end;
            a[k] = r.load(p.gate, t + k, real, 1.f);
            b[k] = r.load(p.update, t + k, real, 0.f);
            cut[k] = r.cut(t + k, real);
        }
        if (p.checkpoints && w == 0)
            for (int v = 0; v < VEC; v++)
                if (v < r.ch.count) p.checkpoints[(long long)(t0 / TILE) * chains + r.ch.c + v] = x[v];
        pieces[odd].put(w, lane, compose<E, VEC, false>(a, b, cut));
        __syncthreads();
        float y[VEC];
        for (int v = 0; v < VEC; v++) y[v] = x[v];
        for (int k = 0; k < W; k++) {
            const Map<VEC> q = pieces[odd].get(k, lane);
            for (int v = 0; v < VEC; v++) {
                if (k == w) y[v] = x[v];
                x[v] = q.at(x[v], v);
            }
        }
#pragma unroll
        for (int k = 0; k < K; k++) {
            Row<E, VEC> h;
            for (int v = 0; v < VEC; v++) h.x[v] = y[v] = cut[k] ? b[k].x[v] : fmaf(a[k].x[v], y[v], b[k].x[v]);
            if (r.ch.count && t + k < end) store_row<E, VEC>(r.at(p.h, t + k), r.ch.count, h);
        }
    }
    if (p.state_out && w == 0 && s == g.count - 1)
        for (int v = 0; v < VEC; v++)
            if (v < r.ch.count) p.state_out[r.ch.c + v] = x[v];
}

// Backwards over the tiles.  h is not read: its 32-bit value before every step comes from the checkpoint at the tile's start and the same joins as in
// the forward pass (update is read in its place, so the bytes are the same and 16-bit rounding of h does not reach d_gate).
template <class E, int VEC>
__global__ __launch_bounds__(MAX_W *WAVE) void recurrence_backward(procgen_amd_recurrence p, Segments g) {
    __shared__ Pieces<VEC> fore[2], back[2];
    const int lane = threadIdx.x, w = threadIdx.y, W = blockDim.y, s = blockIdx.y;
    const Recurrence<E, VEC> r(p, (long long)blockIdx.x * WAVE + lane);
    const long long chains = (long long)p.N * p.D;
    float y[VEC];  // what reaches h from the steps behind the tile
    for (int v = 0; v < VEC; v++) y[v] = p.d_state_out && v < r.ch.count ? p.d_state_out[r.ch.c + v] : 0.f;
    if (s < g.count - 1) run_segments<VEC>(y, g, g.count, s + 1, chains, r.ch, fore[0], w, W, lane);
    const int begin = s * g.tiles * TILE, end = min((long long)p.T, (long long)begin + (long long)g.tiles * TILE);
    for (int t0 = begin + (end - begin - 1) / TILE * TILE, odd = 0; t0 >= begin; t0 -= TILE, odd ^= 1) {
        const int t = t0 + w * K;
        Row<E, VEC> a[K], b[K], d[K];
        bool cut[K];
        float x[VEC], before[VEC], behind[VEC];
#pragma unroll
        for (int k = 0; k < K; k++) {
            const bool real = r.ch.count && t + k < end;
            a[k] = r.load(p.gate, t + k, real, 1.f);
            b[k] = r.load(p.update, t + k, real, 0.f);
            d[k] = r.load(p.d_h, t + k, real && p.d_h.data, 0.f);
            cut[k] = r.cut(t + k, real);
        }
        for (int v = 0; v < VEC; v++) x[v] = v < r.ch.count ? p.checkpoints[(long long)(t0 / TILE) * chains + r.ch.c + v] : 0.f;
        fore[odd].put(w, lane, compose<E, VEC, false>(a, b, cut));
        back[odd].put(w, lane, compose<E, VEC, true>(a, d, cut));
        __syncthreads();
        for (int v = 0; v < VEC; v++) before[v] = x[v], behind[v] = y[v];
        for (int k = 0; k < W; k++) {
            const Map<VEC> f = fore[odd].get(k, lane), q = back[odd].get(W - 1 - k, lane);
            for (int v = 0; v < VEC; v++) {
                if (k == w) before[v] = x[v];
                x[v] = f.at(x[v], v);
                if (W - 1 - k == w) behind[v] = y[v];
                y[v] = q.at(y[v], v);
            }
        }
#pragma unroll
        for (int k = 0; k < K; k++)  // b becomes the value before the step
            for (int v = 0; v < VEC; v++) {
                const float h = cut[k] ? b[k].x[v] : fmaf(a[k].x[v], before[v], b[k].x[v]);
                b[k].x[v] = before[v];
                before[v] = h;
            }
#pragma unroll
        for (int k = K - 1; k >= 0; k--) {
            for (int v = 0; v < VEC; v++) {
                const float gr = d[k].x[v] + behind[v];
                d[k].x[v] = gr;
                b[k].x[v] = cut[k] ? 0.f : gr * b[k].x[v];
                behind[v] = cut[k] ? 0.f : a[k].x[v] * gr;
            }
            if (r.ch.count && t + k < end) {
                if (p.d_update.data) store_row<E, VEC>(r.at(p.d_update, t + k), r.ch.count, d[k]);
                if (p.d_gate.data) store_row<E, VEC>(r.at(p.d_gate, t + k), r.ch.count, b[k]);
            }
        }
    }
    if (p.d_state && w == 0 && s == 0)
        for (int v = 0; v < VEC; v++)
            if (v < r.ch.count) p.d_state[r.ch.c + v] = y[v];
}

// ---- advantages: the recurrence adv[t] = (gamma lam) adv[t+1] + delta[t], from the last step to the first, a chain per env -----------------------------

template <class E>
struct Advantage {
    const procgen_amd_advantage &p;
    const int n;
    const float decay;
    const uint8_t *first;
    const typename E::T *values;
    const float *rew;
    __device__ Advantage(const procgen_amd_advantage &args, int env)
        : p(args), n(env), decay(args.gamma * args.lam), first(args.first + n * args.first_n_stride), values((const typename E::T *)args.values + n * args.values_n_stride),
          rew(args.rew + n * args.rew_n_stride) {}
    // steps t .. t + K - 1: cut[k], a[k] (1 where there is no step), b[k] = delta, v[k] = the value before the step
    __device__ void load(int t, int end, bool *cut, float *a, float *b, float *v) const {
        const bool here = n < p.N;
#pragma unroll
        for (int k = 0; k < K; k++) {
            const bool real = here && t + k < end;
            cut[k] = real && first[(t + k + 1) * p.first_t_stride];
            v[k] = real ? (float)values[(t + k) * p.values_t_stride] : 0.f;
            b[k] = real ? rew[(t + k) * p.rew_t_stride] : 0.f;
        }
        const int next = min(t + K, end);  // the value behind the last of these steps
        const float behind = here && t < end ? (float)values[next * p.values_t_stride] : 0.f;
#pragma unroll
        for (int k = 0; k < K; k++) {
            const bool real = here && t + k < end;
            const float after = k + 1 < K && t + k + 1 < end ? v[k + 1] : behind;
            a[k] = real ? decay : 1.f;
            b[k] = real ? (cut[k] ? b[k] : fmaf(p.gamma, after, b[k])) - v[k] : 0.f;
        }
    }
};
__device__ inline Map<1> compose_back(const bool *cut, const float *a, const float *b) {
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

template <class E>
__global__ __launch_bounds__(MAX_W *WAVE) void advantage_segments(procgen_amd_advantage p, Segments g) {
    __shared__ Pieces<1> pieces;
    const int lane = threadIdx.x, w = threadIdx.y, W = blockDim.y, s = blockIdx.y;
    const Advantage<E> r(p, blockIdx.x * WAVE + lane);
    const Chain<1> ch(blockIdx.x * WAVE + lane, p.N, 1);
    const int begin = s * g.tiles * TILE, end = min((long long)p.T, (long long)begin + (long long)g.tiles * TILE);
    const int part = (g.tiles * TILE + W * K - 1) / (W * K) * K;
    const int from = begin + w * part, to = min(end, from + part);
    Map<1> m;
    m.identity();
    for (int i = 0; i < part; i += K) {
        bool cut[K];
        float a[K], b[K], v[K];
        r.load(from + part - K - i, to, cut, a, b, v);
        m.then(compose_back(cut, a, b));
    }
    pieces.put(w, lane, m);
    __syncthreads();
    if (w) return;
    m.identity();
    for (int k = W - 1; k >= 0; k--) m.then(pieces.get(k, lane));
    put_segment<1>(g, s, p.N, ch, m);
}

template <class E>
__global__ __launch_bounds__(MAX_W *WAVE) void advantages(procgen_amd_advantage p, Segments g) {
    __shared__ Pieces<1> pieces[2];
    const int lane = threadIdx.x, w = threadIdx.y, W = blockDim.y, s = blockIdx.y;
    const Advantage<E> r(p, blockIdx.x * WAVE + lane);
    const Chain<1> ch(blockIdx.x * WAVE + lane, p.N, 1);
    float y = 0.f;
    if (s < g.count - 1) run_segments<1>(&y, g, g.count, s + 1, p.N, ch, pieces[0], w, W, lane);
    const int begin = s * g.tiles * TILE, end = min((long long)p.T, (long long)begin + (long long)g.tiles * TILE);
    for (int t0 = begin + (end - begin - 1) / TILE * TILE, odd = 0; t0 >= begin; t0 -= TILE, odd ^= 1) {
        const int t = t0 + w * K;
        bool cut[K];
        float a[K], b[K], v[K];
        r.load(t, end, cut, a, b, v);
        pieces[odd].put(w, lane, compose_back(cut, a, b));
        __syncthreads();
        float adv = y;
        for (int k = W - 1; k >= 0; k--) {
            if (k == w) adv = y;
            y = pieces[odd].get(k, lane).at(y, 0);
        }
#pragma unroll
        for (int k = K - 1; k >= 0; k--) {
            adv = cut[k] ? b[k] : fmaf(a[k], adv, b[k]);
            if (r.n < p.N && t + k < end) {
                if (p.adv) p.adv[(long long)(t + k) * p.N + r.n] = adv;
                if (p.ret) p.ret[(long long)(t + k) * p.N + r.n] = adv + v[k];
            }
        }
    }
}

// ---- launches ----------------------------------------------------------------------------------------------------------------------------------

bool shape_ok(int dtype, int T, int N, int D) { return known_dtype(dtype) && T >= 0 && T <= 0x7fffff00 && N >= 0 && D >= 0 && (long long)N * D <= 0x7fffff00ll; }

constexpr int FULL = 512;  // blocks of 8 waves that fill the card: two on each of the 256 compute units
int tiles_of(int T) { return (T + TILE - 1) / TILE; }
// how many segments a window of this many blocks' worth of chains is cut into: by its sizes alone, so that the workspace does not depend on strides
int segments_of(int T, long long chains) {
    const long long blocks = (chains + WAVE - 1) / WAVE;
    if (blocks >= FULL / 2) return 1;
    const long long wanted = (FULL + blocks - 1) / blocks, most = tiles_of(T) / 2;  // two tiles each at the least
    return (int)std::max(1ll, std::min(wanted, most));
}
Segments segments(int T, long long chains, void *workspace) {
    Segments g;
    const int wanted = segments_of(T, chains);
    g.tiles = (tiles_of(T) + wanted - 1) / wanted;
    g.count = (tiles_of(T) + g.tiles - 1) / g.tiles;
    g.maps = (float *)workspace;
    g.state = g.maps + 2ll * g.count * chains;
    g.cuts = (uint8_t *)(g.state + chains);
    return g;
}
long long segment_bytes(int T, long long chains) {
    const long long s = segments_of(T, chains);
    return s > 1 ? s * chains * 9 + chains * 4 : 0;
}

// neighbouring channels of a lane: as many as still leave enough blocks, where the arrays have them next to each other
int vec_for(const procgen_amd_recurrence *a, bool backward) {
    const procgen_amd_array3 *all[] = {&a->gate, &a->update, &a->h, &a->d_h, &a->d_gate, &a->d_update};
    for (int i = 0; i < (backward ? 6 : 3); i++)
        if (all[i]->data && all[i]->d_stride != 1 && a->D > 1) return 1;
    if (a->D == 1) return 1;
    for (int vec = backward ? 2 : 4; vec > 1; vec /= 2)
        if ((long long)a->N * ((a->D + vec - 1) / vec) >= (long long)FULL * WAVE) return vec;
    return 1;
}
template <class Fn>
int by_vec(int vec, Fn fn) {
    switch (vec) {
        case 4: return fn(std::integral_constant<int, 4>());
        case 2: return fn(std::integral_constant<int, 2>());
        default: return fn(std::integral_constant<int, 1>());
    }
}

}  // namespace
}  // namespace learner
}  // namespace pgamd

using namespace pgamd::learner;

extern "C" {

LIBENV_API long long procgen_amd_recurrence_checkpoints(int T) { return tiles_of(T); }
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
        return by_vec(vec_for(a, false), [&](auto vec) {
            typedef decltype(e) E;
            constexpr int VEC = decltype(vec)::value;
            const dim3 grid((unsigned)(((long long)a->N * ((a->D + VEC - 1) / VEC) + WAVE - 1) / WAVE), g.count), block(WAVE, std::min(MAX_W, (a->T + K - 1) / K));
            if (g.count > 1) {
                recurrence_segments<E, VEC, false><<<grid, block, 0, (hipStream_t)stream>>>(*a, g);
                if (int err = launched()) return err;
            }
            recurrence_forward<E, VEC><<<grid, block, 0, (hipStream_t)stream>>>(*a, g);
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
        return by_vec(vec_for(a, true), [&](auto vec) {
            typedef decltype(e) E;
            constexpr int VEC = std::min(2, decltype(vec)::value);  // four channels a lane take 187 registers: one block on a compute unit
            const dim3 grid((unsigned)(((long long)a->N * ((a->D + VEC - 1) / VEC) + WAVE - 1) / WAVE), g.count), block(WAVE, std::min(MAX_W, (a->T + K - 1) / K));
            if (g.count > 1) {
                recurrence_segments<E, VEC, true><<<grid, block, 0, (hipStream_t)stream>>>(*a, g);
                if (int err = launched()) return err;
            }
            recurrence_backward<E, VEC><<<grid, block, 0, (hipStream_t)stream>>>(*a, g);
            return launched();
        });
    });
}

LIBENV_API int procgen_amd_advantages(const struct procgen_amd_advantage *a, int device, void *stream) {
    if (!a || !shape_ok(a->dtype, a->T, a->N, 1)) return -1;
    if (a->T == 0 || a->N == 0) return 0;
    const Segments g = segments(a->T, a->N, a->workspace);
    if (!a->rew || !a->values || !a->first || (g.count > 1 && !a->workspace)) return -1;
    OnDevice on(device);
    if (on.err != hipSuccess) return (int)on.err;
    return by_dtype(a->dtype, [&](auto e) {
        typedef decltype(e) E;
        const dim3 grid((a->N + WAVE - 1) / WAVE, g.count), block(WAVE, std::min(MAX_W, (a->T + K - 1) / K));
        if (g.count > 1) {
            advantage_segments<E><<<grid, block, 0, (hipStream_t)stream>>>(*a, g);
            if (int err = launched()) return err;
        }
        advantages<E><<<grid, block, 0, (hipStream_t)stream>>>(*a, g);
        return launched();
    });
}

}  // extern "C"
