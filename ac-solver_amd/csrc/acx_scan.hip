// acx_scan.hip -- the gated linear recurrence of the recurrent agent over a rollout, and its gradient.
//
//   f_t = sigmoid(z_t),   h_t = f_t k_t h_(t-1) + (1 - f_t) c_t,   k_t = 0 where an episode starts at step t, else 1
//   G_t = dh_t + f_(t+1) k_(t+1) G_(t+1)  (+ dlast at the last step)
//   dc_t = (1 - f_t) G_t,   dz_t = f_t (1 - f_t) (k_t h_(t-1) - c_t) G_t,   dstate = f_0 k_0 G_0
//
// Every channel (environment, feature) is a recurrence of its own along time; both directions are affine maps h -> A h + B whose
// composition is associative.  The work is a few dozen vector instructions per element against 3 elements of memory traffic forward and
// 5 backward: bound by HBM where there are channels enough, by the length of the chain where there are not.
//   - A lane owns V neighbouring channels and a SEGMENT of kSeg steps in registers; a wave reads 64 V contiguous elements per step.
//   - W waves of a workgroup take W consecutive segments of the same channels: each composes its own segment, the W maps meet in LDS, and
//     every wave applies the maps before it (behind it in the gradient).  W = 1 where the channels alone fill the chip.
//   - Few channels and many steps: the steps are also cut into chunks over the grid; a first launch composes each chunk, and the second
//     one (the same kernel) folds the chunks before its own.  That reads the operands twice, from the caches mostly.
// Measured: 32 x 32768 x 256 f32 forward 0.59 ms, backward 1.01 ms, 5.6 and 5.4 TB/s of what they move (a copy kernel of torch: 4.8);
// 2000 x 4 x 256 f32 35 us and 32769 x 3 x 130 bf16 126 us for both together, where the vector pipe (25 instructions an element in a composed
// chunk, 37 forward, 58 backward, two of them transcendental) and the second reading share the time with the memory.
// The state is float32 all the way.  The gradient needs h_(t-1) unrounded: the forward pass leaves the state in front of every segment
// (4 bytes for 16 steps) and the backward pass runs the segment again from it in registers, which also saves it reading h.
// k_t = 0 SELECTS zero: an infinite or NaN state of the last episode does not reach the next one through 0 * inf.
#include <initializer_list>
#include <type_traits>

#include "acx_elem.h"

namespace acx {
namespace scan {
using namespace elem;

constexpr int kSeg = 16;  // steps of a segment
template <int V, int W> constexpr bool kCut = V == 1 && W == 8;  // variants that the steps are cut into chunks for (plan_of)

struct Args {
    const void *c, *z, *dh;       // candidate, gate, gradient of hidden
    int64_t c_st, c_sn, z_st, z_sn, dh_st, dh_sn;  // strides of step and row, in elements (features are contiguous)
    const uint8_t* reset;         // [T, N], nullable
    const float* state;           // [N, D], nullable: zero
    const float* dlast;           // [N, D], nullable
    int64_t T, N;
    int D, lpr;                   // features; lanes per row
    void* h;                      // [T, N, D]
    float* last;                  // [N, D]
    float* bounds;                // [segments, N, D], nullable: the state in front of every segment
    void *dc, *dz;
    int64_t dc_st, dc_sn, dz_st, dz_sn;
    float* dstate;                // nullable
    float* agg;                   // [chunks, 2, N, D] composed chunks
    int64_t chunk;                // steps of a chunk (a multiple of W kSeg); T where the steps are not cut
};

// h -> A h + B; A < 0 stands for "an episode starts inside": B, whatever h was
struct Affine {
    float a, b;
};
__device__ __forceinline__ float apply(Affine m, float h) { return m.a < 0.0f ? m.b : __builtin_fmaf(m.a, h, m.b); }

// A lane's place.  The lanes of a wave are neighbours in (row, feature): what differs between them fits 32 bits behind a base that the whole
// wave shares, so an access takes a scalar pointer that moves with the steps and one register of offset for all of them.  (The last lane of a
// row that V does not divide steps back and computes a few channels a second time: the same values, stored twice; the lanes behind the last
// row do its first channels again.)
struct Lane {
    int64_t n, n0;  // row; row of the wave's first lane
    int d;
    __device__ __forceinline__ uint32_t offset(int64_t sn, int bytes) const { return (uint32_t)(((n - n0) * sn + d) * bytes); }
};
template <int V> __device__ __forceinline__ Lane lane_of(const Args& p) {
    const int64_t l = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
    int64_t n = l / p.lpr;
    int j = (int)(l - n * p.lpr);
    if (n >= p.N) {
        n = p.N - 1;
        j = 0;
    }
    const int64_t n0 = (int64_t)blockIdx.x * 64 / p.lpr;
    const int d = j * V;
    return {n, n0, d + V <= p.D ? d : p.D - V};
}

// one segment's operands; steps at or behind `end` read the last step (in bounds) and are made the identity by the caller
template <class E, int V, bool STREAM> __device__ __forceinline__ void load_segment(const void* base, int64_t first, int64_t st, uint32_t offset, int64_t t0, int64_t end, float (&out)[kSeg][V]) {
    const char* p = (const char*)base + (first + t0 * st) * (int64_t)sizeof(E);  // (scalar)
#pragma unroll
    for (int k = 0; k < kSeg; k++) {
        load<E, V, STREAM>((const E*)(p + offset), out[k]);
        p += t0 + k + 1 < end ? st * (int64_t)sizeof(E) : 0;
    }
}
// Where an episode starts: one lane mask per step in scalar registers, so that a select on it is one instruction.  -> whether this lane has any.
// A wave over at most four rows reads all its 16 x 4 flags with one load, a lane each; most segments have none and are done with it.
__device__ __forceinline__ bool load_starts(const Args& p, const Lane& me, int64_t t0, int64_t end, bool (&start)[kSeg]) {
    const int lane = threadIdx.x & 63, mine = (int)(me.n - me.n0), rows = __builtin_amdgcn_readlane(mine, 63);
    if (rows < 4) {
        const int k = lane & 15, r = lane >> 4;
        const int64_t t = t0 + k < end ? t0 + k : end - 1;
        const bool flag = t0 + k < end && r <= rows && p.reset[t * p.N + me.n0 + (r <= rows ? r : 0)] != 0;
        const uint64_t all = __ballot(flag);
        if (all == 0) return false;
        uint32_t bits = (uint32_t)all & 0xFFFFu;
        if (rows > 0) {
            const uint32_t low = mine & 1 ? (uint32_t)all >> 16 : (uint32_t)all & 0xFFFFu, high = mine & 1 ? (uint32_t)(all >> 32) >> 16 : (uint32_t)(all >> 32) & 0xFFFFu;
            bits = mine & 2 ? high : low;
        }
#pragma unroll
        for (int i = 0; i < kSeg; i++) start[i] = bits >> i & 1;
        return bits != 0;
    }
    bool any = false;
    const uint8_t* r = p.reset + t0 * p.N + me.n0;
#pragma unroll
    for (int k = 0; k < kSeg; k++) {
        start[k] = t0 + k < end && r[(uint32_t)mine] != 0;
        any |= start[k];
        r += t0 + k + 1 < end ? p.N : 0;
    }
    return any;
}
// `second` behind `first`
__device__ __forceinline__ Affine join(Affine second, Affine first) {
    return {second.a < 0.0f || first.a < 0.0f ? -1.0f : second.a * first.a, apply(second, first.b)};
}
// The chunks in front of this one (FORWARD; else those behind it), folded into `carry`: every wave composes a few of them, the waves' maps
// meet in LDS.
template <int V, int W, bool FORWARD> __device__ __forceinline__ void fold_chunks(const Args& p, int64_t ch, int64_t nd, int lane, int w, Affine (&s_map)[W][64 * V], float (&carry)[V]) {
    const int n = FORWARD ? (int)blockIdx.y : (int)(gridDim.y - 1 - blockIdx.y), per = (n + W - 1) / W;
    Affine m[V];
#pragma unroll
    for (int i = 0; i < V; i++) m[i] = {1.0f, 0.0f};
    const int k1 = (w + 1) * per < n ? (w + 1) * per : n;
    for (int k = w * per; k < k1; k++) {
        const int q = FORWARD ? k : (int)gridDim.y - 1 - k;
        float a[V], b[V];
        load<float, V>(p.agg + (int64_t)q * 2 * nd + ch, a);
        load<float, V>(p.agg + (int64_t)q * 2 * nd + nd + ch, b);
#pragma unroll
        for (int i = 0; i < V; i++) m[i] = join({a[i], b[i]}, m[i]);
    }
#pragma unroll
    for (int i = 0; i < V; i++) s_map[w][i * 64 + lane] = m[i];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < W; k++)
#pragma unroll
        for (int i = 0; i < V; i++) carry[i] = apply(s_map[k][i * 64 + lane], carry[i]);
    __syncthreads();
}
// This wave's place among the maps of a tile: `mine` in LDS, what the waves before it (w0 = 0, step = 1) or behind it (w0 = W - 1, step = -1) do to
// `carry` into `front`, what all of them do into `carry`.  Two buffers take turns, so one barrier a tile is enough.
template <int V, int W, bool FORWARD> __device__ __forceinline__ void meet(Affine (&s_map)[W][64 * V], int lane, int w, const Affine (&mine)[V], Affine (&carry)[V], float (&front)[V]) {
#pragma unroll
    for (int i = 0; i < V; i++) s_map[w][i * 64 + lane] = mine[i];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < W; k++) {
        const int q = FORWARD ? k : W - 1 - k;
#pragma unroll
        for (int i = 0; i < V; i++) {
            front[i] = q == w ? carry[i].b : front[i];
            carry[i] = join(s_map[q][i * 64 + lane], carry[i]);
        }
    }
}

// f and 1 - f of a segment.  COMPACT holds one register for the two, the smaller one with the sign of z, and makes the larger one from it where it
// is needed (the compiler would keep both across the passes over a segment: `forget` stops it); for two channels a lane.
template <int V, bool COMPACT> struct Gates {
    float s[kSeg][V];
    float u[COMPACT ? 1 : kSeg][COMPACT ? 1 : V];
    template <bool PRECISE> __device__ __forceinline__ void set(int k, int i, float z) {
        const Sigmoid q = sigmoid_pair<PRECISE>(z);
        if constexpr (COMPACT) {
            s[k][i] = __builtin_copysignf(q.small, z);
        } else {
            s[k][i] = keep_of(z, q);
            u[k][i] = take_of(z, q);
        }
    }
    __device__ __forceinline__ void identity(int k, int i) {  // f = 1
        if constexpr (COMPACT) {
            s[k][i] = 0.0f;
        } else {
            s[k][i] = 1.0f;
            u[k][i] = 0.0f;
        }
    }
    __device__ __forceinline__ float f(int k, int i) const {
        if constexpr (COMPACT) return __builtin_signbitf(s[k][i]) ? -s[k][i] : 1.0f - s[k][i];
        else return s[k][i];
    }
    __device__ __forceinline__ float take(int k, int i) const {
        if constexpr (COMPACT) return __builtin_signbitf(s[k][i]) ? 1.0f + s[k][i] : s[k][i];
        else return u[k][i];
    }
    __device__ __forceinline__ void forget() {
        if constexpr (COMPACT) {
#pragma unroll
            for (int k = 0; k < kSeg; k++)
#pragma unroll
                for (int i = 0; i < V; i++) asm volatile("" : "+v"(s[k][i]));
        }
    }
};

// FINAL: write h, last, bounds.  Otherwise only compose the chunk (agg).
template <class E, int V, int W, bool FINAL, bool STREAM> __global__ void __launch_bounds__(64 * W) k_scan_fwd(const Args p) {
    constexpr bool kPrecise = sizeof(E) == 4;
    __shared__ Affine s_map[2][W][64 * V];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Lane me = lane_of<V>(p);
    const int64_t ch = me.n * p.D + me.d, nd = p.N * p.D;
    const int64_t begin = (int64_t)blockIdx.y * p.chunk, end = begin + p.chunk < p.T ? begin + p.chunk : p.T;
    const uint32_t c_off = me.offset(p.c_sn, sizeof(E)), z_off = me.offset(p.z_sn, sizeof(E)), h_off = me.offset(p.D, sizeof(E));
    Affine carry[V];  // FINAL: the state (in b); else the chunk so far
#pragma unroll
    for (int i = 0; i < V; i++) carry[i] = {FINAL ? -1.0f : 1.0f, 0.0f};
    if constexpr (FINAL) {
        float h[V] = {};
        if (p.state) load<float, V>(p.state + ch, h);
        if constexpr (kCut<V, W>)
            if (gridDim.y > 1) fold_chunks<V, W, true>(p, ch, nd, lane, w, s_map[1], h);
#pragma unroll
        for (int i = 0; i < V; i++) carry[i].b = h[i];
    }
    int buf = 0;
    for (int64_t tile = begin; tile < end; tile += W * kSeg, buf ^= 1) {
        const int64_t t0 = tile + w * kSeg;
        float f[kSeg][V], b[kSeg][V];
        bool start[kSeg] = {}, starts = false;
        if (t0 < end) {
            load_segment<E, V, STREAM>(p.z, me.n0 * p.z_sn, p.z_st, z_off, t0, end, f);
            load_segment<E, V, STREAM>(p.c, me.n0 * p.c_sn, p.c_st, c_off, t0, end, b);
            if (p.reset) starts = load_starts(p, me, t0, end, start);
        }
#pragma unroll
        for (int k = 0; k < kSeg; k++)
#pragma unroll
            for (int i = 0; i < V; i++) {
                const float z = f[k][i];
                const Sigmoid s = sigmoid_pair<kPrecise>(z);
                f[k][i] = keep_of(z, s);
                b[k][i] *= take_of(z, s);
            }
        if (t0 + kSeg > end) {  // (uniform) steps behind the end: the identity
#pragma unroll
            for (int k = 0; k < kSeg; k++)
#pragma unroll
                for (int i = 0; i < V; i++) {
                    f[k][i] = t0 + k < end ? f[k][i] : 1.0f;
                    b[k][i] = t0 + k < end ? b[k][i] : 0.0f;
                }
        }
        float h[V];
#pragma unroll
        for (int i = 0; i < V; i++) h[i] = carry[i].b;
        if constexpr (W > 1) {
            Affine m[V];
#pragma unroll
            for (int i = 0; i < V; i++) {
                float a = 1.0f, x = 0.0f;
#pragma unroll
                for (int k = 0; k < kSeg; k++) {
                    a *= f[k][i];
                    x = __builtin_fmaf(f[k][i], start[k] ? 0.0f : x, b[k][i]);
                }
                m[i] = {starts ? -1.0f : a, x};
            }
            meet<V, W, true>(s_map[buf], lane, w, m, carry, h);
        }
        if constexpr (FINAL) {
            if (t0 < end) {
                if (p.bounds) store<float, V>(p.bounds + (t0 / kSeg) * nd + ch, h);
                char* hp = (char*)p.h + (t0 * nd + me.n0 * p.D) * (int64_t)sizeof(E);
#pragma unroll
                for (int k = 0; k < kSeg; k++) {
#pragma unroll
                    for (int i = 0; i < V; i++) h[i] = __builtin_fmaf(f[k][i], start[k] ? 0.0f : h[i], b[k][i]);
                    if (t0 + k < end) store<E, V, STREAM>((E*)(hp + h_off), h);
                    hp += nd * (int64_t)sizeof(E);
                }
                if constexpr (W == 1) {
#pragma unroll
                    for (int i = 0; i < V; i++) carry[i].b = h[i];
                }
            }
        }
    }
    if (w == 0) {
        float a[V], b[V];
#pragma unroll
        for (int i = 0; i < V; i++) a[i] = carry[i].a, b[i] = carry[i].b;
        if constexpr (FINAL) {
            if (end == p.T) store<float, V>(p.last + ch, b);
        } else {
            store<float, V>(p.agg + (int64_t)blockIdx.y * 2 * nd + ch, a);
            store<float, V>(p.agg + (int64_t)blockIdx.y * 2 * nd + nd + ch, b);
        }
    }
}

// The gradient runs from the last step to the first on X_t = what step t + 1 hands back (X_(T-1) = dlast): G_t = dh_t + X_t,
// X_(t-1) = f_t k_t G_t; a segment is the map X -> A X + B of the X behind it to the X in front of it.
template <class E, int V, int W, bool FINAL, bool STREAM> __global__ void __launch_bounds__(64 * W) k_scan_bwd(const Args p) {
    constexpr bool kPrecise = sizeof(E) == 4;
    __shared__ Affine s_map[2][W][64 * V];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Lane me = lane_of<V>(p);
    const int64_t ch = me.n * p.D + me.d, nd = p.N * p.D;
    const int64_t begin = (int64_t)blockIdx.y * p.chunk, end = begin + p.chunk < p.T ? begin + p.chunk : p.T;
    const uint32_t c_off = me.offset(p.c_sn, sizeof(E)), z_off = me.offset(p.z_sn, sizeof(E)), g_off = me.offset(p.dh_sn, sizeof(E));
    const uint32_t dc_off = me.offset(p.dc_sn, sizeof(E)), dz_off = me.offset(p.dz_sn, sizeof(E));
    Affine carry[V];
#pragma unroll
    for (int i = 0; i < V; i++) carry[i] = {FINAL ? -1.0f : 1.0f, 0.0f};
    if constexpr (FINAL) {
        float x[V] = {};
        if (p.dlast) load<float, V>(p.dlast + ch, x);
        if constexpr (kCut<V, W>)
            if (gridDim.y > 1) fold_chunks<V, W, false>(p, ch, nd, lane, w, s_map[1], x);
#pragma unroll
        for (int i = 0; i < V; i++) carry[i].b = x[i];
    }
    int buf = 0;
    const int64_t tiles = (end - begin + W * kSeg - 1) / (W * kSeg);
    for (int64_t tile = begin + (tiles - 1) * (W * kSeg); tile >= begin; tile -= W * kSeg, buf ^= 1) {
        const int64_t t0 = tile + w * kSeg;
        Gates<V, (V > 1)> gate;
        float diff[kSeg][V], g[kSeg][V];  // c, then k h_(t-1) - c; dh
        bool start[kSeg] = {}, starts = false;
        if (t0 < end) {
            load_segment<E, V, STREAM>(p.z, me.n0 * p.z_sn, p.z_st, z_off, t0, end, gate.s);
            if constexpr (FINAL) load_segment<E, V, STREAM>(p.c, me.n0 * p.c_sn, p.c_st, c_off, t0, end, diff);
            load_segment<E, V, STREAM>(p.dh, me.n0 * p.dh_sn, p.dh_st, g_off, t0, end, g);
            if (p.reset) starts = load_starts(p, me, t0, end, start);
        }
#pragma unroll
        for (int k = 0; k < kSeg; k++)
#pragma unroll
            for (int i = 0; i < V; i++) gate.template set<kPrecise>(k, i, gate.s[k][i]);
        if (t0 + kSeg > end) {  // (uniform) steps behind the end: the identity
#pragma unroll
            for (int k = 0; k < kSeg; k++)
                if (t0 + k >= end) {
#pragma unroll
                    for (int i = 0; i < V; i++) gate.identity(k, i), g[k][i] = 0.0f;
                }
        }
        if constexpr (FINAL) {
            if (t0 < end) {
                float h[V];
                load<float, V>(p.bounds + (t0 / kSeg) * nd + ch, h);
#pragma unroll
                for (int k = 0; k < kSeg; k++) {
#pragma unroll
                    for (int i = 0; i < V; i++) {
                        const float c = diff[k][i], before = start[k] ? 0.0f : h[i];
                        h[i] = __builtin_fmaf(gate.f(k, i), before, gate.take(k, i) * c);
                        diff[k][i] = before - c;
                    }
                }
            }
        }
        gate.forget();
        float x[V];  // X behind this segment
#pragma unroll
        for (int i = 0; i < V; i++) x[i] = carry[i].b;
        if constexpr (W > 1) {
            Affine m[V];
#pragma unroll
            for (int i = 0; i < V; i++) {
                float a = 1.0f, b = 0.0f;
#pragma unroll
                for (int k = kSeg - 1; k >= 0; k--) {
                    const float f = gate.f(k, i);
                    a *= f;
                    b = start[k] ? 0.0f : f * (g[k][i] + b);
                }
                m[i] = {starts ? -1.0f : a, b};
            }
            meet<V, W, false>(s_map[buf], lane, w, m, carry, x);
            gate.forget();
        }
        if constexpr (FINAL) {
            if (t0 < end) {
                const int64_t dc_st = p.dc_st * (int64_t)sizeof(E), dz_st = p.dz_st * (int64_t)sizeof(E);
                char* dcp = (char*)p.dc + me.n0 * p.dc_sn * (int64_t)sizeof(E) + (t0 + kSeg - 1) * dc_st;
                char* dzp = (char*)p.dz + me.n0 * p.dz_sn * (int64_t)sizeof(E) + (t0 + kSeg - 1) * dz_st;
#pragma unroll
                for (int k = kSeg - 1; k >= 0; k--) {
                    if (t0 + k < end) {
                        float dc[V], dz[V];
#pragma unroll
                        for (int i = 0; i < V; i++) {
                            const float u = gate.take(k, i), G = g[k][i] + x[i];
                            dc[i] = u * G;
                            const float fG = gate.f(k, i) * G;
                            dz[i] = diff[k][i] * u * fG;
                            x[i] = start[k] ? 0.0f : fG;
                        }
                        store<E, V, STREAM>((E*)(dcp + dc_off), dc);
                        store<E, V, STREAM>((E*)(dzp + dz_off), dz);
                    }
                    dcp -= dc_st, dzp -= dz_st;
                }
                if constexpr (W == 1) {
#pragma unroll
                    for (int i = 0; i < V; i++) carry[i].b = x[i];
                }
            }
        }
    }
    if (w == 0) {
        float a[V], b[V];
#pragma unroll
        for (int i = 0; i < V; i++) a[i] = carry[i].a, b[i] = carry[i].b;
        if constexpr (FINAL) {
            if (begin == 0 && p.dstate) store<float, V>(p.dstate + ch, b);
        } else {
            store<float, V>(p.agg + (int64_t)blockIdx.y * 2 * nd + ch, a);
            store<float, V>(p.agg + (int64_t)blockIdx.y * 2 * nd + nd + ch, b);
        }
    }
}

// How a problem is cut: V channels a lane, W waves over time, `chunks` of `chunk` steps over the grid.
struct Plan {
    int v, w, lpr;
    int64_t groups, chunk, chunks;
};
static Plan plan_of(int64_t T, int64_t N, int64_t D) {
    Plan p;
    const int64_t segments = (T + kSeg - 1) / kSeg;
    auto groups = [&](int v) { return (N * ((D + v - 1) / v) + 63) / 64; };
    // (Times of one forward and one backward pass, episodes of about 200 steps.)  Two channels a lane where that leaves waves enough: 424 x 399 x 150 f32
    // 210 us, 236 with one; with 256 groups or fewer one channel is no slower and leaves more workgroups.
    p.v = D >= 2 && groups(2) >= 256 ? 2 : 1;
    p.lpr = (int)((D + p.v - 1) / p.v);
    p.groups = groups(p.v);
    // Eight waves a compute unit and more from the channels alone: a wave walks all steps.  Else the steps are shared by the waves of a workgroup, 16 where
    // there is about a workgroup for each compute unit (2709 x 19 x 846 bf16, 251 groups: 265 us, 289 with 8 waves) and 8 or 4 where there are more ...
    p.w = p.groups >= 2048 || segments == 1 ? 1 : p.v == 2 || segments <= 4 ? 4 : p.groups >= 128 && p.groups < 512 && segments > 8 ? 16 : 8;
    p.chunks = 1;
    p.chunk = T;
    // ... and where there are fewer, by the workgroups of a grid as well, though that reads the operands twice (2000 x 4 x 256 f32, 16 groups: 35 us, 147
    // in one chunk; 32769 x 3 x 130 bf16, 7 groups: 126 us, 2275 in one).  512 workgroups: that last one takes 149 us with 256 and 144 with 1024.
    const int64_t tile = (int64_t)p.w * kSeg, tiles = (T + tile - 1) / tile;
    if (p.groups < 128 && tiles >= 4) {
        int64_t want = 512 / p.groups;
        if (want > 128) want = 128;
        if (want > tiles) want = tiles;
        p.chunk = (tiles + want - 1) / want * tile;
        p.chunks = (T + p.chunk - 1) / p.chunk;
    }
    return p;
}

template <class E, int V, int W> static void launch(bool forward, const Args& a, const Plan& p, hipStream_t st) {
    const dim3 block(64 * W), grid((unsigned)p.groups, (unsigned)p.chunks);
    if constexpr (kCut<V, W>)
        if (p.chunks > 1) {  // (the last chunk's own map is not asked for by anyone, the first one's in the gradient neither; they cost nothing beside the others)
            if (forward) hipLaunchKernelGGL((k_scan_fwd<E, V, W, false, false>), grid, block, 0, st, a);
            else hipLaunchKernelGGL((k_scan_bwd<E, V, W, false, false>), grid, block, 0, st, a);
        }
    if (W == 1 && a.T * a.N * a.D * (int64_t)sizeof(E) > kStreamBytes) {
        if (forward) hipLaunchKernelGGL((k_scan_fwd<E, V, W, true, W == 1>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((k_scan_bwd<E, V, W, true, W == 1>), grid, block, 0, st, a);
    } else {
        if (forward) hipLaunchKernelGGL((k_scan_fwd<E, V, W, true, false>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((k_scan_bwd<E, V, W, true, false>), grid, block, 0, st, a);
    }
}
template <class E, int V> static void launch_w(bool forward, const Args& a, const Plan& p, hipStream_t st) {
    if (p.w == 1) launch<E, V, 1>(forward, a, p, st);
    else if (p.w == 4) launch<E, V, 4>(forward, a, p, st);
    else if constexpr (V == 1) {
        if (p.w == 8) launch<E, V, 8>(forward, a, p, st);
        else launch<E, V, 16>(forward, a, p, st);
    }
}
static int run(bool forward, Args& a, int dtype, void* work, int64_t work_bytes, hipStream_t st, const char* who) {
    const Plan p = plan_of(a.T, a.N, a.D);
    const int64_t need = p.chunks > 1 ? p.chunks * 2 * a.N * a.D * 4 : 0;
    if (work_bytes < need || (need && !work)) return fail(ACX_E_CAPACITY, "%s: a workspace of %lld bytes is needed (acx_scan_workspace_bytes)", who, (long long)need);
    a.agg = (float*)work;
    a.chunk = p.chunk;
    a.lpr = p.lpr;
    with_element(dtype, [&](auto* e) {
        using E = std::remove_pointer_t<decltype(e)>;
        if (p.v == 1) launch_w<E, 1>(forward, a, p, st);
        else launch_w<E, 2>(forward, a, p, st);
    });
    ACX_HIP_TRY(hipGetLastError());
    return ACX_OK;
}
// the rows of a wave within 32 bits of offset of each other (see Lane)
static bool strides_ok(int64_t D, int dtype, std::initializer_list<int64_t> rows) {
    const int64_t apart = 63 / ((D + 1) / 2) + 1;  // rows that a wave can span
    for (int64_t r : rows)
        if (r < 0 || r > (((int64_t)1 << 32) / element_bytes(dtype) - D) / apart) return false;
    return true;
}
// Whether two states [N, D] have memory in common: one workgroup reads the first where another one, of a later chunk or of the same channels (see Lane), may have
// written the second already.
static bool meet_in_memory(const float* a, const float* b, int64_t n) { return a && b && (a < b ? b - a : a - b) < n; }
static int check_sizes(int64_t T, int64_t N, int64_t D, int dtype, const char* who) {
    if (dtype != ACX_F32 && dtype != ACX_BF16 && dtype != ACX_F16) return fail(ACX_E_INVAL, "%s: activations are ACX_F32, ACX_BF16 or ACX_F16", who);
    if (T < 0 || N < 0 || D < 0 || D > (1 << 20) || T > ((int64_t)1 << 40) || N > ((int64_t)1 << 31)) return fail(ACX_E_INVAL, "%s: bad sizes", who);
    // (a launch has fewer than 2^32 lanes; so many channels have two of them each)
    if (N * ((D + 1) / 2) > ((int64_t)1 << 32) - 64 || (T > 0 && N * D > ((int64_t)1 << 60) / T)) return fail(ACX_E_INVAL, "%s: too many channels", who);
    return ACX_OK;
}

}  // namespace scan
}  // namespace acx

using namespace acx;

extern "C" int64_t acx_scan_bounds_bytes(int64_t T, int64_t N, int64_t D) {
    if (scan::check_sizes(T, N, D, ACX_F32, "acx_scan_bounds_bytes")) return 0;
    return (T + scan::kSeg - 1) / scan::kSeg * N * D * 4;
}
extern "C" int64_t acx_scan_workspace_bytes(int64_t T, int64_t N, int64_t D, int dtype) {
    if (scan::check_sizes(T, N, D, dtype, "acx_scan_workspace_bytes") || T == 0 || N == 0 || D == 0) return 0;
    const scan::Plan p = scan::plan_of(T, N, D);
    return p.chunks > 1 ? p.chunks * 2 * N * D * 4 : 0;
}
extern "C" int acx_scan_forward(const void* d_candidate, int64_t c_step, int64_t c_row, const void* d_gate, int64_t z_step, int64_t z_row, int dtype, const uint8_t* d_reset,
                                const float* d_state, int64_t T, int64_t N, int64_t D, void* d_hidden, float* d_last, float* d_bounds, void* d_work, int64_t work_bytes, void* stream) {
    if (!have_device()) return ACX_E_NODEVICE;
    const int rc = scan::check_sizes(T, N, D, dtype, "acx_scan_forward");
    if (rc) return rc;
    if (N == 0 || D == 0) return ACX_OK;
    if (T == 0) return fail(ACX_E_INVAL, "acx_scan_forward: no steps");
    if (!d_candidate || !d_gate || !d_hidden || !d_last) return fail(ACX_E_INVAL, "acx_scan_forward: null pointer");
    if (scan::meet_in_memory(d_last, d_state, N * D)) return fail(ACX_E_INVAL, "acx_scan_forward: the last state does not replace the first in place");
    if (!scan::strides_ok(D, dtype, {c_row, z_row})) return fail(ACX_E_INVAL, "acx_scan_forward: rows too far apart (4 GiB among the rows of 64 lanes)");
    scan::Args a = {};
    a.c = d_candidate, a.c_st = c_step, a.c_sn = c_row;
    a.z = d_gate, a.z_st = z_step, a.z_sn = z_row;
    a.reset = d_reset, a.state = d_state, a.T = T, a.N = N, a.D = (int)D;
    a.h = d_hidden, a.last = d_last, a.bounds = d_bounds;
    return scan::run(true, a, dtype, d_work, work_bytes, (hipStream_t)stream, "acx_scan_forward");
}
extern "C" int acx_scan_backward(const void* d_candidate, int64_t c_step, int64_t c_row, const void* d_gate, int64_t z_step, int64_t z_row, const void* d_hidden_grad, int64_t g_step,
                                 int64_t g_row, int dtype, const uint8_t* d_reset, const float* d_bounds, const float* d_last_grad, int64_t T, int64_t N, int64_t D,
                                 void* d_candidate_grad, int64_t dc_step, int64_t dc_row, void* d_gate_grad, int64_t dz_step, int64_t dz_row, float* d_state_grad, void* d_work,
                                 int64_t work_bytes, void* stream) {
    if (!have_device()) return ACX_E_NODEVICE;
    const int rc = scan::check_sizes(T, N, D, dtype, "acx_scan_backward");
    if (rc) return rc;
    if (N == 0 || D == 0) return ACX_OK;
    if (T == 0) return fail(ACX_E_INVAL, "acx_scan_backward: no steps");
    if (!d_candidate || !d_gate || !d_hidden_grad || !d_bounds || !d_candidate_grad || !d_gate_grad) return fail(ACX_E_INVAL, "acx_scan_backward: null pointer");
    if (scan::meet_in_memory(d_state_grad, d_last_grad, N * D))
        return fail(ACX_E_INVAL, "acx_scan_backward: the gradient of the first state does not replace that of the last in place");
    if (!scan::strides_ok(D, dtype, {c_row, z_row, g_row, dc_row, dz_row}))
        return fail(ACX_E_INVAL, "acx_scan_backward: rows too far apart (4 GiB among the rows of 64 lanes)");
    scan::Args a = {};
    a.c = d_candidate, a.c_st = c_step, a.c_sn = c_row;
    a.z = d_gate, a.z_st = z_step, a.z_sn = z_row;
    a.dh = d_hidden_grad, a.dh_st = g_step, a.dh_sn = g_row;
    a.reset = d_reset, a.dlast = d_last_grad, a.T = T, a.N = N, a.D = (int)D;
    a.bounds = const_cast<float*>(d_bounds);
    a.dc = d_candidate_grad, a.dc_st = dc_step, a.dc_sn = dc_row;
    a.dz = d_gate_grad, a.dz_st = dz_step, a.dz_sn = dz_row;
    a.dstate = d_state_grad;
    return scan::run(false, a, dtype, d_work, work_bytes, (hipStream_t)stream, "acx_scan_backward");
}
