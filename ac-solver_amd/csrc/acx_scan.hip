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
// The state is float32 all the way.  The gradient needs h_(t-1) unrounded: the forward pass leaves the state in front of every segment
// (4 bytes for 16 steps) and the backward pass runs the segment again from it in registers, which also saves it reading h.
// k_t = 0 SELECTS zero: an infinite or NaN state of the last episode does not reach the next one through 0 * inf.
#include <type_traits>

#include "acx_elem.h"

namespace acx {
namespace scan {
using namespace elem;

constexpr int kSeg = 16;  // steps of a segment

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

struct Lane {
    int64_t n;
    int d;
};
// (the last lane of a row that V does not divide steps back and computes a few channels a second time: the same values, stored twice;
// the same for the lanes behind the last row)
template <int V> __device__ __forceinline__ Lane lane_of(const Args& p) {
    const int64_t l = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
    int64_t n = l / p.lpr;
    int j = (int)(l - n * p.lpr);
    if (n >= p.N) {
        n = p.N - 1;
        j = 0;
    }
    const int d = j * V;
    return {n, d + V <= p.D ? d : p.D - V};
}

// one segment's operands; steps at or behind `end` read the last step (in bounds) and are made the identity by the caller
template <class E, int V> __device__ __forceinline__ void load_segment(const void* base, int64_t st, int64_t t0, int64_t end, float (&out)[kSeg][V]) {
    const E* p = (const E*)base + t0 * st;
#pragma unroll
    for (int k = 0; k < kSeg; k++) {
        load<E, V>(p, out[k]);
        if (t0 + k + 1 < end) p += st;  // (uniform)
    }
}
__device__ __forceinline__ uint32_t load_resets(const Args& p, int64_t n, int64_t t0, int64_t end) {
    uint32_t bits = 0;
    if (p.reset) {
        const uint8_t* r = p.reset + t0 * p.N + n;
#pragma unroll
        for (int k = 0; k < kSeg; k++) {
            bits |= (uint32_t)(*r != 0) << k;
            if (t0 + k + 1 < end) r += p.N;
        }
    }
    return bits;
}

// FINAL: write h, last, bounds.  Otherwise only compose the chunk (agg).
template <class E, int V, int W, bool FINAL> __global__ void __launch_bounds__(64 * W) k_scan_fwd(const Args p) {
    constexpr bool kPrecise = sizeof(E) == 4;
    __shared__ Affine s_map[W > 1 ? 2 : 1][W][64 * V];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Lane me = lane_of<V>(p);
    const int64_t ch = me.n * p.D + me.d, nd = p.N * p.D;
    const int64_t begin = (int64_t)blockIdx.y * p.chunk, end = begin + p.chunk < p.T ? begin + p.chunk : p.T;
    const E* cp = (const E*)p.c + me.n * p.c_sn + me.d;
    const E* zp = (const E*)p.z + me.n * p.z_sn + me.d;
    E* hp = (E*)p.h + ch;
    Affine carry[V];  // FINAL: the state (in b); else the chunk so far
#pragma unroll
    for (int i = 0; i < V; i++) carry[i] = {FINAL ? -1.0f : 1.0f, 0.0f};
    if constexpr (FINAL) {
        if (p.state) {
#pragma unroll
            for (int i = 0; i < V; i++) carry[i].b = p.state[ch + i];
        }
        for (unsigned q = 0; q < blockIdx.y; q++) {
            const float* m = p.agg + (int64_t)q * 2 * nd + ch;
#pragma unroll
            for (int i = 0; i < V; i++) carry[i].b = apply({m[i], m[nd + i]}, carry[i].b);
        }
    }
    auto join = [](Affine second, Affine first) -> Affine {
        return {second.a < 0.0f || first.a < 0.0f ? -1.0f : second.a * first.a, apply(second, first.b)};
    };
    int buf = 0;
    for (int64_t tile = begin; tile < end; tile += W * kSeg, buf ^= 1) {
        const int64_t t0 = tile + w * kSeg;
        float f[kSeg][V], b[kSeg][V];
        uint32_t resets = 0;
        if (t0 < end) {
            load_segment<E, V>(zp, p.z_st, t0, end, f);
            load_segment<E, V>(cp, p.c_st, t0, end, b);
            resets = load_resets(p, me.n, t0, end);
        }
#pragma unroll
        for (int k = 0; k < kSeg; k++) {
            const bool in = t0 + k < end;
#pragma unroll
            for (int i = 0; i < V; i++) {
                const float z = f[k][i], s = small_sigmoid<kPrecise>(z);
                f[k][i] = in ? keep_of(z, s) : 1.0f;
                b[k][i] = in ? take_of(z, s) * b[k][i] : 0.0f;
            }
            if (!in) resets &= ~(1u << k);
        }
        Affine at[V];  // what stands in front of this segment
#pragma unroll
        for (int i = 0; i < V; i++) at[i] = carry[i];
        if constexpr (W > 1 || !FINAL) {
            Affine m[V];
#pragma unroll
            for (int i = 0; i < V; i++) {
                float a = 1.0f, h = 0.0f;
#pragma unroll
                for (int k = 0; k < kSeg; k++) {
                    const bool r = resets >> k & 1;
                    a *= f[k][i];
                    h = __builtin_fmaf(f[k][i], r ? 0.0f : h, b[k][i]);
                }
                m[i] = {resets ? -1.0f : a, h};
            }
            if constexpr (W == 1) {
#pragma unroll
                for (int i = 0; i < V; i++) carry[i] = join(m[i], carry[i]);
            } else {
#pragma unroll
                for (int i = 0; i < V; i++) s_map[buf][w][i * 64 + lane] = m[i];
                __syncthreads();  // (two buffers: the next tile's maps go into the other one, so one barrier a tile is enough)
                for (int q = 0; q < W; q++) {
#pragma unroll
                    for (int i = 0; i < V; i++) {
                        if (q == w) at[i] = carry[i];
                        carry[i] = join(s_map[buf][q][i * 64 + lane], carry[i]);
                    }
                }
            }
        }
        if constexpr (FINAL) {
            if (t0 < end) {
                float h[V];
#pragma unroll
                for (int i = 0; i < V; i++) h[i] = at[i].b;
                if (p.bounds) store<float, V>(p.bounds + (t0 / kSeg) * nd + ch, h);
                E* out = hp + t0 * nd;
#pragma unroll
                for (int k = 0; k < kSeg; k++) {
                    const bool r = resets >> k & 1;
#pragma unroll
                    for (int i = 0; i < V; i++) h[i] = __builtin_fmaf(f[k][i], r ? 0.0f : h[i], b[k][i]);
                    if (t0 + k < end) {
                        store<E, V>(out, h);
                        out += nd;
                    }
                }
                if constexpr (W == 1) {
#pragma unroll
                    for (int i = 0; i < V; i++) carry[i].b = h[i];
                }
            }
        }
    }
    if constexpr (FINAL) {
        if (w == 0 && end == p.T) {
            float h[V];
#pragma unroll
            for (int i = 0; i < V; i++) h[i] = carry[i].b;
            store<float, V>(p.last + ch, h);
        }
    } else {
        if (w == 0) {
            float a[V], b[V];
#pragma unroll
            for (int i = 0; i < V; i++) a[i] = carry[i].a, b[i] = carry[i].b;
            float* m = p.agg + (int64_t)blockIdx.y * 2 * nd + ch;
            store<float, V>(m, a);
            store<float, V>(m + nd, b);
        }
    }
}

// The gradient runs from the last step to the first on X_t = what step t + 1 hands back (X_(T-1) = dlast): G_t = dh_t + X_t,
// X_(t-1) = f_t k_t G_t; a segment is the map X -> A X + B of the X behind it to the X in front of it.
template <class E, int V, int W, bool FINAL> __global__ void __launch_bounds__(64 * W) k_scan_bwd(const Args p) {
    constexpr bool kPrecise = sizeof(E) == 4;
    __shared__ Affine s_map[W > 1 ? 2 : 1][W][64 * V];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Lane me = lane_of<V>(p);
    const int64_t ch = me.n * p.D + me.d, nd = p.N * p.D;
    const int64_t begin = (int64_t)blockIdx.y * p.chunk, end = begin + p.chunk < p.T ? begin + p.chunk : p.T;
    const E* cp = (const E*)p.c + me.n * p.c_sn + me.d;
    const E* zp = (const E*)p.z + me.n * p.z_sn + me.d;
    const E* gp = (const E*)p.dh + me.n * p.dh_sn + me.d;
    E* dcp = (E*)p.dc + me.n * p.dc_sn + me.d;
    E* dzp = (E*)p.dz + me.n * p.dz_sn + me.d;
    Affine carry[V];
#pragma unroll
    for (int i = 0; i < V; i++) carry[i] = {FINAL ? -1.0f : 1.0f, 0.0f};
    if constexpr (FINAL) {
        if (p.dlast) {
#pragma unroll
            for (int i = 0; i < V; i++) carry[i].b = p.dlast[ch + i];
        }
        for (unsigned q = gridDim.y - 1; q > blockIdx.y; q--) {
            const float* m = p.agg + (int64_t)q * 2 * nd + ch;
#pragma unroll
            for (int i = 0; i < V; i++) carry[i].b = apply({m[i], m[nd + i]}, carry[i].b);
        }
    }
    auto join = [](Affine second, Affine first) -> Affine {
        return {second.a < 0.0f || first.a < 0.0f ? -1.0f : second.a * first.a, apply(second, first.b)};
    };
    int buf = 0;
    const int64_t tiles = (end - begin + W * kSeg - 1) / (W * kSeg);
    for (int64_t tile = begin + (tiles - 1) * (W * kSeg); tile >= begin; tile -= W * kSeg, buf ^= 1) {
        const int64_t t0 = tile + w * kSeg;
        float s[kSeg][V], diff[kSeg][V], g[kSeg][V];  // +-small_sigmoid (the sign is z's), k h_(t-1) - c, dh
        uint32_t resets = 0, steps = 0;
        if (t0 < end) {
            steps = end - t0 < kSeg ? (uint32_t)(end - t0) : kSeg;
            load_segment<E, V>(zp, p.z_st, t0, end, s);
            load_segment<E, V>(gp, p.dh_st, t0, end, g);
            resets = load_resets(p, me.n, t0, end);
            if constexpr (FINAL) load_segment<E, V>(cp, p.c_st, t0, end, diff);
        }
        if (steps < kSeg) resets &= (1u << steps) - 1;
        // the sign of s tells which side of zero z was on: f = s for z < 0 (s held as -s), else 1 - s
        auto fkeep = [](float v) { return __builtin_signbitf(v) ? -v : 1.0f - v; };
        auto ftake = [](float v) { return __builtin_signbitf(v) ? 1.0f + v : v; };
#pragma unroll
        for (int k = 0; k < kSeg; k++) {
            const bool in = (uint32_t)k < steps;
#pragma unroll
            for (int i = 0; i < V; i++) {
                const float z = s[k][i], v = small_sigmoid<kPrecise>(z);
                s[k][i] = in ? (z < 0.0f ? -v : v) : 0.0f;  // (a step behind the end: f = 1)
                g[k][i] = in ? g[k][i] : 0.0f;
            }
        }
        if constexpr (FINAL) {
            if (t0 < end) {
                float h[V];
                load<float, V>(p.bounds + (t0 / kSeg) * nd + ch, h);
#pragma unroll
                for (int k = 0; k < kSeg; k++) {
                    const bool r = resets >> k & 1;
#pragma unroll
                    for (int i = 0; i < V; i++) {
                        const float c = diff[k][i], before = r ? 0.0f : h[i];
                        h[i] = __builtin_fmaf(fkeep(s[k][i]), before, ftake(s[k][i]) * c);
                        diff[k][i] = before - c;
                    }
                }
            }
        }
        float x[V];  // X behind this segment
#pragma unroll
        for (int i = 0; i < V; i++) x[i] = carry[i].b;
        if constexpr (W > 1 || !FINAL) {
            Affine m[V];
#pragma unroll
            for (int i = 0; i < V; i++) {
                float a = 1.0f, b = 0.0f;
#pragma unroll
                for (int k = kSeg - 1; k >= 0; k--) {
                    const bool r = resets >> k & 1;
                    const float f = fkeep(s[k][i]);
                    a *= f;
                    b = r ? 0.0f : f * (g[k][i] + b);
                }
                m[i] = {resets ? -1.0f : a, b};
            }
            if constexpr (W == 1) {
#pragma unroll
                for (int i = 0; i < V; i++) carry[i] = join(m[i], carry[i]);
            } else {
#pragma unroll
                for (int i = 0; i < V; i++) s_map[buf][w][i * 64 + lane] = m[i];
                __syncthreads();
                for (int q = W - 1; q >= 0; q--) {
#pragma unroll
                    for (int i = 0; i < V; i++) {
                        if (q == w) x[i] = carry[i].b;
                        carry[i] = join(s_map[buf][q][i * 64 + lane], carry[i]);
                    }
                }
            }
        }
        if constexpr (FINAL) {
            if (t0 < end) {
#pragma unroll
                for (int k = kSeg - 1; k >= 0; k--) {
                    const bool r = resets >> k & 1;
                    float dc[V], dz[V];
#pragma unroll
                    for (int i = 0; i < V; i++) {
                        const float f = fkeep(s[k][i]), u = ftake(s[k][i]), G = g[k][i] + x[i];
                        dc[i] = u * G;
                        dz[i] = f * u * diff[k][i] * G;
                        x[i] = (uint32_t)k < steps ? (r ? 0.0f : f * G) : x[i];
                    }
                    if ((uint32_t)k < steps) {
                        store<E, V>(dcp + (t0 + k) * p.dc_st, dc);
                        store<E, V>(dzp + (t0 + k) * p.dz_st, dz);
                    }
                }
                if constexpr (W == 1) {
#pragma unroll
                    for (int i = 0; i < V; i++) carry[i].b = x[i];
                }
            }
        }
    }
    if constexpr (FINAL) {
        if (w == 0 && begin == 0 && p.dstate) {
            float d[V];
#pragma unroll
            for (int i = 0; i < V; i++) d[i] = carry[i].b;
            store<float, V>(p.dstate + ch, d);
        }
    } else {
        if (w == 0) {
            float a[V], b[V];
#pragma unroll
            for (int i = 0; i < V; i++) a[i] = carry[i].a, b[i] = carry[i].b;
            float* m = p.agg + (int64_t)blockIdx.y * 2 * nd + ch;
            store<float, V>(m, a);
            store<float, V>(m + nd, b);
        }
    }
}

// How a problem is cut: V channels a lane, W waves over time, `chunks` of `chunk` steps over the grid.
struct Plan {
    int v, w, lpr;
    int64_t groups, chunk, chunks;
};
static Plan plan_of(int64_t T, int64_t N, int64_t D, int dtype) {
    Plan p;
    p.v = D >= 2 ? 2 : 1;
    p.lpr = (int)((D + p.v - 1) / p.v);
    p.groups = (N * p.lpr + 63) / 64;
    const int64_t segments = (T + kSeg - 1) / kSeg;
    p.w = p.groups >= 2048 || segments == 1 ? 1 : p.groups >= 512 || segments <= 4 ? 4 : 16;
    p.chunks = 1;
    p.chunk = T;
    const int64_t tile = (int64_t)p.w * kSeg, tiles = (T + tile - 1) / tile;
    if (p.groups < 128 && tiles >= 16) {
        int64_t want = 256 / p.groups;
        if (want > 64) want = 64;
        if (want > tiles / 4) want = tiles / 4;
        p.chunk = (tiles + want - 1) / want * tile;
        p.chunks = (T + p.chunk - 1) / p.chunk;
    }
    return p;
}

template <class E, int V, int W> static void launch(bool forward, const Args& a, const Plan& p, hipStream_t st) {
    const dim3 block(64 * W);
    const unsigned gx = (unsigned)p.groups, gy = (unsigned)p.chunks;
    if (forward) {
        // (the last chunk's own map is not asked for by anyone, the first one's in the gradient neither; they cost nothing beside the others)
        if (gy > 1) hipLaunchKernelGGL((k_scan_fwd<E, V, W, false>), dim3(gx, gy), block, 0, st, a);
        hipLaunchKernelGGL((k_scan_fwd<E, V, W, true>), dim3(gx, gy), block, 0, st, a);
    } else {
        if (gy > 1) hipLaunchKernelGGL((k_scan_bwd<E, V, W, false>), dim3(gx, gy), block, 0, st, a);
        hipLaunchKernelGGL((k_scan_bwd<E, V, W, true>), dim3(gx, gy), block, 0, st, a);
    }
}
template <class E, int V> static void launch_w(bool forward, const Args& a, const Plan& p, hipStream_t st) {
    if (p.w == 1) launch<E, V, 1>(forward, a, p, st);
    else if (p.w == 4) launch<E, V, 4>(forward, a, p, st);
    else launch<E, V, 16>(forward, a, p, st);
}
static int run(bool forward, Args& a, int dtype, void* work, int64_t work_bytes, hipStream_t st, const char* who) {
    const Plan p = plan_of(a.T, a.N, a.D, dtype);
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
static int check_sizes(int64_t T, int64_t N, int64_t D, int dtype, const char* who) {
    if (dtype != ACX_F32 && dtype != ACX_BF16 && dtype != ACX_F16) return fail(ACX_E_INVAL, "%s: activations are ACX_F32, ACX_BF16 or ACX_F16", who);
    if (T < 0 || N < 0 || D < 0 || D > (1 << 20) || T > ((int64_t)1 << 40) || N > ((int64_t)1 << 31)) return fail(ACX_E_INVAL, "%s: bad sizes", who);
    if ((N * D) / 64 >= ((int64_t)1 << 31) || (T > 0 && N * D > ((int64_t)1 << 60) / T)) return fail(ACX_E_INVAL, "%s: too many channels", who);
    return ACX_OK;
}

}  // namespace scan
}  // namespace acx

using namespace acx;

extern "C" int64_t acx_scan_bounds_bytes(int64_t T, int64_t N, int64_t D) {
    if (T < 0 || N < 0 || D < 0) return 0;
    return (T + scan::kSeg - 1) / scan::kSeg * N * D * 4;
}
extern "C" int64_t acx_scan_workspace_bytes(int64_t T, int64_t N, int64_t D, int dtype) {
    if (T <= 0 || N <= 0 || D <= 0) return 0;
    const scan::Plan p = scan::plan_of(T, N, D, dtype);
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
    if (d_last == d_state) return fail(ACX_E_INVAL, "acx_scan_forward: the last state does not replace the first in place");
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
