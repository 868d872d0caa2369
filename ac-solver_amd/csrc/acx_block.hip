// acx_block.hip -- the end of a block of the recurrent agent: the norm behind the block, its gate and residual scale, and the norm in
// front of the next block, in one pass over the rows; the gradient of that; and the whole block for one step of the environments.
//
//   new = x + scale * silu(gate) * rms(y) weight,   u = rms(new) next_weight,   rms(v) = v / sqrt(mean(v^2) + eps)
//
// Forward: 3 rows read, 2 written, two row sums; backward: 5 read, 3 written, two row sums, and three sums over all rows (the gradients
// of weight, scale and next_weight).  About 50 vector instructions per element: bound by HBM.
//   - A row belongs to LR neighbouring lanes that hold all of it in registers, R vectors of V elements each (16 bytes a load); narrow rows
//     share a wave, rows over 64 lanes take a workgroup (row sums through LDS).
//   - The backward pass recomputes `new` from x, y and gate (it reads them anyway) unrounded and takes the two reciprocal roots of a row
//     from the forward pass (8 bytes a row instead of two more row sums).
//   - Sums over rows: every lane adds its features over the rows that its workgroup walks, the workgroup's row groups join in LDS, and a second
//     launch adds the workgroups' partial sums in a fixed order: the result does not depend on which workgroup came first.
#include <type_traits>

#include "acx_elem.h"

namespace acx {
namespace block {
using namespace elem;

struct Args {
    const void *x, *y, *g;           // y null: u = rms(x) next_weight alone; g null: no gate
    int64_t x_sn, y_sn, g_sn;        // row strides in elements
    const float *w, *scale, *next;   // [D]; scale null: 1; next null: no u
    float eps, inv_d;
    int64_t M;
    int D;
    void *out, *u;                   // contiguous
    float* stats;                    // [M, 2]: 1 / rms of y and of new; nullable in the forward pass
    // one step of the recurrence in front (k_block_fwd<STEP>): y is the new state, candidate / gate of it and the output gate lie in one row
    const void* proj;
    int64_t p_sn;
    const uint8_t* reset;
    const float* state;
    float* next_state;
    // gradient
    const void *d_out, *d_u;         // nullable
    int64_t do_sn, du_sn;
    void *dx, *dy, *dg;              // dx, dy contiguous
    int64_t dg_sn;
    float* partial;                  // [workgroups, 3, D]
};

// sum over the LR lanes of a row, in every one of them (s_red: one float per wave of the workgroup)
template <int LR> __device__ __forceinline__ float row_sum(float v, float* s_red) {
    v = lane_sum<(LR < 64 ? LR : 64)>(v);
    if constexpr (LR > 64) {
        constexpr int kWaves = LR / 64;
        __syncthreads();  // (the sums of the last call have been read)
        if ((threadIdx.x & 63) == 0) s_red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.0f;
        const float* mine = s_red + threadIdx.x / LR * kWaves;
#pragma unroll
        for (int i = 0; i < kWaves; i++) v += mine[i];
    }
    return v;
}

template <int V> __device__ __forceinline__ void load_weight(const float* p, int d, int D, float fallback, float (&out)[V]) {
#pragma unroll
    for (int i = 0; i < V; i++) out[i] = p && d + i < D ? p[d + i] : fallback;
}

template <class E, int V, int LR, int R, bool STEP> __global__ void __launch_bounds__(LR > 256 ? LR : 256) k_block_fwd(const Args p) {
    constexpr bool kPrecise = sizeof(E) == 4;
    constexpr int kThreads = LR > 256 ? LR : 256, kRows = kThreads / LR;
    __shared__ float s_red[kThreads / 64];
    const int j = threadIdx.x % LR;
    float w[R][V], scale[R][V], next[R][V];
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int d = (r * LR + j) * V;
        load_weight<V>(p.w, d, p.D, 0.0f, w[r]);
        load_weight<V>(p.scale, d, p.D, 1.0f, scale[r]);
        load_weight<V>(p.next, d, p.D, 0.0f, next[r]);
    }
    for (int64_t row0 = (int64_t)blockIdx.x * kRows; row0 < p.M; row0 += (int64_t)gridDim.x * kRows) {
        const int64_t row = row0 + threadIdx.x / LR;
        const bool live = row < p.M;  // (lanes behind the last row run along for the row sums)
        float x[R][V], y[R][V], g[R][V];
        float sum = 0.0f;
#pragma unroll
        for (int r = 0; r < R; r++) {
            const int d = (r * LR + j) * V, valid = live ? p.D - d : 0;
            load_some<E, V>((const E*)p.x + row * p.x_sn + d, valid, x[r]);
            if constexpr (STEP) {
                const E* proj = (const E*)p.proj + row * p.p_sn + d;
                float c[V], z[V], h[V];
                load_some<E, V>(proj, valid, c);
                load_some<E, V>(proj + p.D, valid, z);
                load_some<E, V>(proj + 2 * (int64_t)p.D, valid, g[r]);
                load_some<float, V>(p.state + row * p.D + d, valid, h);
                const bool start = live && p.reset && p.reset[row];
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const Sigmoid s = sigmoid_pair<kPrecise>(z[i]);
                    y[r][i] = __builtin_fmaf(keep_of(z[i], s), start ? 0.0f : h[i], take_of(z[i], s) * c[i]);
                }
                store_some<float, V>(p.next_state + row * p.D + d, valid, y[r]);
            } else if (p.y) {
                load_some<E, V>((const E*)p.y + row * p.y_sn + d, valid, y[r]);
                if (p.g) load_some<E, V>((const E*)p.g + row * p.g_sn + d, valid, g[r]);
            }
            if (STEP || p.y) {
#pragma unroll
                for (int i = 0; i < V; i++) sum = i < valid ? __builtin_fmaf(y[r][i], y[r][i], sum) : sum;
            }
        }
        float ry = 0.0f;
        if (STEP || p.y) {
            ry = rsqrtf(__builtin_fmaf(row_sum<LR>(sum, s_red), p.inv_d, p.eps));
            sum = 0.0f;
        }
#pragma unroll
        for (int r = 0; r < R; r++) {
            const int d = (r * LR + j) * V, valid = live ? p.D - d : 0;
            if (STEP || p.y) {
#pragma unroll
                for (int i = 0; i < V; i++) {
                    float a = scale[r][i];
                    if (STEP || p.g) {
                        const float gv = g[r][i];
                        a *= gv * keep_of(gv, sigmoid_pair<kPrecise>(gv));
                    }
                    x[r][i] = __builtin_fmaf(a, y[r][i] * ry * w[r][i], x[r][i]);
                }
                store_some<E, V>((E*)p.out + row * p.D + d, valid, x[r]);
            }
#pragma unroll
            for (int i = 0; i < V; i++) sum = i < valid ? __builtin_fmaf(x[r][i], x[r][i], sum) : sum;
        }
        float rx = 0.0f;
        if (p.next) {
            rx = rsqrtf(__builtin_fmaf(row_sum<LR>(sum, s_red), p.inv_d, p.eps));
#pragma unroll
            for (int r = 0; r < R; r++) {
                const int d = (r * LR + j) * V, valid = live ? p.D - d : 0;
                float u[V];
#pragma unroll
                for (int i = 0; i < V; i++) u[i] = x[r][i] * rx * next[r][i];
                store_some<E, V>((E*)p.u + row * p.D + d, valid, u);
            }
        }
        if (!STEP && p.stats && live && j == 0) {
            p.stats[2 * row] = ry;
            p.stats[2 * row + 1] = rx;
        }
    }
}

template <class E, int V, int LR, int R> __global__ void __launch_bounds__(LR > 256 ? LR : 256) k_block_bwd(const Args p) {
    constexpr bool kPrecise = sizeof(E) == 4;
    constexpr int kThreads = LR > 256 ? LR : 256, kRows = kThreads / LR;
    __shared__ float s_red[kThreads / 64];
    __shared__ float s_join[kRows > 1 ? kThreads * R * V : 1];
    const int j = threadIdx.x % LR;
    float w[R][V], scale[R][V], next[R][V];
    float dw[R][V] = {}, dscale[R][V] = {}, dnext[R][V] = {};
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int d = (r * LR + j) * V;
        load_weight<V>(p.w, d, p.D, 0.0f, w[r]);
        load_weight<V>(p.scale, d, p.D, 1.0f, scale[r]);
        load_weight<V>(p.next, d, p.D, 0.0f, next[r]);
    }
    // The next row's operands are on their way while the current row is worked on (as they lie in memory: 16-bit types take half the registers).
    typename Vec<E, V>::type in[5][R];
    float in_ry = 0.0f, in_rx = 0.0f;
    auto fetch = [&](int64_t row) {
        const bool live = row < p.M;
        if (live) in_ry = p.stats[2 * row], in_rx = p.stats[2 * row + 1];
#pragma unroll
        for (int r = 0; r < R; r++) {
            const int d = (r * LR + j) * V, valid = live ? p.D - d : 0;
            in[0][r] = load_raw<E, V>((const E*)p.x + row * p.x_sn + d, valid);
            if (p.y) in[1][r] = load_raw<E, V>((const E*)p.y + row * p.y_sn + d, valid);
            if (p.g) in[2][r] = load_raw<E, V>((const E*)p.g + row * p.g_sn + d, valid);
            if (p.d_out) in[3][r] = load_raw<E, V>((const E*)p.d_out + row * p.do_sn + d, valid);
            if (p.d_u) in[4][r] = load_raw<E, V>((const E*)p.d_u + row * p.du_sn + d, valid);
        }
    };
    constexpr bool kAhead = LR <= 256 && R == 1;  // (wider rows have no registers left for it)
    if (kAhead) fetch((int64_t)blockIdx.x * kRows + threadIdx.x / LR);
    for (int64_t row0 = (int64_t)blockIdx.x * kRows; row0 < p.M; row0 += (int64_t)gridDim.x * kRows) {
        const int64_t row = row0 + threadIdx.x / LR;
        const bool live = row < p.M;
        if (!kAhead) fetch(row);
        float x[R][V], yn[R][V], g[R][V], dx[R][V], t[R][V];
        const float ry = live ? in_ry : 0.0f, rx = live ? in_rx : 0.0f;
        float sum = 0.0f;
#pragma unroll
        for (int r = 0; r < R; r++) {
            widen<E, V>(in[0][r], x[r]);
            if (p.y) widen<E, V>(in[1][r], yn[r]);
            if (p.g) widen<E, V>(in[2][r], g[r]);
            if (p.d_out) widen<E, V>(in[3][r], dx[r]);
            if (p.d_u) widen<E, V>(in[4][r], t[r]);
        }
        if (kAhead) fetch(row + (int64_t)gridDim.x * kRows);
        // yn = y ry; x becomes xn = new rx; t = d_u (then d_u next)
#pragma unroll
        for (int r = 0; r < R; r++) {
#pragma unroll
            for (int i = 0; i < V; i++) {
                if (!p.d_out) dx[r][i] = 0.0f;
                if (!p.d_u) t[r][i] = 0.0f;
                if (p.y) {
                    yn[r][i] *= ry;
                    float a = scale[r][i];
                    if (p.g) {
                        const float gv = g[r][i];
                        a *= gv * keep_of(gv, sigmoid_pair<kPrecise>(gv));
                    }
                    x[r][i] = __builtin_fmaf(a, yn[r][i] * w[r][i], x[r][i]);
                }
                x[r][i] *= rx;
                dnext[r][i] = __builtin_fmaf(t[r][i], x[r][i], dnext[r][i]);
                t[r][i] *= next[r][i];
                sum = __builtin_fmaf(t[r][i], x[r][i], sum);
            }
        }
        if (p.d_u) {
            const float mean = row_sum<LR>(sum, s_red) * p.inv_d;
#pragma unroll
            for (int r = 0; r < R; r++)
#pragma unroll
                for (int i = 0; i < V; i++) dx[r][i] = __builtin_fmaf(rx, __builtin_fmaf(-mean, x[r][i], t[r][i]), dx[r][i]);
        }
#pragma unroll
        for (int r = 0; r < R; r++) {
            const int d = (r * LR + j) * V, valid = live ? p.D - d : 0;
            store_some<E, V>((E*)p.dx + row * p.D + d, valid, dx[r]);
        }
        if (!p.y) continue;
        sum = 0.0f;
#pragma unroll
        for (int r = 0; r < R; r++) {
            const int d = (r * LR + j) * V, valid = live ? p.D - d : 0;
#pragma unroll
            for (int i = 0; i < V; i++) {
                const float n = yn[r][i] * w[r][i], dp = dx[r][i] * scale[r][i];
                float a = 1.0f;
                if (p.g) {
                    const float gv = g[r][i];
                    const Sigmoid s = sigmoid_pair<kPrecise>(gv);
                    const float sig = keep_of(gv, s);
                    a = gv * sig;
                    g[r][i] = dp * n * __builtin_fmaf(a, take_of(gv, s), sig);
                }
                dscale[r][i] = __builtin_fmaf(dx[r][i], a * n, dscale[r][i]);
                const float dn = dp * a;
                dw[r][i] = __builtin_fmaf(dn, yn[r][i], dw[r][i]);
                t[r][i] = dn * w[r][i];
                sum = __builtin_fmaf(t[r][i], yn[r][i], sum);
            }
            if (p.g) store_some<E, V>((E*)p.dg + row * p.dg_sn + d, valid, g[r]);
        }
        const float mean = row_sum<LR>(sum, s_red) * p.inv_d;
#pragma unroll
        for (int r = 0; r < R; r++) {
            const int d = (r * LR + j) * V, valid = live ? p.D - d : 0;
            float dy[V];
#pragma unroll
            for (int i = 0; i < V; i++) dy[i] = ry * __builtin_fmaf(-mean, yn[r][i], t[r][i]);
            store_some<E, V>((E*)p.dy + row * p.D + d, valid, dy);
        }
    }
    // this workgroup's share of the three sums over rows
    float* out = p.partial + (int64_t)blockIdx.x * 3 * p.D;
#pragma unroll
    for (int q = 0; q < 3; q++) {
        float(&acc)[R][V] = q == 0 ? dw : q == 1 ? dscale : dnext;
        if constexpr (kRows > 1) {
            __syncthreads();
#pragma unroll
            for (int r = 0; r < R; r++)
#pragma unroll
                for (int i = 0; i < V; i++) s_join[((threadIdx.x / LR) * R * V + r * V + i) * LR + j] = acc[r][i];
            __syncthreads();
            if (threadIdx.x < LR) {
#pragma unroll
                for (int r = 0; r < R; r++)
#pragma unroll
                    for (int i = 0; i < V; i++) {
                        float v = 0.0f;
#pragma unroll
                        for (int k = 0; k < kRows; k++) v += s_join[(k * R * V + r * V + i) * LR + j];
                        acc[r][i] = v;
                    }
            }
        }
        if (threadIdx.x < LR) {
#pragma unroll
            for (int r = 0; r < R; r++)
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const int d = (r * LR + j) * V + i;
                    if (d < p.D) out[q * p.D + d] = acc[r][i];
                }
        }
    }
}

// out[c] = sum over k of partial[k][c], in a fixed order: 64 columns a workgroup, four a lane, 64 threads over the workgroups' sums
__global__ void __launch_bounds__(1024) k_block_sum(const float* __restrict__ partial, int n, int columns, float* __restrict__ out) {
    __shared__ float s[64][65];
    const int q = threadIdx.x & 15, part = threadIdx.x >> 4;
    const int c = blockIdx.x * 64 + q * 4, valid = columns - c;
    float a[4] = {};
#pragma unroll 8
    for (int k = part; k < n; k += 64) {
        float v[4];
        load_some<float, 4>(partial + (int64_t)k * columns + c, valid, v);
#pragma unroll
        for (int i = 0; i < 4; i++) a[i] += v[i];
    }
#pragma unroll
    for (int i = 0; i < 4; i++) s[part][q * 4 + i] = a[i];
    __syncthreads();
    const int column = threadIdx.x & 63, w = threadIdx.x >> 6;
    const float v = (s[w * 4][column] + s[w * 4 + 1][column]) + (s[w * 4 + 2][column] + s[w * 4 + 3][column]);
    __syncthreads();
    s[w][column] = v;
    __syncthreads();
    if (w == 0 && blockIdx.x * 64 + column < columns) {
        float t = 0.0f;
#pragma unroll
        for (int k = 0; k < 16; k++) t += s[k][column];
        out[blockIdx.x * 64 + column] = t;
    }
}

constexpr int kMaxWidth = 4096;  // 1024 lanes with a vector of 4 each; with two they would spill

// lanes of a row and vectors of a lane, by width.  16-bit rows of up to 512 take vectors of 8 (16-byte loads); beyond, a lane with two of them would
// hold 256 registers in the backward pass: vectors of 4 and more lanes.
template <class E, class F> static void with_shape(int64_t D, F&& fn) {
    using std::integral_constant;
    auto pick = [&](auto v) {
        constexpr int V = decltype(v)::value;
        const int64_t n = (D + V - 1) / V;
        constexpr integral_constant<int, 1> one{};
        if (n <= 8) fn(v, integral_constant<int, 8>{}, one);
        else if (n <= 16) fn(v, integral_constant<int, 16>{}, one);
        else if (n <= 32) fn(v, integral_constant<int, 32>{}, one);
        else if (n <= 64) fn(v, integral_constant<int, 64>{}, one);
        else if constexpr (V == 4) {
            if (n <= 128) fn(v, integral_constant<int, 128>{}, one);
            else if (n <= 256) fn(v, integral_constant<int, 256>{}, one);
            else if (n <= 512) fn(v, integral_constant<int, 256>{}, integral_constant<int, 2>{});
            else fn(v, integral_constant<int, 1024>{}, one);
        }
    };
    if (sizeof(E) == 2 && D <= 512) pick(integral_constant<int, 8>{});
    else pick(integral_constant<int, 4>{});
}
static int64_t workgroups(int64_t M, int lr) {
    const int rows = lr > 256 ? 1 : 256 / lr;
    const int64_t n = (M + rows - 1) / rows, most = lr > 256 ? 256 : 1024;
    return n < most ? n : most;
}
static int64_t partial_floats(int64_t M, int64_t D, int dtype) {
    int64_t n = 0;
    with_element(dtype, [&](auto* e) {
        using E = std::remove_pointer_t<decltype(e)>;
        with_shape<E>(D, [&](auto, auto lr, auto) { n = workgroups(M, decltype(lr)::value) * 3 * D; });
    });
    return n;
}
static int check_sizes(int64_t M, int64_t D, int dtype, float eps, const char* who) {
    if (dtype != ACX_F32 && dtype != ACX_BF16 && dtype != ACX_F16) return fail(ACX_E_INVAL, "%s: activations are ACX_F32, ACX_BF16 or ACX_F16", who);
    if (M < 0 || D < 0 || M > ((int64_t)1 << 40)) return fail(ACX_E_INVAL, "%s: bad sizes", who);
    if (D > kMaxWidth) return fail(ACX_E_INVAL, "%s: rows of up to %d features (%lld asked for)", who, kMaxWidth, (long long)D);
    if (!(eps >= 0.0f)) return fail(ACX_E_INVAL, "%s: eps is negative or NaN", who);
    return ACX_OK;
}

}  // namespace block
}  // namespace acx

using namespace acx;

extern "C" int64_t acx_block_workspace_bytes(int64_t M, int64_t D, int dtype) {
    if (M <= 0 || D <= 0 || D > block::kMaxWidth) return 0;
    return block::partial_floats(M, D, dtype) * 4;
}
extern "C" int acx_block_forward(const void* d_x, int64_t x_row, const void* d_y, int64_t y_row, const void* d_gate, int64_t g_row, int dtype, const float* d_weight,
                                 const float* d_scale, const float* d_next_weight, float eps, int64_t M, int64_t D, void* d_new, void* d_u, float* d_stats, void* stream) {
    if (!have_device()) return ACX_E_NODEVICE;
    const int rc = block::check_sizes(M, D, dtype, eps, "acx_block_forward");
    if (rc) return rc;
    if (M == 0 || D == 0) return ACX_OK;
    if (!d_x || (d_y ? !d_weight || !d_new : !d_next_weight) || (d_next_weight && !d_u) || (d_gate && !d_y)) return fail(ACX_E_INVAL, "acx_block_forward: null pointer");
    block::Args a = {};
    a.x = d_x, a.x_sn = x_row, a.y = d_y, a.y_sn = y_row, a.g = d_gate, a.g_sn = g_row;
    a.w = d_weight, a.scale = d_scale, a.next = d_next_weight, a.eps = eps, a.inv_d = 1.0f / (float)D, a.M = M, a.D = (int)D;
    a.out = d_new, a.u = d_u, a.stats = d_stats;
    elem::with_element(dtype, [&](auto* e) {
        using E = std::remove_pointer_t<decltype(e)>;
        block::with_shape<E>(D, [&](auto v, auto lr, auto r) {
            constexpr int LR = decltype(lr)::value;
            hipLaunchKernelGGL((block::k_block_fwd<E, decltype(v)::value, LR, decltype(r)::value, false>), dim3((unsigned)block::workgroups(M, LR)), dim3(LR > 256 ? LR : 256), 0,
                               (hipStream_t)stream, a);
        });
    });
    ACX_HIP_TRY(hipGetLastError());
    return ACX_OK;
}
extern "C" int acx_block_step(const void* d_x, int64_t x_row, const void* d_projected, int64_t p_row, int dtype, const uint8_t* d_reset, const float* d_state, const float* d_weight,
                              const float* d_scale, const float* d_next_weight, float eps, int64_t M, int64_t D, float* d_next_state, void* d_new, void* d_u, void* stream) {
    if (!have_device()) return ACX_E_NODEVICE;
    const int rc = block::check_sizes(M, D, dtype, eps, "acx_block_step");
    if (rc) return rc;
    if (M == 0 || D == 0) return ACX_OK;
    if (!d_x || !d_projected || !d_state || !d_weight || !d_next_state || !d_new || (d_next_weight && !d_u)) return fail(ACX_E_INVAL, "acx_block_step: null pointer");
    block::Args a = {};
    a.x = d_x, a.x_sn = x_row, a.proj = d_projected, a.p_sn = p_row, a.reset = d_reset, a.state = d_state, a.next_state = d_next_state;
    a.w = d_weight, a.scale = d_scale, a.next = d_next_weight, a.eps = eps, a.inv_d = 1.0f / (float)D, a.M = M, a.D = (int)D;
    a.out = d_new, a.u = d_u;
    elem::with_element(dtype, [&](auto* e) {
        using E = std::remove_pointer_t<decltype(e)>;
        block::with_shape<E>(D, [&](auto v, auto lr, auto r) {
            constexpr int LR = decltype(lr)::value;
            hipLaunchKernelGGL((block::k_block_fwd<E, decltype(v)::value, LR, decltype(r)::value, true>), dim3((unsigned)block::workgroups(M, LR)), dim3(LR > 256 ? LR : 256), 0,
                               (hipStream_t)stream, a);
        });
    });
    ACX_HIP_TRY(hipGetLastError());
    return ACX_OK;
}
extern "C" int acx_block_backward(const void* d_x, int64_t x_row, const void* d_y, int64_t y_row, const void* d_gate, int64_t g_row, const void* d_new_grad, int64_t dn_row,
                                  const void* d_u_grad, int64_t du_row, int dtype, const float* d_weight, const float* d_scale, const float* d_next_weight, const float* d_stats,
                                  int64_t M, int64_t D, void* d_x_grad, void* d_y_grad, void* d_gate_grad, int64_t dg_row, float* d_weight_grads, void* d_work, int64_t work_bytes,
                                  void* stream) {
    if (!have_device()) return ACX_E_NODEVICE;
    const int rc = block::check_sizes(M, D, dtype, 0.0f, "acx_block_backward");
    if (rc) return rc;
    if (M == 0 || D == 0) return ACX_OK;
    if (!d_x || !d_stats || !d_x_grad || !d_weight_grads || (d_y && (!d_weight || !d_y_grad)) || (d_gate && (!d_y || !d_gate_grad)) || (d_u_grad && !d_next_weight))
        return fail(ACX_E_INVAL, "acx_block_backward: null pointer");
    const int64_t need = block::partial_floats(M, D, dtype) * 4;
    if (!d_work || work_bytes < need) return fail(ACX_E_CAPACITY, "acx_block_backward: a workspace of %lld bytes is needed (acx_block_workspace_bytes)", (long long)need);
    block::Args a = {};
    a.x = d_x, a.x_sn = x_row, a.y = d_y, a.y_sn = y_row, a.g = d_gate, a.g_sn = g_row;
    a.w = d_weight, a.scale = d_scale, a.next = d_next_weight, a.inv_d = 1.0f / (float)D, a.M = M, a.D = (int)D;
    a.stats = const_cast<float*>(d_stats);
    a.d_out = d_new_grad, a.do_sn = dn_row, a.d_u = d_u_grad, a.du_sn = du_row;
    a.dx = d_x_grad, a.dy = d_y_grad, a.dg = d_gate_grad, a.dg_sn = dg_row, a.partial = (float*)d_work;
    int64_t n = 0;
    elem::with_element(dtype, [&](auto* e) {
        using E = std::remove_pointer_t<decltype(e)>;
        block::with_shape<E>(D, [&](auto v, auto lr, auto r) {
            constexpr int LR = decltype(lr)::value;
            n = block::workgroups(M, LR);
            hipLaunchKernelGGL((block::k_block_bwd<E, decltype(v)::value, LR, decltype(r)::value>), dim3((unsigned)n), dim3(LR > 256 ? LR : 256), 0, (hipStream_t)stream, a);
        });
    });
    ACX_HIP_TRY(hipGetLastError());
    hipLaunchKernelGGL(block::k_block_sum, dim3((unsigned)((3 * D + 63) / 64)), dim3(1024), 0, (hipStream_t)stream, (const float*)d_work, (int)n, (int)(3 * D), d_weight_grads);
    ACX_HIP_TRY(hipGetLastError());
    return ACX_OK;
}
