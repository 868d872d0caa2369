// acx_block.hip -- the end of a block of the recurrent agent: the norm behind the block, its gate and residual scale, and the norm in
// front of the next block, in one pass over the rows; the gradient of that; and the whole block for one step of the environments.
//
//   new = x + scale * silu(gate) * rms(y) weight,   u = rms(new) next_weight,   rms(v) = v / sqrt(mean(v^2) + eps)
//
// Forward: 3 rows read, 2 written, two row sums; backward: 5 read, 3 written, two row sums, and three sums over all rows (the gradients
// of weight, scale and next_weight).  About 50 vector instructions per element: bound by HBM.
//   - A row belongs to LR neighbouring lanes that hold all of it in registers, a vector of V elements each (16 bytes a load); narrow rows share a
//     wave, a row over 64 lanes takes a workgroup of as many waves as it needs (row sums through LDS).
//   - The backward pass recomputes `new` from x, y and gate (it reads them anyway) unrounded and takes the two reciprocal roots of a row
//     from the forward pass (8 bytes a row instead of two more row sums).
// Measured: 1 Mi x 256 bf16 forward 0.565 ms (4.75 TB/s of what it moves), backward 0.91 ms (4.7 TB/s), the sums over rows 8 us; 4099 x 2048 f32
// 30 + 50 + 4 us; one step of 131072 x 256 bf16 0.133 ms (5.0 TB/s).  The backward pass without the next row's operands on the way: 1.28 ms; the
// forward pass has the waves to hide its loads and loses by it (0.584 ms).
//   - Sums over rows: every lane adds its features over the rows that its workgroup walks, the workgroup's row groups join through the lanes of a wave and LDS, and a second
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

// V elements of row `row` from feature d on; the vector may end behind the row where the tensor goes on that far
template <class E, int V> __device__ __forceinline__ typename Vec<E, V>::type load_row(const Args& p, const void* base, int64_t sn, int64_t row, int d, int valid) {
    const int64_t at = row * sn + d;
    return load_raw<E, V>((const E*)base + at, valid, at <= (p.M - 1) * sn + (p.D - V));
}

// LR > 64 stands for rows of a workgroup: LR is then the largest workgroup of the variant, and blockDim.x lanes have the row.
template <int LR> constexpr int kThreads = LR > 64 ? LR : 256;
template <int LR> constexpr int kRows = LR > 64 ? 1 : 256 / LR;  // rows that a workgroup holds at a time

// sum over the lanes of a row, in every one of them (s_red: one float per wave of the workgroup)
template <int LR> __device__ __forceinline__ float row_sum(float v, float* s_red) {
    v = lane_sum<(LR < 64 ? LR : 64)>(v);
    if constexpr (LR > 64) {
        __syncthreads();  // (the sums of the last call have been read)
        if ((threadIdx.x & 63) == 0) s_red[threadIdx.x >> 6] = v;
        __syncthreads();
        const int waves = blockDim.x >> 6;
        v = 0.0f;
        for (int i = 0; i < waves; i++) v += s_red[i];
    }
    return v;
}

template <int V> __device__ __forceinline__ void load_weight(const float* p, int d, int D, float fallback, float (&out)[V]) {
#pragma unroll
    for (int i = 0; i < V; i++) out[i] = p && d + i < D ? p[d + i] : fallback;
}

template <class E, int V, int LR, bool STEP> __global__ void __launch_bounds__(kThreads<LR>) k_block_fwd(const Args p) {
    constexpr bool kPrecise = sizeof(E) == 4;
    __shared__ float s_red[kThreads<LR> / 64];
    const int j = LR > 64 ? threadIdx.x : threadIdx.x % LR, d = j * V;
    float w[V], scale[V], next[V];
    load_weight<V>(p.w, d, p.D, 0.0f, w);
    load_weight<V>(p.scale, d, p.D, 1.0f, scale);
    load_weight<V>(p.next, d, p.D, 0.0f, next);
    for (int64_t row0 = (int64_t)blockIdx.x * kRows<LR>; row0 < p.M; row0 += (int64_t)gridDim.x * kRows<LR>) {
        const int64_t row = row0 + (LR > 64 ? 0 : threadIdx.x / LR);
        const bool live = row < p.M;  // (lanes behind the last row run along for the row sums)
        const int valid = live ? p.D - d : 0;
        float x[V], y[V], g[V];
        float sum = 0.0f;
        const auto x_raw = load_row<E, V>(p, p.x, p.x_sn, row, d, valid);
        if constexpr (STEP) {
            const E* proj = (const E*)p.proj + row * p.p_sn + d;
            const auto c_raw = load_raw<E, V>(proj, valid, p.D >= V), z_raw = load_raw<E, V>(proj + p.D, valid, p.D >= V);  // (another third of the row follows)
            const auto g_raw = load_row<E, V>(p, (const E*)p.proj + 2 * (int64_t)p.D, p.p_sn, row, d, valid);
            const auto h_raw = load_row<float, V>(p, p.state, p.D, row, d, valid);
            const bool start = live && p.reset && p.reset[row];
            float c[V], z[V], h[V];
            widen<E, V>(c_raw, valid, c);
            widen<E, V>(z_raw, valid, z);
            widen<E, V>(g_raw, valid, g);
            widen<float, V>(h_raw, valid, h);
#pragma unroll
            for (int i = 0; i < V; i++) {
                const Sigmoid s = sigmoid_pair<kPrecise>(z[i]);
                y[i] = __builtin_fmaf(keep_of(z[i], s), start ? 0.0f : h[i], take_of(z[i], s) * c[i]);
            }
            store_some<float, V>(p.next_state + row * p.D + d, valid, y);
        } else if (p.y) {
            const auto y_raw = load_row<E, V>(p, p.y, p.y_sn, row, d, valid);
            if (p.g) widen<E, V>(load_row<E, V>(p, p.g, p.g_sn, row, d, valid), valid, g);
            widen<E, V>(y_raw, valid, y);
        }
        widen<E, V>(x_raw, valid, x);
        float ry = 0.0f;
        if (STEP || p.y) {
#pragma unroll
            for (int i = 0; i < V; i++) sum = __builtin_fmaf(y[i], y[i], sum);
            ry = rsqrtf(__builtin_fmaf(row_sum<LR>(sum, s_red), p.inv_d, p.eps));
#pragma unroll
            for (int i = 0; i < V; i++) {
                float a = scale[i];
                if (STEP || p.g) a *= g[i] * keep_of(g[i], sigmoid_pair<kPrecise>(g[i]));
                x[i] = __builtin_fmaf(a, y[i] * ry * w[i], x[i]);
            }
            store_some<E, V>((E*)p.out + row * p.D + d, valid, x);
        }
        float rx = 0.0f;
        if (p.next) {
            sum = 0.0f;
#pragma unroll
            for (int i = 0; i < V; i++) sum = __builtin_fmaf(x[i], x[i], sum);
            rx = rsqrtf(__builtin_fmaf(row_sum<LR>(sum, s_red), p.inv_d, p.eps));
            float u[V];
#pragma unroll
            for (int i = 0; i < V; i++) u[i] = x[i] * rx * next[i];
            store_some<E, V>((E*)p.u + row * p.D + d, valid, u);
        }
        if (!STEP && p.stats && live && j == 0) {
            p.stats[2 * row] = ry;
            p.stats[2 * row + 1] = rx;
        }
    }
}

template <class E, int V, int LR> __global__ void __launch_bounds__(kThreads<LR>) k_block_bwd(const Args p) {
    constexpr bool kPrecise = sizeof(E) == 4;
    __shared__ float s_red[kThreads<LR> / 64];
    __shared__ float s_join[kRows<LR> > 1 ? 4 * LR * V : 1];
    const int j = LR > 64 ? threadIdx.x : threadIdx.x % LR, d = j * V;
    float w[V], scale[V], next[V], dw[V] = {}, dscale[V] = {}, dnext[V] = {};
    load_weight<V>(p.w, d, p.D, 0.0f, w);
    load_weight<V>(p.scale, d, p.D, 1.0f, scale);
    load_weight<V>(p.next, d, p.D, 0.0f, next);
    // The next row's operands are on their way while the current row is worked on (as they lie in memory: 16-bit types take half the registers).
    typename Vec<E, V>::type in[5];
    float in_ry = 0.0f, in_rx = 0.0f;
    auto fetch = [&](int64_t row) {
        const int valid = row < p.M ? p.D - d : 0;
        if (row < p.M) in_ry = p.stats[2 * row], in_rx = p.stats[2 * row + 1];
        in[0] = load_row<E, V>(p, p.x, p.x_sn, row, d, valid);
        if (p.y) in[1] = load_row<E, V>(p, p.y, p.y_sn, row, d, valid);
        if (p.g) in[2] = load_row<E, V>(p, p.g, p.g_sn, row, d, valid);
        if (p.d_out) in[3] = load_row<E, V>(p, p.d_out, p.do_sn, row, d, valid);
        if (p.d_u) in[4] = load_row<E, V>(p, p.d_u, p.du_sn, row, d, valid);
    };
    constexpr bool kAhead = LR <= 512;  // (workgroups of 1024 lanes have no registers left for it)
    const int64_t row_of_lane = LR > 64 ? 0 : threadIdx.x / LR;
    if (kAhead) fetch((int64_t)blockIdx.x * kRows<LR> + row_of_lane);
    for (int64_t row0 = (int64_t)blockIdx.x * kRows<LR>; row0 < p.M; row0 += (int64_t)gridDim.x * kRows<LR>) {
        const int64_t row = row0 + row_of_lane;
        const bool live = row < p.M;
        const int valid = live ? p.D - d : 0;
        if (!kAhead) fetch(row);
        float x[V], yn[V], g[V], dx[V] = {}, t[V] = {};
        const float ry = live ? in_ry : 0.0f, rx = live ? in_rx : 0.0f;
        widen<E, V>(in[0], valid, x);
        if (p.y) widen<E, V>(in[1], valid, yn);
        if (p.g) widen<E, V>(in[2], valid, g);
        if (p.d_out) widen<E, V>(in[3], valid, dx);
        if (p.d_u) widen<E, V>(in[4], valid, t);
        if (kAhead) fetch(row + (int64_t)gridDim.x * kRows<LR>);
        // yn = y ry; x becomes xn = new rx; t = d_u (then d_u next)
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < V; i++) {
            if (p.y) {
                yn[i] *= ry;
                float a = scale[i];
                if (p.g) a *= g[i] * keep_of(g[i], sigmoid_pair<kPrecise>(g[i]));
                x[i] = __builtin_fmaf(a, yn[i] * w[i], x[i]);
            }
            x[i] *= rx;
            dnext[i] = __builtin_fmaf(t[i], x[i], dnext[i]);
            t[i] *= next[i];
            sum = __builtin_fmaf(t[i], x[i], sum);
        }
        if (p.d_u) {
            const float mean = row_sum<LR>(sum, s_red) * p.inv_d;
#pragma unroll
            for (int i = 0; i < V; i++) dx[i] = __builtin_fmaf(rx, __builtin_fmaf(-mean, x[i], t[i]), dx[i]);
        }
        store_some<E, V>((E*)p.dx + row * p.D + d, valid, dx);
        if (!p.y) continue;
        sum = 0.0f;
#pragma unroll
        for (int i = 0; i < V; i++) {
            const float n = yn[i] * w[i], dp = dx[i] * scale[i];
            float a = 1.0f;
            if (p.g) {
                const Sigmoid s = sigmoid_pair<kPrecise>(g[i]);
                const float sig = keep_of(g[i], s);
                a = g[i] * sig;
                g[i] = dp * n * __builtin_fmaf(a, take_of(g[i], s), sig);
            }
            dscale[i] = __builtin_fmaf(dx[i], a * n, dscale[i]);
            const float dn = dp * a;
            dw[i] = __builtin_fmaf(dn, yn[i], dw[i]);
            t[i] = dn * w[i];
            sum = __builtin_fmaf(t[i], yn[i], sum);
        }
        if (p.g) store_some<E, V>((E*)p.dg + row * p.dg_sn + d, valid, g);
        const float mean = row_sum<LR>(sum, s_red) * p.inv_d;
        float dy[V];
#pragma unroll
        for (int i = 0; i < V; i++) dy[i] = ry * __builtin_fmaf(-mean, yn[i], t[i]);
        store_some<E, V>((E*)p.dy + row * p.D + d, valid, dy);
    }
    // this workgroup's share of the three sums over rows
    float* out = p.partial + (int64_t)blockIdx.x * 3 * p.D;
#pragma unroll
    for (int q = 0; q < 3; q++) {
        float(&acc)[V] = q == 0 ? dw : q == 1 ? dscale : dnext;
        if constexpr (kRows<LR> > 1) {  // the row groups of a wave among themselves, then the four waves
#pragma unroll
            for (int i = 0; i < V; i++)
#pragma unroll
                for (int m = LR; m < 64; m *= 2) acc[i] += __shfl_xor(acc[i], m);
            __syncthreads();
            if ((threadIdx.x & 63) < LR) {
#pragma unroll
                for (int i = 0; i < V; i++) s_join[((threadIdx.x >> 6) * V + i) * LR + j] = acc[i];
            }
            __syncthreads();
            if (threadIdx.x < LR) {
#pragma unroll
                for (int i = 0; i < V; i++) acc[i] = (s_join[i * LR + j] + s_join[(V + i) * LR + j]) + (s_join[(2 * V + i) * LR + j] + s_join[(3 * V + i) * LR + j]);
            }
        }
        if (LR > 64 || threadIdx.x < LR) {
#pragma unroll
            for (int i = 0; i < V; i++)
                if (d + i < p.D) out[q * p.D + d + i] = acc[i];
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

constexpr int kMaxWidth = 4096;  // a workgroup's lanes with a vector each

// lanes of a row, by its vectors: fn(V, LR, workgroup).  16-byte loads.  (16-bit rows of more than 2048 with 8-byte ones in up to 1024
// lanes, which have no registers left for the next row: 56005 x 3302 bf16 632 + 1354 us forward and backward, 396 + 860 like this; float32
// ones keep to 1024 lanes, 16001 x 2050 takes 183 + 357 us with 32 bytes a lane and 136 + 297 with 16.)  Rows of one or two vectors take
// two lanes: 487495 x 2 f16 12 + 40 us, 41 + 108 with eight.
template <class E, class F> static void with_shape(int64_t D, F&& fn) {
    using std::integral_constant;
    auto narrow = [&](auto v) {
        const int n = (int)((D + decltype(v)::value - 1) / decltype(v)::value);
        if (n <= 2) fn(v, integral_constant<int, 2>{}, 256);
        else if (n <= 8) fn(v, integral_constant<int, 8>{}, 256);
        else if (n <= 16) fn(v, integral_constant<int, 16>{}, 256);
        else if (n <= 32) fn(v, integral_constant<int, 32>{}, 256);
        else if (n <= 64) fn(v, integral_constant<int, 64>{}, 256);
        else fn(v, integral_constant<int, 256>{}, (n + 63) / 64 * 64);
    };
    if constexpr (sizeof(E) == 2) {
        if (D <= 2048) narrow(integral_constant<int, 8>{});
        else fn(integral_constant<int, 8>{}, integral_constant<int, 512>{}, (int)(D + 511) / 512 * 64);
    } else {
        if (D <= 1024) narrow(integral_constant<int, 4>{});
        else if (D <= 2048) fn(integral_constant<int, 4>{}, integral_constant<int, 512>{}, (int)(D + 255) / 256 * 64);
        else fn(integral_constant<int, 4>{}, integral_constant<int, 1024>{}, (int)(D + 255) / 256 * 64);
    }
}
// Workgroups of 1024 lanes a compute unit: as many as stay resident where the backward pass has up to 128 registers (float32 rows, but for those of a whole
// wave), two rounds of them for 16-bit rows, whose backward pass has 168 to 206; what is gained by more is less than their partial sums cost.
// The same number for each of the 256 compute units: 819 of 320 lanes on 49016 x 1104 f32, the backward pass takes 592 us and 484 with 768,
// because 51 of them start when the others end.
static int64_t workgroups(int64_t M, int lr, int threads, int lanes = 1024) {
    const int rows = lr > 64 ? 1 : 256 / lr;
    const int64_t n = (M + rows - 1) / rows, most = lanes / threads * 256;
    return n < most ? n : most;
}
// (the forward pass has no partial sums and fewer registers: with 1024 lanes a compute unit workgroups of 576 to 960 would be alone on one; 16001 x 2050
// f32 136 us, 162 with one each; 56005 x 3302 bf16, 448 lanes, 396 us with two each, 458 with four)
static int forward_lanes(int threads) { return threads > 512 ? 1920 : 1024; }
static int64_t partial_floats(int64_t M, int64_t D, int dtype) {
    int64_t n = 0;
    with_element(dtype, [&](auto* e) {
        using E = std::remove_pointer_t<decltype(e)>;
        with_shape<E>(D, [&](auto, auto lr, int threads) { n = workgroups(M, decltype(lr)::value, threads) * 3 * D; });
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
    if (block::check_sizes(M, D, dtype, 0.0f, "acx_block_workspace_bytes") || M == 0 || D == 0) return 0;
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
        block::with_shape<E>(D, [&](auto v, auto lr, int threads) {
            constexpr int LR = decltype(lr)::value;
            hipLaunchKernelGGL((block::k_block_fwd<E, decltype(v)::value, LR, false>), dim3((unsigned)block::workgroups(M, LR, threads, block::forward_lanes(threads))), dim3(threads), 0, (hipStream_t)stream, a);
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
        block::with_shape<E>(D, [&](auto v, auto lr, int threads) {
            constexpr int LR = decltype(lr)::value;
            hipLaunchKernelGGL((block::k_block_fwd<E, decltype(v)::value, LR, true>), dim3((unsigned)block::workgroups(M, LR, threads, block::forward_lanes(threads))), dim3(threads), 0, (hipStream_t)stream, a);
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
        block::with_shape<E>(D, [&](auto v, auto lr, int threads) {
            constexpr int LR = decltype(lr)::value;
            n = block::workgroups(M, LR, threads);
            hipLaunchKernelGGL((block::k_block_bwd<E, decltype(v)::value, LR>), dim3((unsigned)n), dim3(threads), 0, (hipStream_t)stream, a);
        });
    });
    ACX_HIP_TRY(hipGetLastError());
    hipLaunchKernelGGL(block::k_block_sum, dim3((unsigned)((3 * D + 63) / 64)), dim3(1024), 0, (hipStream_t)stream, (const float*)d_work, (int)n, (int)(3 * D), d_weight_grads);
    ACX_HIP_TRY(hipGetLastError());
    return ACX_OK;
}
