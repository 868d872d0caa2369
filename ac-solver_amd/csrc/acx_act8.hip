// acx_act8.hip -- activations kept in 8 bits for the backward pass, and the weight gradient that reads them.
//
//   checkpoint of x [M, K]:  blocks of 32 features of a row share a power of two 2^e, the smallest for which the block's largest magnitude
//   rounds to at most 127 (never below 2^-126);  q = rint(x 2^-e) as int8, ties to even;  e + 127 as one byte.  1.03 bytes a value.
//   weight gradient:  dW [O, I] = sum over m of dy[m, o] (q[m, i] 2^e[m, i / 32]),   db[o] = sum over m of dy[m, o]
//
// A power of two as the scale makes q 2^e EXACT in bfloat16 (7 bits of magnitude, bfloat16's own exponent range): the product runs on the bf16
// matrix instructions without rounding the checkpoint again.  dy is brought there without rounding either: a float32 is the sum of three
// bfloat16 (8 + 8 + 8 bits, each the truncated rest of the last), a float16 of two, a bfloat16 of one; the accumulators are float32.  So dW has
// the accuracy of a float32 product, at one to three times the matrix work of a bf16 one and 1 byte instead of 4 read per x.
// A block with an infinity or a NaN is marked with the exponent byte 255 and restores to NaN: it is not hidden.  Finite values restore to finite ones: where rounding up left
// the type, to its largest.
// Measured: 1 Mi x 256 f32 packed in 0.275 ms and restored in 0.275 ms (4.9 TB/s).  Weight gradient of 1 Mi rows, 768 x 256: dy bf16 0.52 to 0.54 ms (4.6 TB/s of
// what it moves: three tiles of outputs read q), f16 0.83 to 0.86, f32 1.19 to 1.27 by the card: 1.24 TFLOP of bf16 products at 1.04 to 0.98 PFLOP/s, where the chip's clock drops to
// 1.5 GHz under the matrix units' load (a library's bf16 product of 8192^3: 1.16 PFLOP/s).  65537 x 256 x 72 bf16 20 + 5 us: five steps a workgroup,
// their latency and the join.  Between the tiles the padding is staged and multiplied, too: 65 x 129 f32 0.36 ms, 0.09 by its bytes.
#include <type_traits>

#include "acx_elem.h"

namespace acx {
namespace act8 {
using namespace elem;

constexpr int kBlock = 32;

__device__ __forceinline__ float exponent_factor(uint32_t e) { return __builtin_bit_cast(float, e == 255 ? 0x7FC00000u : e << 23); }

template <int N> struct Bytes;
template <> struct Bytes<2> {
    typedef uint16_t type __attribute__((aligned(1)));
};
template <> struct Bytes<4> {
    typedef uint32_t type __attribute__((aligned(1)));
};
template <> struct Bytes<8> {
    typedef uint64_t type __attribute__((aligned(1)));
};

// V features a lane, 32 / V lanes a block
template <class E, int V, bool STREAM> __global__ void __launch_bounds__(256) k_pack8(const E* __restrict__ x, int64_t x_sn, int64_t M, int K, int lpr, int8_t* __restrict__ q, uint8_t* __restrict__ exps) {
    const int64_t l = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t row = l / lpr;
    const int j = (int)(l - row * lpr), d = j * V, valid = row < M ? K - d : 0;
    float v[V];
    load_some<E, V, STREAM>(x + row * x_sn + d, valid, v, row * x_sn + d <= (M - 1) * x_sn + (K - V));
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < V; i++) {
        const uint32_t b = __builtin_bit_cast(uint32_t, v[i]) & 0x7FFFFFFFu;
        top = b > top ? b : top;  // (as bits: an infinity is above every number, a NaN above that)
    }
#pragma unroll
    for (int m = 1; m < kBlock / V; m *= 2) {
        const uint32_t o = __shfl_xor((int)top, m);
        top = o > top ? o : top;
    }
    // the exponent field, one more where the mantissa is 1.9921875 or above (it would round to 128), minus 6
    const int field = (int)((top + 0x10000u) >> 23) - 6;
    const uint32_t e = top >= 0x7F800000u ? 255u : field < 1 ? 1u : (uint32_t)field;
    const float inv = e == 255 ? 0.0f : __builtin_bit_cast(float, (254u - e) << 23);
    uint64_t bytes = 0;
#pragma unroll
    for (int i = 0; i < V; i++) {
        const int n = e == 255 ? 0 : (int)__builtin_rintf(v[i] * inv);
        bytes |= (uint64_t)(uint8_t)n << (8 * i);
    }
    int8_t* out = q + row * K + d;
    if (valid >= V) {
        *(typename Bytes<V>::type*)out = (typename Bytes<V>::type)bytes;
    } else {
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i < valid) out[i] = (int8_t)(bytes >> (8 * i));
    }
    if (valid > 0 && j % (kBlock / V) == 0) exps[row * ((K + kBlock - 1) / kBlock) + d / kBlock] = (uint8_t)e;
}

template <class E, int V, bool STREAM> __global__ void __launch_bounds__(256) k_unpack8(const int8_t* __restrict__ q, const uint8_t* __restrict__ exps, int64_t M, int K, int lpr, E* __restrict__ out) {
    const int64_t l = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t row = l / lpr;
    if (row >= M) return;
    const int j = (int)(l - row * lpr), d = j * V, valid = K - d;
    const uint32_t e = exps[row * ((K + kBlock - 1) / kBlock) + d / kBlock];
    const float factor = exponent_factor(e);
    // Rounding up to the next exponent can carry a finite value past the largest one of its type (65504 in float16: 64 2^10): it restores to that
    // largest one, and so does what `E` has no room for.  (Up to the exponent looked at 127 2^e fits; the comparison is false for the NaN of a marked block.)
    constexpr bool kHalf = std::is_same<E, f16_t>::value;
    constexpr float kLargest = sizeof(E) == 4 ? 0x1.fffffep127f : kHalf ? 65504.0f : 0x1.fep127f;
    auto saturate = [&](float (&v)[V]) {
        if (e > (kHalf ? 136u : 248u)) {
#pragma unroll
            for (int i = 0; i < V; i++) v[i] = __builtin_fabsf(v[i]) > kLargest ? __builtin_copysignf(kLargest, v[i]) : v[i];
        }
    };
    const int8_t* p = q + row * K + d;
    float v[V];
    if (valid >= V) {
        const uint64_t bytes = *(const typename Bytes<V>::type*)p;
#pragma unroll
        for (int i = 0; i < V; i++) v[i] = (float)(int8_t)(bytes >> (8 * i)) * factor;
        saturate(v);
        store<E, V, STREAM>(out + row * K + d, v);
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) v[i] = i < valid ? (float)p[i] * factor : 0.0f;
        saturate(v);
        store_some<E, V, STREAM>(out + row * K + d, valid, v);
    }
}

// ---- weight gradient ----------------------------------------------------------------------------------------------------------------
// A workgroup owns a TO x TI tile of dW and a share of the rows, ROWS at a time: dy and q of these rows go from memory through registers into
// LDS as the 16-byte operands of v_mfma_f32_32x32x16_bf16, 8 rows of one column each.  Columns are stored in the order in which the threads
// bring them (column c of a vector of V stands at (c % V) TO / V + c / V): a wave's stores and its operand loads are both contiguous, and
// the order is undone when dW is written (a lane's products then are neighbours in a row of dW: whole vectors are stored).
// LDS holds two sets of rows and registers a third that is on its way from memory: a step multiplies one set and writes the next.  The two
// waves of a SIMD take these halves in opposite order, so one's conversions (vector pipe) run under the other's products (matrix pipe).  (Workgroups of
// 8 waves; the tile of 64 outputs has 4, one a SIMD, and does the halves one after the other.)
typedef __bf16 frag __attribute__((ext_vector_type(8)));
typedef float acc16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct Args {
    const void* dy;
    int64_t dy_sn;
    const int8_t* q;
    const uint8_t* exps;
    int64_t M, share, whole;  // rows; rows of a workgroup's share, rows that are read in whole vectors (multiples of the rows of a step)
    int O, I, nb;
    float *dw, *db;    // [shares, O, I], [shares, O] (db nullable)
};

__device__ __forceinline__ uint32_t bits_of(float v) { return __builtin_bit_cast(uint32_t, v); }
// the high halves of two floats, side by side
__device__ __forceinline__ uint32_t high_halves(float lo, float hi) { return __builtin_amdgcn_perm(bits_of(hi), bits_of(lo), 0x07060302u); }
__device__ __forceinline__ float truncated(float v) { return __builtin_bit_cast(float, bits_of(v) & 0xFFFF0000u); }

// bfloat16 pieces of a value, and the rows of a step (as many as two sets of 256 + 256 columns leave room for in LDS)
template <class E> struct Pieces { static constexpr int n = 3, rows = 32; };
template <> struct Pieces<bf16_t> { static constexpr int n = 1, rows = 64; };
template <> struct Pieces<f16_t> { static constexpr int n = 2, rows = 32; };

template <class E, int TO, int TI, int NT> struct Tile {
    static constexpr int kP = Pieces<E>::n, kRows = Pieces<E>::rows, kChunks = kRows / 8;
    static constexpr int VO = kRows / 16, VI = TI == 64 ? 2 : 4;  // values of a load of dy and of q
    // waves over the tile, 32 x 32 products of a wave: as many across as a load of q has values, so that a lane ends up with neighbouring columns
    static constexpr int kWaves = NT / 64, kFI = VI, kWI = TI / 32 / kFI, kWO = kWaves / kWI, kFO = TO / kWO / 32;
    static_assert(kFO >= 1 && kFO * kWO * 32 == TO && kFI * kWI * 32 == TI && kWO * kWI == kWaves, "tile");
    static constexpr int kItemsA = kChunks * (TO / VO), kItemsB = kChunks * (TI / VI);
    static constexpr int kPerA = (kItemsA + NT - 1) / NT, kPerB = (kItemsB + NT - 1) / NT;
    static constexpr int kSet = (kP * TO + TI) * kChunks;  // 16-byte operands of a set
    static constexpr size_t kLds = (size_t)2 * kSet * 16;
};

// PART kTail: the last few rows of all, value by value with every bound checked, as a share of their own; else a share of the rows that are read in
// whole vectors, kStageFirst and kMultiplyFirst for the two halves of the workgroup's waves (apart from each other as functions: together
// they need more registers than there are).
enum { kTail, kStageFirst, kMultiplyFirst };
template <class E, int TO, int TI, int NT, int PART> __device__ __forceinline__ void weight_grad8(const Args& p) {
    using T = Tile<E, TO, TI, NT>;
    constexpr bool TAIL = PART == kTail;
    constexpr int kP = T::kP, kRows = T::kRows, kChunks = T::kChunks, VO = T::VO, VI = T::VI, kFO = T::kFO, kFI = T::kFI;
    extern __shared__ u32x4 s_mem[];  // two sets of [piece][chunk][TO], [chunk][TI]
    int tid = threadIdx.x;
    asm volatile("; part %1" : "+v"(tid) : "n"(PART));  // (the parts have nothing in common from here on that would be worked out, and held, in front of the branch between them)
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int o0 = blockIdx.x * TO, i0 = blockIdx.y * TI;
    const int64_t begin = TAIL ? p.whole : (int64_t)blockIdx.z * p.share, end = TAIL ? p.M : begin + p.share < p.whole ? begin + p.share : p.whole;
    // two steps on their way from memory
    struct Rows {
        typename Vec<E, VO>::type a[T::kPerA][8];
        uint32_t b[T::kPerB][8], e[T::kPerB];
    } in[2];
    float bias[T::kPerA][VO] = {};
    // The rows of a step start at a pointer that the whole workgroup shares; a lane's place among them takes 32 bits (the host checks that).  Whole
    // vectors are read whatever O and I are: behind the last column stand values of the next row, which end up in columns of the tile that are not
    // written; p.whole leaves rows enough behind it for that.
    uint32_t off_a[T::kPerA], off_b[T::kPerB], off_e[T::kPerB];
#pragma unroll
    for (int k = 0; k < T::kPerA; k++) {
        const int item = tid + k * NT, chunk = item / (TO / VO), o = o0 + item % (TO / VO) * VO;
        off_a[k] = item < T::kItemsA && o < p.O ? ((uint32_t)(chunk * 8) * (uint32_t)p.dy_sn + (uint32_t)o) * (uint32_t)sizeof(E) : 0;
    }
#pragma unroll
    for (int k = 0; k < T::kPerB; k++) {
        const int item = tid + k * NT, chunk = item / (TI / VI), i = i0 + item % (TI / VI) * VI;
        const bool on = item < T::kItemsB;
        off_b[k] = on && i < p.I ? (uint32_t)(chunk * 8) * (uint32_t)p.I + (uint32_t)i : 0;
        // (eight neighbouring lanes read the same block of features: they bring the exponents of one row each, those behind the last feature too)
        off_e[k] = on && i / kBlock < p.nb ? (uint32_t)(chunk * 8 + (tid & 7)) * (uint32_t)p.nb + (uint32_t)(i / kBlock) : 0;
    }
    auto fetch = [&](Rows& to, int64_t m0) {
        const char* dy = (const char*)p.dy + m0 * p.dy_sn * (int64_t)sizeof(E);
        const int8_t* q = p.q + m0 * p.I;
#pragma unroll
        for (int k = 0; k < T::kPerB; k++) to.e[k] = p.exps[m0 * p.nb + off_e[k]];
#pragma unroll
        for (int r = 0; r < 8; r++) {
#pragma unroll
            for (int k = 0; k < T::kPerA; k++) to.a[k][r] = *(const typename Vec<E, VO>::type*)(dy + off_a[k]);
#pragma unroll
            for (int k = 0; k < T::kPerB; k++) to.b[k][r] = *(const typename Bytes<VI>::type*)(q + off_b[k]);
            dy += p.dy_sn * (int64_t)sizeof(E), q += p.I;
        }
    };
    // eight rows of an item's columns -> the 16-byte operands of every column (and the column sums)
    auto write_a = [&](u32x4* sA, int chunk, int g, int v, float (&x)[8], float& sum, bool count) {
        const float s8 = ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
        sum += count ? s8 : 0.0f;
        // what a piece leaves out of an infinity would be NaN: 0 then.  The sum tells whether there is one (or finite values that add up to one).
        const bool wild = kP > 1 && __any(!(__builtin_fabsf(s8) < __builtin_inff()));
#pragma unroll
        for (int piece = 0; piece < kP; piece++) {
            u32x4 w;
#pragma unroll
            for (int r = 0; r < 4; r++) w[r] = high_halves(x[2 * r], x[2 * r + 1]);
            sA[(piece * kChunks + chunk) * TO + v * (TO / VO) + g] = w;
            if (piece + 1 < kP) {
                if (!wild) {
#pragma unroll
                    for (int r = 0; r < 8; r++) x[r] -= truncated(x[r]);
                } else {
#pragma unroll
                    for (int r = 0; r < 8; r++) {
                        const float t = truncated(x[r]);
                        x[r] = t == x[r] ? 0.0f : x[r] - t;
                    }
                }
            }
        }
    };
    // `edge`: some exponent is 249 or above, where 64 2^122, the largest finite activation rounded up, comes out as an infinity: written a second time, with
    // bfloat16's largest number in its place
    auto write_b = [&](u32x4* sB, int chunk, int g, const uint32_t (&q)[8], const uint32_t (&e)[8], bool edge) {
        float f[8];
#pragma unroll
        for (int r = 0; r < 8; r++) f[r] = exponent_factor(e[r]);
        auto column = [&](int v) {
            u32x4 w;
#pragma unroll
            for (int r = 0; r < 4; r++) w[r] = high_halves((float)(int8_t)(q[2 * r] >> (8 * v)) * f[2 * r], (float)(int8_t)(q[2 * r + 1] >> (8 * v)) * f[2 * r + 1]);
            return w;
        };
#pragma unroll
        for (int v = 0; v < VI; v++) {
            sB[chunk * TI + v * (TI / VI) + g] = column(v);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (edge) {
#pragma unroll 1
            for (int v = 0; v < VI; v++) {
                u32x4 w = column(v);
#pragma unroll
                for (int r = 0; r < 4; r++) w[r] -= ((w[r] & 0x7FFFu) == 0x7F80u ? 1u : 0u) + ((w[r] & 0x7FFF0000u) == 0x7F800000u ? 0x10000u : 0u);
                sB[chunk * TI + v * (TI / VI) + g] = w;
            }
        }
    };
    auto at_edge = [](uint32_t e) { return e - 249u < 6u; };
    auto stage = [&](u32x4* set, const Rows& from, bool count) {
#pragma unroll
        for (int k = 0; k < T::kPerA; k++) {
            const int item = tid + k * NT;
            if (item < T::kItemsA) {
#pragma unroll
                for (int v = 0; v < VO; v++) {
                    float x[8];
#pragma unroll
                    for (int r = 0; r < 8; r++) x[r] = (float)from.a[k][r][v];
                    write_a(set, item / (TO / VO), item % (TO / VO), v, x, bias[k][v], count);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < T::kPerB; k++) {
            const int item = tid + k * NT;
            if (item < T::kItemsB) {
                uint32_t e[8];
                // (ds_swizzle, bit mask mode: the lane of the same eight whose low bits are r)
                e[0] = __builtin_amdgcn_ds_swizzle(from.e[k], 0x0018 | 0 << 5);
                e[1] = __builtin_amdgcn_ds_swizzle(from.e[k], 0x0018 | 1 << 5);
                e[2] = __builtin_amdgcn_ds_swizzle(from.e[k], 0x0018 | 2 << 5);
                e[3] = __builtin_amdgcn_ds_swizzle(from.e[k], 0x0018 | 3 << 5);
                e[4] = __builtin_amdgcn_ds_swizzle(from.e[k], 0x0018 | 4 << 5);
                e[5] = __builtin_amdgcn_ds_swizzle(from.e[k], 0x0018 | 5 << 5);
                e[6] = __builtin_amdgcn_ds_swizzle(from.e[k], 0x0018 | 6 << 5);
                e[7] = __builtin_amdgcn_ds_swizzle(from.e[k], 0x0018 | 7 << 5);
                write_b(set + kP * kChunks * TO, item / (TI / VI), item % (TI / VI), from.b[k], e, __any(at_edge(from.e[k])));
            }
        }
    };
    auto stage_tail = [&](u32x4* set, int64_t m0) {
#pragma unroll
        for (int k = 0; k < T::kPerA; k++) {
            const int item = tid + k * NT, chunk = item / (TO / VO), g = item % (TO / VO);
            if (item < T::kItemsA) {
#pragma unroll
                for (int v = 0; v < VO; v++) {
                    float x[8];
#pragma unroll
                    for (int r = 0; r < 8; r++) {
                        const int64_t m = m0 + chunk * 8 + r;
                        x[r] = m < p.M && o0 + g * VO + v < p.O ? (float)((const E*)p.dy)[m * p.dy_sn + o0 + g * VO + v] : 0.0f;
                    }
                    write_a(set, chunk, g, v, x, bias[k][v], true);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < T::kPerB; k++) {
            const int item = tid + k * NT, chunk = item / (TI / VI), g = item % (TI / VI);
            if (item < T::kItemsB) {
                uint32_t q[8], e[8];
                bool edge = false;
#pragma unroll
                for (int r = 0; r < 8; r++) {
                    const int64_t m = m0 + chunk * 8 + r;
                    q[r] = 0, e[r] = 0;
                    if (m < p.M && i0 + g * VI < p.I) {
                        e[r] = p.exps[m * p.nb + (i0 + g * VI) / kBlock];
#pragma unroll
                        for (int v = 0; v < VI; v++)
                            if (i0 + g * VI + v < p.I) q[r] |= (uint32_t)(uint8_t)p.q[m * p.I + i0 + g * VI + v] << (8 * v);
                    }
                }
#pragma unroll
                for (int r = 0; r < 8; r++) edge |= at_edge(e[r]);  // (behind all the loads, which wait for each other otherwise)
                write_b(set + kP * kChunks * TO, chunk, g, q, e, __any(edge));
            }
        }
    };
    const int wo = wave % T::kWO, wi = wave / T::kWO;
    acc16 acc[kFO][kFI];
#pragma unroll
    for (int x = 0; x < kFO; x++)
#pragma unroll
        for (int y = 0; y < kFI; y++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[x][y][r] = 0.0f;
    auto multiply = [&](const u32x4* set) {
        const u32x4 *sA = set, *sB = set + kP * kChunks * TO;
#pragma unroll
        for (int ks = 0; ks < kRows / 16; ks++) {
            const int chunk = 2 * ks + (lane >> 5), col = lane & 31;
            frag fb[kFI];
#pragma unroll
            for (int y = 0; y < kFI; y++) fb[y] = __builtin_bit_cast(frag, sB[chunk * TI + y * (TI / VI) + wi * 32 + col]);
#pragma unroll
            for (int piece = kP - 1; piece >= 0; piece--) {
#pragma unroll
                for (int x = 0; x < kFO; x++) {
                    const frag fa = __builtin_bit_cast(frag, sA[(piece * kChunks + chunk) * TO + (wo * kFO + x) * 32 + col]);
#pragma unroll
                    for (int y = 0; y < kFI; y++) acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa, fb[y], acc[x][y], 0, 0, 0);
                }
            }
            __builtin_amdgcn_sched_barrier(0);  // (operands of one k-step at a time: there are no registers for more)
        }
    };
    if constexpr (TAIL) {
#pragma unroll 1
        for (int64_t m0 = begin; m0 < end; m0 += kRows) {
            stage_tail(s_mem, m0);
            __syncthreads();
            multiply(s_mem);
            __syncthreads();
        }
    } else {
        // Everything on the way is unconditional (behind the last step the last one again, not counted and not multiplied): the waits before a use
        // then count the loads issued since, and the other set of registers stays in flight.
        auto at_most = [&](int64_t m) { return m < end ? m : end - kRows; };
        auto renew = [&](Rows& rows, u32x4* to, int64_t m0) {  // step m0 from its registers into LDS, the registers to the step two further on
            stage(to, rows, m0 < end);
            __builtin_amdgcn_sched_barrier(0);
            fetch(rows, at_most(m0 + 2 * kRows));
            __builtin_amdgcn_sched_barrier(0);
        };
        auto product = [&](const u32x4* from, int64_t m0) {
            if (m0 < end) multiply(from);
            __builtin_amdgcn_sched_barrier(0);
        };
        u32x4 *const s0 = s_mem, *const s1 = s_mem + T::kSet;
        fetch(in[0], begin);
        fetch(in[1], at_most(begin + kRows));
        renew(in[0], s0, begin);
        __syncthreads();
        if constexpr (PART == kStageFirst) {
#pragma unroll 1
            for (int64_t m0 = begin; m0 < end; m0 += 2 * kRows) {
                renew(in[1], s1, m0 + kRows);
                product(s0, m0);
                __syncthreads();  // (the set that was multiplied may be written again, the other one is complete)
                renew(in[0], s0, m0 + 2 * kRows);
                product(s1, m0 + kRows);
                __syncthreads();
            }
        } else {
#pragma unroll 1
            for (int64_t m0 = begin; m0 < end; m0 += 2 * kRows) {
                product(s0, m0);
                renew(in[1], s1, m0 + kRows);
                __syncthreads();
                product(s1, m0 + kRows);
                renew(in[0], s0, m0 + 2 * kRows);
                __syncthreads();
            }
        }
    }
    float* dw = p.dw + (int64_t)blockIdx.z * p.O * p.I;
    const int i = i0 + (wi * 32 + (lane & 31)) * VI;
#pragma unroll
    for (int x = 0; x < kFO; x++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
            const int uo = (wo * kFO + x) * 32 + (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5), o = o0 + uo % (TO / VO) * VO + uo / (TO / VO);
            float v[VI];
#pragma unroll
            for (int y = 0; y < VI; y++) v[y] = acc[x][y][r];
            if (o < p.O) store_some<float, VI>(dw + (int64_t)o * p.I + i, p.I - i, v);
        }
    if (p.db && blockIdx.y == 0) {
        float* s = (float*)s_mem;  // [chunk][TO]
#pragma unroll
        for (int k = 0; k < T::kPerA; k++) {
            const int item = tid + k * NT, chunk = item / (TO / VO), g = item % (TO / VO);
            if (item < T::kItemsA) {
#pragma unroll
                for (int v = 0; v < VO; v++) s[chunk * TO + g * VO + v] = bias[k][v];
            }
        }
        __syncthreads();
        for (int o = tid; o < TO && o0 + o < p.O; o += NT) {
            float v = 0.0f;
#pragma unroll
            for (int c = 0; c < kChunks; c++) v += s[c * TO + o];
            p.db[(int64_t)blockIdx.z * p.O + o0 + o] = v;
        }
    }
}

template <class E, int TO, int TI, int NT> __global__ void __launch_bounds__(NT) k_weight_grad8(const Args p) {
    if (blockIdx.z + 1 == gridDim.z) weight_grad8<E, TO, TI, NT, kTail>(p);
    else if (__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) < NT / 128) weight_grad8<E, TO, TI, NT, kStageFirst>(p);
    else weight_grad8<E, TO, TI, NT, kMultiplyFirst>(p);
}

// out[c] = sum over the shares, in a fixed order; dW and db in one launch.  64 columns a workgroup, four a lane, 16 threads over the shares.
__global__ void __launch_bounds__(256) k_join_shares(const float* __restrict__ dw, const float* __restrict__ db, int n, int64_t size, int O, int64_t dw_groups, float* __restrict__ out,
                                                     float* __restrict__ out_db) {
    __shared__ float s[16][65];
    const bool bias = blockIdx.x >= dw_groups;
    const float* src = bias ? db : dw;
    const int64_t columns = bias ? O : size, c0 = (blockIdx.x - (bias ? dw_groups : 0)) * 64;
    const int q = threadIdx.x & 15, part = threadIdx.x >> 4;
    const int valid = columns - c0 - q * 4 > 4 ? 4 : (int)(columns - c0 - q * 4);
    float a[4] = {};
#pragma unroll 8
    for (int k = part; k < n; k += 16) {
        float v[4];
        load_some<float, 4>(src + k * columns + c0 + q * 4, valid, v);
#pragma unroll
        for (int i = 0; i < 4; i++) a[i] += v[i];
    }
#pragma unroll
    for (int i = 0; i < 4; i++) s[part][q * 4 + i] = a[i];
    __syncthreads();
    if (threadIdx.x < 64 && c0 + threadIdx.x < columns) {
        float v = 0.0f;
#pragma unroll
        for (int k = 0; k < 16; k++) v += s[k][threadIdx.x];
        (bias ? out_db : out)[c0 + threadIdx.x] = v;
    }
}

struct Plan {
    int to, ti;
    int64_t go, gi, whole, share, shares;
};
static Plan plan_of(int64_t M, int64_t O, int64_t I) {
    constexpr int kStep = 64;  // rows of a step of every type divide it
    Plan p;
    p.to = O <= 64 ? 64 : 256;
    p.ti = p.to == 64 || I > 128 ? 256 : I <= 64 ? 64 : 128;
    p.go = (O + p.to - 1) / p.to;
    p.gi = (I + p.ti - 1) / p.ti;
    p.whole = M >= 4 ? (M - 4) / kStep * kStep : 0;  // behind these rows at least four more: a vector of up to four values that starts in them ends in bounds
    // A share costs its step's time, ~1.3 us where the chip is not full, and 8 O I bytes of partial sums written and read again at ~4.7 TB/s: n shares of
    // `steps` cost steps / n * 1.3 us + n * 8 O I / 4.7e12 s, least at n^2 = steps * 764000 / (O I).  (65540 x 256 x 256 bf16: 64 us with 256 shares,
    // 33 with the 109 of this rule.)  No more than the chip takes at once.
    const int64_t steps = p.whole / kStep, most = 256 / (p.go * p.gi) - 1;
    int64_t want = (int64_t)__builtin_sqrt((double)steps * 764000.0 / ((double)O * (double)I));
    if (want > most) want = most;
    if (want < 1) want = 1;
    const int64_t per = (steps + want - 1) / want;
    p.share = (per < 4 ? 4 : per) * kStep;
    p.shares = (p.whole + p.share - 1) / p.share + 1;  // and the rows behind them
    return p;
}
static int64_t work_floats(const Plan& p, int64_t O, int64_t I) { return p.shares > 1 ? p.shares * O * (I + 1) : 0; }

template <class E, int TO, int TI, int NT> static hipError_t launch(const Args& a, const Plan& p, hipStream_t st) {
    constexpr size_t lds = Tile<E, TO, TI, NT>::kLds;
    const hipError_t e = hipFuncSetAttribute((const void*)k_weight_grad8<E, TO, TI, NT>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((k_weight_grad8<E, TO, TI, NT>), dim3((unsigned)p.go, (unsigned)p.gi, (unsigned)p.shares), dim3(NT), lds, st, a);
    return hipGetLastError();
}

static int check_rows(int64_t M, int64_t K, int dtype, const char* who) {
    if (dtype != ACX_F32 && dtype != ACX_BF16 && dtype != ACX_F16) return fail(ACX_E_INVAL, "%s: activations are ACX_F32, ACX_BF16 or ACX_F16", who);
    if (M < 0 || K < 0 || K > (1 << 20) || M > ((int64_t)1 << 38)) return fail(ACX_E_INVAL, "%s: bad sizes (rows of up to 2^20 values)", who);
    return ACX_OK;
}
static int check_weights(int64_t M, int64_t O, int64_t I, const char* who) {
    if (M < 1 || O < 1 || I < 1 || M > ((int64_t)1 << 38)) return fail(ACX_E_INVAL, "%s: no rows, outputs or inputs", who);
    if (O > (1 << 16) || I > (1 << 16) || O * I > (1 << 29)) return fail(ACX_E_INVAL, "%s: up to 65536 outputs and inputs, 2^29 weights", who);
    return ACX_OK;
}
// fn(first row, rows) over launches of fewer than 2^32 lanes, `lpr` lanes a row
template <class F> static void launches(int64_t M, int64_t lpr, F&& fn) {
    const int64_t most = (((int64_t)1 << 32) - 256) / lpr;
    for (int64_t m = 0; m < M; m += most) fn(m, M - m < most ? M - m : most);
}

}  // namespace act8
}  // namespace acx

using namespace acx;

extern "C" int acx_act8_pack(const void* d_x, int64_t x_row, int dtype, int64_t M, int64_t K, int8_t* d_q, uint8_t* d_exponent, void* stream) {
    if (!have_device()) return ACX_E_NODEVICE;
    const int rc = act8::check_rows(M, K, dtype, "acx_act8_pack");
    if (rc) return rc;
    if (M == 0 || K == 0) return ACX_OK;
    if (!d_x || !d_q || !d_exponent) return fail(ACX_E_INVAL, "acx_act8_pack: null pointer");
    const int64_t nb = (K + act8::kBlock - 1) / act8::kBlock, lpr = nb * (dtype == ACX_F32 ? 8 : 4);
    elem::with_element(dtype, [&](auto* e) {
        using E = std::remove_pointer_t<decltype(e)>;
        auto* kernel = M * K * (int64_t)sizeof(E) > elem::kStreamBytes ? act8::k_pack8<E, sizeof(E) == 4 ? 4 : 8, true> : act8::k_pack8<E, sizeof(E) == 4 ? 4 : 8, false>;
        act8::launches(M, lpr, [&](int64_t m, int64_t rows) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)((rows * lpr + 255) / 256)), dim3(256), 0, (hipStream_t)stream, (const E*)d_x + m * x_row, x_row, rows, (int)K, (int)lpr, d_q + m * K,
                               d_exponent + m * nb);
        });
    });
    ACX_HIP_TRY(hipGetLastError());
    return ACX_OK;
}
extern "C" int acx_act8_unpack(const int8_t* d_q, const uint8_t* d_exponent, int64_t M, int64_t K, void* d_x, int dtype, void* stream) {
    if (!have_device()) return ACX_E_NODEVICE;
    const int rc = act8::check_rows(M, K, dtype, "acx_act8_unpack");
    if (rc) return rc;
    if (M == 0 || K == 0) return ACX_OK;
    if (!d_x || !d_q || !d_exponent) return fail(ACX_E_INVAL, "acx_act8_unpack: null pointer");
    const int v = dtype == ACX_F32 ? 4 : 8;
    const int64_t nb = (K + act8::kBlock - 1) / act8::kBlock, lpr = (K + v - 1) / v;
    elem::with_element(dtype, [&](auto* e) {
        using E = std::remove_pointer_t<decltype(e)>;
        auto* kernel = M * K * (int64_t)sizeof(E) > elem::kStreamBytes ? act8::k_unpack8<E, sizeof(E) == 4 ? 4 : 8, true> : act8::k_unpack8<E, sizeof(E) == 4 ? 4 : 8, false>;
        act8::launches(M, lpr, [&](int64_t m, int64_t rows) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)((rows * lpr + 255) / 256)), dim3(256), 0, (hipStream_t)stream, d_q + m * K, d_exponent + m * nb, rows, (int)K, (int)lpr, (E*)d_x + m * K);
        });
    });
    ACX_HIP_TRY(hipGetLastError());
    return ACX_OK;
}
extern "C" int64_t acx_act8_workspace_bytes(int64_t M, int64_t O, int64_t I) {
    if (act8::check_weights(M, O, I, "acx_act8_workspace_bytes")) return 0;
    return act8::work_floats(act8::plan_of(M, O, I), O, I) * 4;
}
extern "C" int acx_act8_weight_grad(const void* d_out_grad, int64_t o_row, int dtype, const int8_t* d_q, const uint8_t* d_exponent, int64_t M, int64_t O, int64_t I, float* d_weight_grad,
                                    float* d_bias_grad, void* d_work, int64_t work_bytes, void* stream) {
    if (!have_device()) return ACX_E_NODEVICE;
    int rc = act8::check_rows(M, O, dtype, "acx_act8_weight_grad");
    if (!rc) rc = act8::check_weights(M, O, I, "acx_act8_weight_grad");
    if (rc) return rc;
    if (o_row < O || o_row >= ((int64_t)1 << 24)) return fail(ACX_E_INVAL, "acx_act8_weight_grad: rows of d_out_grad overlap or lie too far apart (2^24 elements)");
    if (!d_out_grad || !d_q || !d_exponent || !d_weight_grad) return fail(ACX_E_INVAL, "acx_act8_weight_grad: null pointer");
    const act8::Plan p = act8::plan_of(M, O, I);
    const int64_t need = act8::work_floats(p, O, I) * 4;
    if (need && (!d_work || work_bytes < need)) return fail(ACX_E_CAPACITY, "acx_act8_weight_grad: a workspace of %lld bytes is needed (acx_act8_workspace_bytes)", (long long)need);
    act8::Args a = {};
    a.dy = d_out_grad, a.dy_sn = o_row, a.q = d_q, a.exps = d_exponent, a.M = M, a.share = p.share, a.O = (int)O, a.I = (int)I, a.nb = (int)((I + act8::kBlock - 1) / act8::kBlock);
    a.whole = p.whole;
    a.dw = need ? (float*)d_work : d_weight_grad;
    a.db = !d_bias_grad ? nullptr : need ? (float*)d_work + p.shares * O * I : d_bias_grad;
    hipError_t err = hipSuccess;
    elem::with_element(dtype, [&](auto* e) {
        using E = std::remove_pointer_t<decltype(e)>;
        const hipStream_t st = (hipStream_t)stream;
        if (p.to == 64) err = act8::launch<E, 64, 256, 256>(a, p, st);
        else if (p.ti == 64) err = act8::launch<E, 256, 64, 512>(a, p, st);
        else if (p.ti == 128) err = act8::launch<E, 256, 128, 512>(a, p, st);
        else err = act8::launch<E, 256, 256, 512>(a, p, st);
    });
    ACX_HIP_TRY(err);
    if (need) {
        const int64_t groups = (O * I + 63) / 64;
        hipLaunchKernelGGL(act8::k_join_shares, dim3((unsigned)(groups + (d_bias_grad ? (O + 63) / 64 : 0))), dim3(256), 0, (hipStream_t)stream, a.dw, a.db, (int)p.shares, O * I, (int)O,
                           groups, d_weight_grad, d_bias_grad);
        ACX_HIP_TRY(hipGetLastError());
    }
    return ACX_OK;
}
