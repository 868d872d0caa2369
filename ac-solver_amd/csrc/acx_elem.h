// acx_elem.h -- element types and wave helpers of the recurrent agent's operators (acx_scan.hip, acx_block.hip, acx_act8.hip).
#pragma once
#include "acx_common.h"

namespace acx {
namespace elem {

// Activations are float, bfloat16 or float16; every computation on them is in float32.  A rounding to 16 bits is the hardware's, to
// nearest even, and happens once, at the store.
typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// V elements of E behind a pointer that is aligned for E alone: a strided slice, or a row of odd width, may start anywhere, and global
// memory takes 16-byte accesses at any address on this chip (a misaligned one costs a second cache line at most)
template <class E, int V> struct Vec {
    typedef E type __attribute__((ext_vector_type(V), aligned(sizeof(E))));
};
template <class E> struct Vec<E, 1> {
    typedef E type;
};

// STREAM: past the caches, for tensors that do not fit them anyway: what is in the Infinity Cache stays there, and the lines of a stream do not wait
// to be written back (a pass over 1 GB tensors 5 to 7 % faster; over 34 MB ones, which the next kernel finds in the cache, 11 % slower).
constexpr int64_t kStreamBytes = (int64_t)256 << 20;
template <class E, int V, bool STREAM> __device__ __forceinline__ typename Vec<E, V>::type load_vec(const E* p) {
    if constexpr (STREAM) return __builtin_nontemporal_load((const typename Vec<E, V>::type*)p);
    else return *(const typename Vec<E, V>::type*)p;
}
template <class E, int V, bool STREAM = false> __device__ __forceinline__ void load(const E* p, float (&out)[V]) {
    if constexpr (V == 1) {
        out[0] = (float)*p;
    } else {
        const typename Vec<E, V>::type v = load_vec<E, V, STREAM>(p);
#pragma unroll
        for (int i = 0; i < V; i++) out[i] = (float)v[i];
    }
}
template <class E, int V, bool STREAM = false> __device__ __forceinline__ void store(E* p, const float (&in)[V]) {
    if constexpr (V == 1) {
        *p = (E)in[0];
    } else {
        typename Vec<E, V>::type v;
#pragma unroll
        for (int i = 0; i < V; i++) v[i] = (E)in[i];
        if constexpr (STREAM) __builtin_nontemporal_store(v, (typename Vec<E, V>::type*)p);
        else *(typename Vec<E, V>::type*)p = v;
    }
}
// The first `valid` of V elements (the end of a row, or nothing at all), in two steps, for loads that are started well before their values are looked
// at.  `ahead`: V elements can be read all the same, what stands behind the row's end is another row's or a gap's -- one load, where an
// element at a time costs V.  `widen` takes the values and makes those behind the end zero.
template <class E, int V, bool STREAM = false> __device__ __forceinline__ typename Vec<E, V>::type load_raw(const E* p, int valid, bool ahead) {
    typename Vec<E, V>::type v = {};
    if (valid >= V || (valid > 0 && ahead)) {
        v = load_vec<E, V, STREAM>(p);
    } else {
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i < valid) v[i] = p[i];
    }
    return v;
}
template <class E, int V> __device__ __forceinline__ void widen(const typename Vec<E, V>::type& v, int valid, float (&out)[V]) {
#pragma unroll
    for (int i = 0; i < V; i++) out[i] = (float)v[i];
    if (valid < V) {
#pragma unroll
        for (int i = 0; i < V; i++) out[i] = i < valid ? out[i] : 0.0f;
    }
}
template <class E, int V, bool STREAM = false> __device__ __forceinline__ void load_some(const E* p, int valid, float (&out)[V], bool ahead = false) {
    widen<E, V>(load_raw<E, V, STREAM>(p, valid, ahead), valid, out);
}
// (in pieces of 4, 2 and 1, by the bits of `valid`)
template <class E, int V, bool STREAM = false> __device__ __forceinline__ void store_some(E* p, int valid, const float (&in)[V]) {
    static_assert(V == 2 || V == 4 || V == 8, "pieces");
    if (valid >= V) {
        store<E, V, STREAM>(p, in);
    } else if (valid > 0) {
        float v[V];
#pragma unroll
        for (int i = 0; i < V; i++) v[i] = in[i];
        if constexpr (V > 4) {
            if (valid & 4) {
                const float a[4] = {v[0], v[1], v[2], v[3]};
                store<E, 4>(p, a);
                p += 4;
#pragma unroll
                for (int i = 0; i < 4; i++) v[i] = v[i + 4];
            }
        }
        if constexpr (V > 2) {
            if (valid & 2) {
                const float a[2] = {v[0], v[1]};
                store<E, 2>(p, a);
                p += 2;
                v[0] = v[2];
            }
        }
        if (valid & 1) *p = (E)v[0];
    }
}

// v + the value of the lane that a DPP control names: neighbours 1, 2, 4 and 8 apart cost one vector instruction and no trip through LDS
template <int CTRL> __device__ __forceinline__ float add_dpp(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}
// sum over groups of LANES (1 ... 64, a power of two) neighbouring lanes, the same bits in every one of them
template <int LANES> __device__ __forceinline__ float lane_sum(float v) {
    if constexpr (LANES > 1) v = add_dpp<0xB1>(v);   // quad_perm 1 0 3 2
    if constexpr (LANES > 2) v = add_dpp<0x4E>(v);   // quad_perm 2 3 0 1
    if constexpr (LANES > 4) v = add_dpp<0x141>(v);  // mirrored within 8
    if constexpr (LANES > 8) v = add_dpp<0x140>(v);  // mirrored within 16
    if constexpr (LANES > 16) v += __shfl_xor(v, 16);
    if constexpr (LANES > 32) v += __shfl_xor(v, 32);
    return v;
}

// sigmoid of z and of -z from one exponential: with e = exp(-|z|) the larger of the two is 1 / (1 + e) and the smaller e / (1 + e), which
// keeps its accuracy where 1 - sigmoid would lose it.  exp(-|z|) = 2^t (1 + l ln 2) with t = -|z| log2 e rounded and l what the rounding
// and the constant left out: the error of t alone would grow to |z| 2^-24.  PRECISE false leaves l out: for 16-bit results.
// NaN comes out as NaN, +-infinity as 0 and 1.
struct Sigmoid {
    float large, small;
};
template <bool PRECISE> __device__ __forceinline__ Sigmoid sigmoid_pair(float z) {
    constexpr float kLog2e = 1.44269502162933349609375f, kLog2eLow = 1.92596299e-8f, kLn2 = 0.693147182464599609375f;
    const float a = -__builtin_fabsf(z);
    const float t = a * kLog2e;
    float e = __builtin_amdgcn_exp2f(t);
    if constexpr (PRECISE) {
        const float l = __builtin_fmaf(a, kLog2eLow, __builtin_fmaf(a, kLog2e, -t));
        // (at infinity l is NaN and e is 0: the comparison keeps the 0, and a NaN of z is in e already)
        e = t < -126.0f ? e : __builtin_fmaf(e * l, kLn2, e);
    }
    const float r = __builtin_amdgcn_rcpf(1.0f + e);
    return {r, e * r};
}
// sigmoid(z) and 1 - sigmoid(z)
__device__ __forceinline__ float keep_of(float z, Sigmoid s) { return z < 0.0f ? s.small : s.large; }
__device__ __forceinline__ float take_of(float z, Sigmoid s) { return z < 0.0f ? s.large : s.small; }

// run fn.template operator()<E>() for the element type of an ACX_* code; false for any other code
template <class F> static inline bool with_element(int dtype, F&& fn) {
    switch (dtype) {
        case ACX_F32: fn((float*)nullptr); return true;
        case ACX_BF16: fn((bf16_t*)nullptr); return true;
        case ACX_F16: fn((f16_t*)nullptr); return true;
        default: return false;
    }
}
static inline int element_bytes(int dtype) { return dtype == ACX_F32 ? 4 : 2; }

}  // namespace elem
}  // namespace acx
