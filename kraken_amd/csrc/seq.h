// What the operators on sequence rows share (conv_seq.hip, scan_seq.hip, attn_seq.hip, constrain.hip): element types, vector access,
// the activations at fp32 accuracy, and their launchers.
#pragma once
#include "common.h"
#include "../../include/kraken_amd.h"

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

template <class T> __device__ __forceinline__ float to_f(T v) { return (float)v; }
template <class T> __device__ __forceinline__ T from_f(float v) { return (T)v; }   // round to nearest even, once

template <class T> struct VecOf { static constexpr int V = 16 / sizeof(T); };     // elements of a 16-byte access

// V elements at p, of which the first nv exist.  Rows of odd widths start at any element: global memory takes 16-byte accesses at
// element alignment, so a whole vector is one instruction wherever it starts; only the last channel group of a row goes by elements.
template <class T, int V> __device__ __forceinline__ void load_vec(const T* p, int nv, float (&v)[V]) {
    typedef T Tv __attribute__((ext_vector_type(V)));
    if (nv >= V) {
        Tv t;
        __builtin_memcpy(&t, p, sizeof(T) * V);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = to_f<T>(t[i]);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = i < nv ? to_f<T>(p[i]) : 0.f;
    }
}
// the same without the conversion, for loads that are to stay in flight
template <class T, int V> __device__ __forceinline__ auto load_raw(const T* p, int nv) {
    typedef T Tv __attribute__((ext_vector_type(V)));
    Tv t = (Tv)(T)0.f;
    if (nv >= V) __builtin_memcpy(&t, p, sizeof(T) * V);
    else
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < nv) t[i] = p[i];
    return t;
}
template <class T, int V> __device__ __forceinline__ void store_vec(T* p, int nv, const float (&v)[V]) {
    typedef T Tv __attribute__((ext_vector_type(V)));
    if (nv >= V) {
        Tv t;
#pragma unroll
        for (int i = 0; i < V; ++i) t[i] = from_f<T>(v[i]);
        __builtin_memcpy(p, &t, sizeof(T) * V);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < nv) p[i] = from_f<T>(v[i]);
    }
}

__device__ __forceinline__ float seq_silu(float p) { return p * __builtin_amdgcn_rcpf(1.f + __expf(-p)); }

// softplus(v) = max(v, 0) + log1p(e), e = exp(-|v|) in (0, 1].  log1p(e) = 2 atanh(r), r = e / (2 + e) <= 1/3, by its odd series up to r^15
// (the rest is below 2^-27 of it): one exp, one rcp, and full relative accuracy where the result is tiny, which log(1 + e) does not have.
// The exponent's product with log2 e would be off by |v| 2^-24, which a step width passes on whole; what its rounding and the constant's lose
// goes into e as a factor 1 + loss ln 2.
__device__ __forceinline__ float seq_softplus(float v) {
    constexpr float L = 1.4426950408889634f, REST = (float)(1.4426950408889634 - (double)L), LN2 = 0.6931471805599453f;
    const float a = fabsf(v) > 200.f ? 200.f : fabsf(v), t = a * L;    // beyond 200: e is zero, and an infinite a would have no rest
    const float loss = __builtin_fmaf(a, REST, __builtin_fmaf(a, L, -t));
    float e = __builtin_amdgcn_exp2f(-t);
    e = __builtin_fmaf(e, loss * -LN2, e);
    const float r = e * __builtin_amdgcn_rcpf(2.f + e), q = r * r;
    float p = 2.f / 15.f;
    p = __builtin_fmaf(p, q, 2.f / 13.f);
    p = __builtin_fmaf(p, q, 2.f / 11.f);
    p = __builtin_fmaf(p, q, 2.f / 9.f);
    p = __builtin_fmaf(p, q, 2.f / 7.f);
    p = __builtin_fmaf(p, q, 2.f / 5.f);
    p = __builtin_fmaf(p, q, 2.f / 3.f);
    p = __builtin_fmaf(p, q, 2.f);
    return __builtin_fmaf(p, r, fmaxf(v, 0.f));
}

__device__ __forceinline__ int seq_len(const int* lens, int n, int T) {
    return lens ? min(max(lens[n], 0), T) : T;
}

// a grid's threads fit 32 bits
inline bool seq_grid_too_large(long blocks, int threads) { return blocks > 0xffffffffL / threads; }

// launchers: 0, -1 when the launch failed, -4 for more rows than a grid holds
int krk_launch_causal_conv(const krk_conv_args& a, hipStream_t s);
long krk_scan_workspace(const krk_scan_args& a);
int krk_launch_selective_scan(const krk_scan_args& a, hipStream_t s);
long krk_attn_workspace(const krk_attention_args& a);
int krk_launch_attention(const krk_attention_args& a, hipStream_t s);
int krk_launch_constrain(const krk_constrain_args& a, hipStream_t s);
