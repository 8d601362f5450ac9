// What the two attention kernels share: the cap, and what the masks say about a query.
#pragma once
#include "seq.h"

constexpr float LOG2E = 1.4426950408889634f;

// 16-bit results take cap tanh's error of 2^-23 of the cap up to this one (2^-13 of a weight then, a quarter of fp16's half step)
constexpr float COARSE_CAP = 1024.f;

// cap tanh(s / cap).  fp32: the odd series below 0.45 (the rest is under 2^-25 of it), where 1 - 2 / (1 + e^2x) would cancel; 16-bit results
// need no more than the latter up to COARSE_CAP.
template <class T> __device__ __forceinline__ float seq_cap(float s, float cap, float rcap) {
    const float x = s * rcap, ax = fabsf(x);
    const float e = __builtin_amdgcn_exp2f(-2.f * LOG2E * ax);
    float big = (1.f - e) * __builtin_amdgcn_rcpf(1.f + e);
    if constexpr (sizeof(T) == 4) {
        const float q = x * x;
        float p = 21844.f / 6081075.f;
        p = __builtin_fmaf(p, q, -1382.f / 155925.f);
        p = __builtin_fmaf(p, q, 62.f / 2835.f);
        p = __builtin_fmaf(p, q, -17.f / 315.f);
        p = __builtin_fmaf(p, q, 2.f / 15.f);
        p = __builtin_fmaf(p, q, -1.f / 3.f);
        p = __builtin_fmaf(p * q, ax, ax);
        big = ax < 0.45f ? p : big;
    }
    return cap * __builtin_copysignf(big, x);
}

struct AttnRow {               // what the masks say about one query
    int klen, limit, p;    // keys [0, klen), of which j < limit or (not causal): limit = max(p + 1, prefix)
};
__device__ __forceinline__ AttnRow query_row(const krk_attention_args& a, int n, int i) {
    AttnRow r;
    const int qlen = seq_len(a.q_lens, n, a.Tq);
    r.klen = seq_len(a.k_lens, n, a.Tk);
    r.p = a.align_end ? r.klen - qlen + i : i;
    r.limit = r.klen;
    if (a.causal) r.limit = min(r.klen, max(r.p + 1, a.prefix ? a.prefix[n] : 0));
    if (i >= qlen) r.limit = 0;
    return r;
}

// queries of a workgroup, keys of a tile, and splits of the key axis of the tile kernel (attn_tile.hip); its scratch in front of the joined rows
struct AttnTiles {
    int rows, keys, splits;
    long range_bytes;
};
AttnTiles krk_attn_tiles(const krk_attention_args& a);
int krk_launch_attn_tiles(const krk_attention_args& a, const AttnTiles& g, void* range_scratch, hipStream_t s);
