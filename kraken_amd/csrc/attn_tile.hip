// Attention of many queries: a workgroup of NW waves holds NW * 32 queries of one head and walks the key tiles that its masks leave.
//
// Scores are computed transposed, S^T = K Q^T on 32x32 matrix instructions: a lane then owns ONE query (its column) and 16 keys per block, so
// the running maximum and sum of the softmax are registers of a lane plus one exchange with the lane 32 away, and the weights are already the B
// operand of the second product O^T = V^T P^T -- the order of the keys inside a contraction is free, so V is read in the order in which the
// scores lie.  16-bit types: 32x32x16, V^T by transposing LDS reads (ds_read_b64_tr_b16) from row-major tiles.  fp32: the exact 32x32x2.
// Key tiles pass through two LDS buffers, the next one's loads are in flight while a tile is computed; one barrier a tile.
//
// What bounds it: 16-bit heads of 64 channels the vector units (per score a multiply-add, an exponential, a maximum, a sum and two to three for the weight in two parts
// against 24 matrix instructions per 64 x 32 scores; the cap adds an exponential and a reciprocal): 2 x 4000 x 16 x 64 fp16, capped, causal with a prefix:
// 184 us, 293 TFLOP/s.  fp32 the matrix units on long rows (16 x 2048 x 8 x 64: 118 of 154 TFLOP/s), on short lines the loads in front of each
// workgroup, which two waves per SIMD do not cover (256 ragged lines of 150 x 8 x 50: 132 us, 46 of them matrix time).  Packed documents
// (8192 steps, 24 of them, 16 x 128 bf16): 78 + 5 us, most of it the latency of 1 to 16 tiles per workgroup.  Both units are far from full there: the
// vector units issue in 43 % of the CUs' busy cycles and the matrix units run in 25 % (capped prefix 63 and 21 %), at 1.6 to 1.9 waves per SIMD.
#include "attn_seq.h"

namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x16 mfma16(bf16_t, const s16x8& a, const s16x8& b, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma16(f16_t, const s16x8& a, const s16x8& b, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma16(float, const s16x8&, const s16x8&, const f32x16& c) { return c; }

// Two weights, each as the sum of two numbers of the type: the nearest one, and what is left of the weight.
typedef float f32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void two_parts(f16_t, f32x2 w, unsigned& first, unsigned& rest) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    first = __builtin_bit_cast(unsigned, __builtin_convertvector(w, f16x2));
    // w - first, with half a word as operand: no conversion back.  An exponential's result must not be read by the very next instruction, which the
    // compiler does not see to for assembly: the conversion above stands in between.
    f32x2 r;
    asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r.x) : "v"(first), "v"(w.x));
    asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r.y) : "v"(first), "v"(w.y));
    rest = __builtin_bit_cast(unsigned, __builtin_convertvector(r, f16x2));
}
__device__ __forceinline__ void two_parts(bf16_t, f32x2 w, unsigned& first, unsigned& rest) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    first = __builtin_bit_cast(unsigned, __builtin_convertvector(w, bf16x2));
    const f32x2 r = {w.x - __builtin_bit_cast(float, first << 16), w.y - __builtin_bit_cast(float, first & 0xffff0000u)};
    rest = __builtin_bit_cast(unsigned, __builtin_convertvector(r, bf16x2));
}

// A head is read in chunks of 16 bytes; where its E channels are no whole number of them, the last chunk is loaded so that it ENDS there: one load
// without a condition whatever E is, and none past the row.  Its first channels are in the chunk before as well: values are kept so,
// the query and the keys have zeros in their place (both: 0 times an infinite key is no number), and the result of such a channel is stored once.
// Chunks behind the last repeat it, query and key zero.
template <class T> __device__ __forceinline__ u32x4 load_chunk(const T* row, int e, int E) {
    u32x4 r;
    __builtin_memcpy(&r, row + min(e, E - VecOf<T>::V), 16);
    return r;
}
// the query's or a key's chunk at e: without the channels that the chunk before has, and nothing behind the end
template <class T> __device__ __forceinline__ u32x4 own_chunk(u32x4 r, int e, int E) {
    typedef T Tv __attribute__((ext_vector_type(VecOf<T>::V)));
    Tv v = __builtin_bit_cast(Tv, r);
#pragma unroll
    for (int i = 0; i < VecOf<T>::V; ++i) v[i] = i >= e - (E - VecOf<T>::V) && e < E ? v[i] : (T)0.f;
    return __builtin_bit_cast(u32x4, v);
}

// the lane 32 away: a query's keys lie in two lanes
__device__ __forceinline__ float other_half_max(float v) {
    const unsigned u = __builtin_bit_cast(unsigned, v);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__builtin_bit_cast(float, (unsigned)r[0]), __builtin_bit_cast(float, (unsigned)r[1]));
}
__device__ __forceinline__ unsigned other_half_or(unsigned u) {
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return (unsigned)r[0] | (unsigned)r[1];
}
__device__ __forceinline__ float other_half_sum(float v) {
    const unsigned u = __builtin_bit_cast(unsigned, v);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
}

// exponent bits all ones: infinity or NaN
template <class T> __device__ __forceinline__ bool odd_value(unsigned short v) {
    constexpr unsigned short M = sizeof(T) == 2 && __is_same(T, bf16_t) ? 0x7f80 : 0x7c00;
    return (v & M) == M;
}
__device__ __forceinline__ bool odd_float(float v) { return (__builtin_bit_cast(unsigned, v) & 0x7f800000u) == 0x7f800000u; }

// the largest magnitude bits so far (both halves of a word apart), and whether one of them is odd
template <class T> __device__ __forceinline__ unsigned odd_max(unsigned high, unsigned w) {
    if constexpr (sizeof(T) == 4) return max(high, w & 0x7fffffffu);
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(u16x2, high), __builtin_bit_cast(u16x2, w & 0x7fff7fffu)));
}
template <class T> __device__ __forceinline__ bool odd_found(unsigned high) {
    if constexpr (sizeof(T) == 4) return high >= 0x7f800000u;
    return odd_value<T>(high & 0xffff) || odd_value<T>(high >> 16);
}

template <class T, int EP, int NW> struct Geo {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int BK = F32 || NW < 4 ? 32 : 64;                    // keys of a tile
    static constexpr int SB = BK / 32, EB = EP / 32;
    static constexpr int KLD = F32 ? EP + 4 : EP + 8;                     // row pitches (elements) that spread a read over the banks:
    static constexpr int VLD = F32 ? EP + 8 : EP + (EP % 128 ? (EP % 64 ? 0 : 32) : 32);   // K rows by 16 bytes, V rows by quads of rows
    static constexpr int CV = VecOf<T>::V;                                // elements of a 16-byte chunk
    static constexpr int CHUNKS = BK * EP / CV;
};

// tile key ranges of the documents: min and max id of every tile's valid keys
__global__ __launch_bounds__(256) void attn_ranges_kernel(krk_attention_args a, int2* out, int tiles, int keys) {
    const long id = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (id >= (long)a.N * tiles) return;
    const int n = id / tiles, t = id % tiles, lane = threadIdx.x & 63;
    const int j = t * keys + lane;
    const bool in = lane < keys && j < seq_len(a.k_lens, n, a.Tk);
    int lo = in ? a.documents[n * a.doc_n + j] : 0x7fffffff, hi = in ? lo : (int)0x80000000;
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) lo = min(lo, __shfl_xor(lo, x)), hi = max(hi, __shfl_xor(hi, x));
    if (lane == 0) out[id] = make_int2(lo, hi);
}

// four channels at p, the first `from` of which are stored already
template <class T> __device__ __forceinline__ void put_four(T* p, int from, const float (&v)[4]) {
    if (from == 0) store_vec<T, 4>(p, 4, v);
    else
#pragma unroll
        for (int i = 1; i < 4; ++i)
            if (i >= from) p[i] = from_f<T>(v[i]);
}

// a statement for every score of a lane: s[x][i]
#define EACH(...)                          \
    _Pragma("unroll") for (int x = 0; x < NJ; ++x) _Pragma("unroll") for (int i = 0; i < 16; ++i) { __VA_ARGS__; }

template <class T, int EP, int NW>
__global__ __launch_bounds__(NW * 64, EP * sizeof(T) > 256 ? 1 : 2) void attn_tile_kernel(krk_attention_args a, int qblocks, int cut, int batch, int splits, int tiles, const int2* ranges) {
    using G = Geo<T, EP, NW>;
    constexpr bool F32 = G::F32;
    constexpr int BK = G::BK, SB = G::SB, EB = G::EB, KLD = G::KLD, VLD = G::VLD, CV = G::CV, NT = NW * 64;
    // fp16 weights are raised by 2^7, to 2^15 at most: their smallest step, 2^-24, is then 2^-31 of the row's largest weight
    constexpr float LIFT = __is_same(T, f16_t) ? 7.f : 0.f;
    constexpr int NJ = !F32 && NW == 4 && EP <= 64 ? 2 : 1;               // blocks of 32 keys at once: more to overlap, where the registers allow it
    constexpr int CPT = (G::CHUNKS + NT - 1) / NT, CPR = EP / CV;         // chunks per thread and per row
    __shared__ __attribute__((aligned(16))) T Kbuf[2][BK * KLD];
    __shared__ __attribute__((aligned(16))) T Vbuf[2][BK * VLD];
    __shared__ __attribute__((aligned(16))) int dbuf[2][BK];
    __shared__ int odd[4];
    __shared__ unsigned infs[2][2][SB][EP];                               // where the tile's odd values were: +inf / -inf (NaN: both), a bit per key

    // All query blocks and heads that share a key head run on one XCD (workgroups go round the eight of them), so its L2 holds their keys; where
    // the key heads do not go round evenly each is cut into `cut` interleaved parts.  `batch` of them, as many as the L2 holds, are taken together,
    // the blocks with the longest causal rows first, so that the short ones fill the end.
    const int rep = a.H / a.Hk, inner = qblocks * rep, part_size = (inner + cut - 1) / cut;
    const long id = blockIdx.x / 8, per_xcd = gridDim.x / 8 / part_size, first = id / ((long)part_size * batch) * batch;
    const int width = (int)min((long)batch, per_xcd - first), at = (int)(id - first * part_size);
    const long group = (blockIdx.x & 7) + 8 * (first + at % width);
    const int in = at / width * cut + (int)(group % cut);
    if (in >= inner) return;
    const long kvh = group / cut;
    const int n = kvh / a.Hk, hk = kvh % a.Hk;
    const int h = hk * rep + in % rep, q0 = (qblocks - 1 - in / rep) * NW * 32;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, col = lane & 31;
    const int qlen = seq_len(a.q_lens, n, a.Tq), split = blockIdx.y;
    const int qi = q0 + wave * 32 + col;                                  // this lane's query
    T* out = (T*)a.out + n * a.o_n + h * a.o_h;
    const int* docs = a.documents ? a.documents + n * a.doc_n : nullptr;

    // what the masks say: about this lane's query, about the wave's first (the shortest reach) and last one, about the workgroup
    const int klen = seq_len(a.k_lens, n, a.Tk);
    const AttnRow mine = query_row(a, n, min(qi, a.Tq - 1));
    const int lim = qi < qlen ? mine.limit : 0;
    const int wfirst = q0 + wave * 32, wlast = min(wfirst + 31, qlen - 1);
    const bool awake = wfirst < qlen;
    const int wmin = awake ? query_row(a, n, wfirst).limit : 0, wmax = awake ? query_row(a, n, wlast).limit : 0;
    const int bfirst = min(q0, qlen - 1), blast = min(q0 + NW * 32, qlen) - 1;
    const int bmax = q0 < qlen ? query_row(a, n, blast).limit : 0;
    const int bmin = q0 < qlen ? query_row(a, n, bfirst).limit : 0;
    int doc = 0, wlo = 0, whi = 0, blo = 0, bhi = 0;
    if (docs && q0 < qlen) {
        doc = docs[min(qi, qlen - 1)];
        wlo = whi = doc;
        blo = 0x7fffffff, bhi = (int)0x80000000;
        for (int i = lane; i < NW * 32; i += 64) {
            const int d = docs[min(q0 + i, qlen - 1)];
            blo = min(blo, d), bhi = max(bhi, d);
        }
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) {
            wlo = min(wlo, __shfl_xor(wlo, x)), whi = max(whi, __shfl_xor(whi, x));
            blo = min(blo, __shfl_xor(blo, x)), bhi = max(bhi, __shfl_xor(bhi, x));
        }
    }

    // the query as B operand: column = query.  16-bit: 8 channels from 16 ks + 8 half; fp32: 4 from 8 g + 4 half.  A negative scale turns its sign.
    const float sign = a.scale > 0.f ? 1.f : a.scale < 0.f ? -1.f : 0.f;
    const float c = (a.scale != 0.f ? fabsf(a.scale) : 1.f) * LOG2E;
    s16x8 q16[F32 ? 1 : EP / 16];
    f32x4 q32[F32 ? EP / 8 : 1];
    constexpr int NQ = F32 ? EP / 8 : EP / 16, STEP = F32 ? 8 : 16;
    u32x4 raw[NQ];
    {
        const T* qp = (const T*)a.q + n * a.q_n + (long)min(qi, a.Tq - 1) * a.q_t + h * a.q_h;
#pragma unroll
        for (int x = 0; x < NQ; ++x) raw[x] = load_chunk<T>(qp, STEP * x + STEP / 2 * half, a.E);
    }
    const float slope = a.slopes ? a.slopes[h] * LOG2E : 0.f;
    const float rcap = a.cap > 0.f ? 1.f / a.cap : 0.f;
    const bool plain = a.cap <= 0.f && !a.slopes;

    f32x16 o[EB];
#pragma unroll
    for (int eb = 0; eb < EB; ++eb)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[eb][i] = 0.f;
    float m = -INFINITY, l = 0.f;

    // the tiles of this split that the masks leave, 64 at a time as bits
    const int want = (bmax + BK - 1) / BK;
    const int span = (tiles + splits - 1) / splits;
    const int t1 = min(want, (split + 1) * span);
    int base = split * span - 64;
    unsigned long long left = 0;
    int2 here = make_int2(0, 0), now = make_int2(0, 0);                   // id ranges: of the tile that this lane looked at, of the one taken
    auto next = [&]() -> int {
        while (!left) {
            base += 64;
            if (base >= t1) return -1;
            const int t = base + lane;
            bool in = t < t1;
            if (docs && in) {
                here = ranges[(long)n * tiles + t];
                in = here.x <= bhi && here.y >= blo;
            }
            left = __ballot(in);
        }
        const int b = __builtin_ctzll(left);
        left &= left - 1;
        now = make_int2(__builtin_amdgcn_readlane(here.x, b), __builtin_amdgcn_readlane(here.y, b));
        return base + b;
    };

    const T* kp = (const T*)a.k + n * a.k_n + hk * a.k_h;
    const T* vp = (const T*)a.v + n * a.v_n + hk * a.v_h;
    u32x4 kr[CPT], vr[CPT];
    int dr = 0;
    auto fetch = [&](int t) {                                             // rows behind the last valid key repeat it: they are masked
#pragma unroll
        for (int x = 0; x < CPT; ++x) {
            const int id = threadIdx.x + x * NT, row = id / CPR, e = (id - row * CPR) * CV;
            const int j = min(t * BK + (G::CHUNKS % NT == 0 ? row : min(row, BK - 1)), klen - 1);
            kr[x] = load_chunk<T>(kp + (long)j * a.k_t, e, a.E);
            vr[x] = load_chunk<T>(vp + (long)j * a.v_t, e, a.E);
        }
        if (docs && threadIdx.x < BK) dr = docs[min(t * BK + (int)threadIdx.x, klen - 1)];
    };

    // A value that is not finite must not reach the queries that may not see it: 0 x NaN is NaN.  Only tiles that some query of the workgroup sees
    // in part can do that; they are searched while they go to LDS.
    // 16-bit types search every tile: their weights are two numbers, whose products with an infinity may be of either sign, or none at all.
    auto search = [&](int t) { return !F32 || docs || (t + 1) * BK > bmin; };
    constexpr bool ONE = NT % CPR == 0;                                   // a thread's chunks are all of the same channels
    // (ANDed with a mask kept in registers: 131 -> 132.5 us on the lines above; chosen anew for every tile 137)
    const u32x4 all = {~0u, ~0u, ~0u, ~0u}, keep = own_chunk<T>(all, (int)threadIdx.x % CPR * CV, a.E);
    auto put = [&](int t, int buf, int turn) {
        bool hit = false;
        if (a.E != EP)
#pragma unroll
            for (int x = 0; x < CPT; ++x) kr[x] &= ONE ? keep : own_chunk<T>(all, (int)(threadIdx.x + x * NT) % CPR * CV, a.E);
        if (search(t)) {
            unsigned high = 0;
#pragma unroll
            for (int x = 0; x < CPT; ++x)
#pragma unroll
                for (int i = 0; i < 4; ++i) high = odd_max<T>(high, vr[x][i]);
            hit = odd_found<T>(high);
            if (hit) odd[turn & 3] = 1;
        }
#pragma unroll
        for (int x = 0; x < CPT; ++x) {
            const int id = threadIdx.x + x * NT, row = id / CPR, e = (id - row * CPR) * CV;
            if (G::CHUNKS % NT == 0 || id < G::CHUNKS) {
                *(u32x4*)&Kbuf[buf][row * KLD + e] = kr[x];
                *(u32x4*)&Vbuf[buf][row * VLD + e] = vr[x];
                if (hit)                                                  // its own elements again, one by one
                    for (int i = 0; i < CV; ++i) {
                        const float v = to_f<T>(Vbuf[buf][row * VLD + e + i]);
                        if (!odd_float(v)) continue;
                        if (!(v < 0.f)) atomicOr(&infs[buf][0][row >> 5][e + i], 1u << (row & 31));
                        if (!(v > 0.f)) atomicOr(&infs[buf][1][row >> 5][e + i], 1u << (row & 31));
                        Vbuf[buf][row * VLD + e + i] = from_f<T>(0.f);
                    }
            }
        }
        if (docs && threadIdx.x < BK) dbuf[buf][threadIdx.x] = dr;
    };
    auto clear = [&](int buf) {
        for (int i = threadIdx.x; i < 2 * SB * EP; i += NT) (&infs[buf][0][0][0])[i] = 0;
    };

    for (int x = 0; x < 2; ++x) clear(x);
    if (threadIdx.x < 4) odd[threadIdx.x] = 0;
    __syncthreads();
    int tile = next(), turn = 0;
    bool was = false;
    if (tile >= 0) fetch(tile);
#pragma unroll
    for (int x = 0; x < NQ; ++x) {
        if (a.E != EP) raw[x] = own_chunk<T>(raw[x], STEP * x + STEP / 2 * half, a.E);
        if constexpr (F32) q32[x] = __builtin_bit_cast(f32x4, raw[x]) * sign;
        else {
            q16[x] = __builtin_bit_cast(s16x8, raw[x]);
            if (a.scale <= 0.f)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const short one = q16[x][i];                          // a copy: a bit cast of a vector's element reads its first one
                    q16[x][i] = __builtin_bit_cast(short, from_f<T>(to_f(__builtin_bit_cast(T, one)) * sign));
                }
        }
    }
    if (tile >= 0) put(tile, 0, 0);
    __builtin_amdgcn_s_waitcnt(0x0f70);                                   // vmcnt(0): nothing of the prologue is waited for behind the loop's own loads
    __syncthreads();
    while (tile >= 0) {
        const int t = tile, k0 = t * BK, buf = turn & 1;
        const int2 r = now;
        const bool bad = search(t) && odd[turn & 3];
        if (threadIdx.x == 0) odd[(turn + 2) & 3] = 0;                    // the flag that the next turn sets, read two turns ago
        if (was) {                                                        // the places that the next tile's go to, read in the last turn
            clear(buf ^ 1);
            __syncthreads();
        }
        was = bad;
        ++turn;
        tile = next();
        if (tile >= 0) fetch(tile);

        bool see = awake && k0 < wmax, part = k0 + BK > wmin;
        if (docs && see) {
            see = r.x <= whi && r.y >= wlo;
            part = part || r.x != r.y || wlo != whi;
        }
        if (see) {
            const T *Ks = Kbuf[buf], *Vs = Vbuf[buf];
#pragma unroll
            for (int b0 = 0; b0 < SB; b0 += NJ) {
                // S^T = K Q^T of NJ blocks of 32 keys; register i of block b: key k0 + 32 b + 8 (i / 4) + 4 half + i % 4
                f32x16 s[NJ];
#pragma unroll
                for (int x = 0; x < NJ; ++x) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[x][i] = 0.f;
                    const T* kb = &Ks[((b0 + x) * 32 + col) * KLD];
                    if constexpr (F32) {
#pragma unroll
                        for (int g = 0; g < EP / 8; ++g) {
                            const f32x4 k = *(const f32x4*)&kb[8 * g + 4 * half];
#pragma unroll
                            for (int i = 0; i < 4; ++i) s[x] = __builtin_amdgcn_mfma_f32_32x32x2f32(k[i], q32[g][i], s[x], 0, 0, 0);
                        }
                    } else {
#pragma unroll
                        for (int ks = 0; ks < EP / 16; ++ks) s[x] = mfma16(T{}, *(const s16x8*)&kb[16 * ks + 8 * half], q16[ks], s[x]);
                    }
                }
                float scale = c;
                if (!plain) {
                    scale = 1.f;
                    if (a.cap > 0.f) {
                        if (F32 || a.cap > COARSE_CAP) {
                            const float raw = c * (1.f / LOG2E);
                            EACH(s[x][i] = seq_cap<float>(s[x][i] * raw, a.cap, rcap) * LOG2E);
                        } else {                                          // cap tanh(x) = cap - 2 cap / (1 + e^2x): 2^-23 of cap off at most
                            const float cl = a.cap * LOG2E, cx = 2.f * c * rcap;
                            EACH(s[x][i] = __builtin_fmaf(-2.f * cl, __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(s[x][i] * cx)), cl));
                        }
                    } else {
                        EACH(s[x][i] *= c);
                    }
                    if (a.slopes) {
                        const float d0 = (float)(mine.p - k0 - 32 * b0 - 4 * half);
                        EACH(s[x][i] = __builtin_fmaf(-slope, fabsf(d0 - (float)(32 * x + 8 * (i / 4) + i % 4)), s[x][i]));
                    }
                }
                if (part) {
                    const int room = lim - k0 - 32 * b0 - 4 * half;
                    EACH(s[x][i] = 32 * x + 8 * (i / 4) + i % 4 < room ? s[x][i] : -INFINITY);
                    if (docs)
#pragma unroll
                        for (int x = 0; x < NJ; ++x) {
                            int4 ids[4];
#pragma unroll
                            for (int g = 0; g < 4; ++g) ids[g] = *(const int4*)&dbuf[buf][32 * (b0 + x) + 8 * g + 4 * half];
#pragma unroll
                            for (int i = 0; i < 16; ++i) s[x][i] = (&ids[i / 4].x)[i % 4] == doc ? s[x][i] : -INFINITY;
                        }
                }
                float top = s[0][0];
                EACH(top = fmaxf(top, s[x][i]));
                top = other_half_max(top) * scale;
                // The reference point moves only when a score passes it by 2^8: weights up to 256 are as exact, and most tiles leave the sums alone.
                if (__ballot(top > m + 8.f)) {
                    const float nm = fmaxf(m, top), f = __builtin_amdgcn_exp2f(m - (nm == -INFINITY ? 0.f : nm));
                    m = nm;
                    l *= f;
#pragma unroll
                    for (int eb = 0; eb < EB; ++eb)
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[eb][i] *= f;
                }
                const float ref = m == -INFINITY ? 0.f : m - LIFT;
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
                EACH(s[x][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][i], scale, -ref)); sum[i % 4] += s[x][i]);
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);

                // O^T += V^T P^T
                unsigned seen[NJ];                                        // of this half's keys, those with a weight
                if (bad) {
                    EACH(seen[x] = (i ? seen[x] : 0u) | (s[x][i] != 0.f ? 1u << (8 * (i / 4) + i % 4) : 0u));
                }
                if constexpr (F32) {
#pragma unroll
                    for (int eb = 0; eb < EB; ++eb)
#pragma unroll
                        for (int x = 0; x < NJ; ++x) {
                            const T* vb = &Vs[((b0 + x) * 32 + 4 * half) * VLD + eb * 32 + col];
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                                o[eb] = __builtin_amdgcn_mfma_f32_32x32x2f32(vb[(8 * (i / 4) + i % 4) * VLD], s[x][i], o[eb], 0, 0, 0);
                        }
                } else {
                    // Weights as two numbers of the values' type, a matrix instruction for each: the first alone is half a step off (2^-8 bf16,
                    // 2^-11 fp16), more than the one rounding at the end; with the rest 2^-16 and 2^-22.  The first alone: capped prefix
                    // 162 us instead of 184, documents 83 instead of 90.
                    u32x4 p[2 * NJ], rest[2 * NJ];
#pragma unroll
                    for (int x = 0; x < NJ; ++x)
#pragma unroll
                        for (int i = 0; i < 16; i += 2) {
                            unsigned first, left_over;
                            two_parts(T{}, (f32x2){s[x][i], s[x][i + 1]}, first, left_over);
                            p[2 * x + i / 8][i % 8 / 2] = first;
                            rest[2 * x + i / 8][i % 8 / 2] = left_over;
                        }
                    // lane l gets, for channel l % 32, the four keys of its half: 16 lanes hold four rows of 16 channels, read transposed
                    const T* vb = &Vs[(32 * b0 + 4 * half + (col & 15) / 4) * VLD + 16 * (col >> 4) + 4 * (col & 3)];
#pragma unroll
                    for (int x = 0; x < 2 * NJ; ++x) {                    // both parts of all channels in turn: part by part 93 us (documents)
                        typedef __attribute__((address_space(3))) s16x4 lds4;
                        s16x8 keys[EB];
#pragma unroll
                        for (int eb = 0; eb < EB; ++eb) {
                            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)&vb[16 * x * VLD + eb * 32]);
                            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)&vb[(16 * x + 8) * VLD + eb * 32]);
                            keys[eb] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                        }
#pragma unroll
                        for (int eb = 0; eb < EB; ++eb) o[eb] = mfma16(T{}, keys[eb], __builtin_bit_cast(s16x8, p[x]), o[eb]);
#pragma unroll
                        for (int eb = 0; eb < EB; ++eb) o[eb] = mfma16(T{}, keys[eb], __builtin_bit_cast(s16x8, rest[x]), o[eb]);
                    }
                }
                if (bad)                                                  // what an odd value does, to those that see it
#pragma unroll
                    for (int x = 0; x < NJ; ++x) {
                        const unsigned see = other_half_or(seen[x] << (4 * half));
#pragma unroll
                        for (int eb = 0; eb < EB; ++eb)
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                const int e = eb * 32 + 8 * (i / 4) + 4 * half + i % 4;
                                const bool pos = infs[buf][0][b0 + x][e] & see, neg = infs[buf][1][b0 + x][e] & see;
                                if (pos || neg) o[eb][i] += pos && neg ? __builtin_nanf("") : pos ? INFINITY : -INFINITY;
                            }
                    }
            }
        }
        if (tile >= 0) put(tile, buf ^ 1, turn);                      // last read a turn ago, behind the barrier
        __syncthreads();
    }

    l = other_half_sum(l);
    if (qi >= a.Tq) return;
    // four neighbouring rows of O^T at a time: their channel, and how many of them the chunk before has stored
    auto each_four = [&](auto store) {
#pragma unroll
        for (int eb = 0; eb < EB; ++eb)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int e = eb * 32 + 8 * g + 4 * half, chunk = e / CV * CV;        // O^T's rows lie as the chunks of V do
                if (chunk >= a.E) continue;
                const int shift = max(0, chunk - (a.E - CV)), from = min(4, max(0, shift - (e - chunk)));
                float v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = o[eb][4 * g + i];
                store(e - shift, from, v);
            }
    };
    if (splits == 1) {
        const float r = lim > 0 && l != 0.f ? 1.f / l : 0.f;
        each_four([&](int e, int from, float (&v)[4]) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = lim > 0 && l != 0.f ? v[i] * r : 0.f;
            put_four<T>(out + (long)qi * a.o_t + e, from, v);
        });
    } else {
        float* ws = (float*)((char*)a.workspace);
        const long rows = (long)a.N * a.Tq * a.H, at = (((long)n * a.Tq + qi) * a.H + h) * splits + split;
        const bool any = lim > 0;
        each_four([&](int e, int from, float (&v)[4]) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = any ? v[i] : 0.f;
            put_four<float>(ws + at * a.E + e, from, v);
        });
        if (half == 0) {
            ws[rows * splits * a.E + at * 2] = any ? m : -INFINITY;
            ws[rows * splits * a.E + at * 2 + 1] = any ? l : 0.f;
        }
    }
}

template <class T, int EP, int NW>
int launch(const krk_attention_args& a, const AttnTiles& g, void* scratch, hipStream_t s) {
    const int qblocks = (a.Tq + NW * 32 - 1) / (NW * 32), tiles = (a.Tk + g.keys - 1) / g.keys;
    const int2* ranges = nullptr;
    if (a.documents) {
        if (seq_grid_too_large((long)a.N * tiles, 64)) return -4;
        int2* r = (int2*)scratch;
        ranges = r;
        hipLaunchKernelGGL(attn_ranges_kernel, dim3((unsigned)(((long)a.N * tiles + 3) / 4)), dim3(256), 0, s, a, r, tiles, g.keys);
    }
    const long groups = (long)a.N * a.Hk;
    const int cut = groups % 8 == 0 ? 1 : groups % 4 == 0 ? 2 : groups % 2 == 0 ? 4 : 8;
    // only causal rows differ in length by their place; elsewhere one key head at a time is better for the L2 (lines: 138 against 143 us)
    const int batch = !a.causal || a.documents ? 1 : (int)max(1L, min(64L, (4L << 20) / (2L * a.Tk * a.E * (long)sizeof(T) / cut + 1)));
    const long blocks = groups * cut * ((qblocks * (long)(a.H / a.Hk) + cut - 1) / cut);
    if (seq_grid_too_large(blocks, NW * 64)) return -4;
    hipLaunchKernelGGL((attn_tile_kernel<T, EP, NW>), dim3((unsigned)blocks, g.splits), dim3(NW * 64), 0, s, a, qblocks, cut, batch, g.splits, tiles, ranges);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

template <class T, int EP>
int by_waves(const krk_attention_args& a, const AttnTiles& g, void* scratch, hipStream_t s) {
    if constexpr (EP * sizeof(T) <= 256)
        if (g.rows == 64) return launch<T, EP, 2>(a, g, scratch, s);
    return launch<T, EP, 4>(a, g, scratch, s);
}

template <class T>
int by_width(const krk_attention_args& a, const AttnTiles& g, void* scratch, hipStream_t s) {
    if (a.E <= 32) return by_waves<T, 32>(a, g, scratch, s);
    if (a.E <= 64) return by_waves<T, 64>(a, g, scratch, s);
    if (a.E <= 96) return by_waves<T, 96>(a, g, scratch, s);
    if (a.E <= 128) return by_waves<T, 128>(a, g, scratch, s);
    return by_waves<T, 256>(a, g, scratch, s);
}

}  // namespace

AttnTiles krk_attn_tiles(const krk_attention_args& a) {
    AttnTiles g;
    // A block of 128 queries reads the keys half as often, but leaves more of it empty on short lines: 8 heads of 50 fp32, 65536 steps in all, rows of
    // 192 284 us with 64 and 353 with 128, 256 363 / 333, 300 470 / 518, 384 516 / 472, 1024 1268 / 1177.  Wide heads have no registers for two waves.
    const bool f32 = a.type == KRK_TYPE_F32;
    g.rows = a.Tq > 256 || a.E > (f32 ? 64 : 128) ? 128 : 64;
    g.keys = f32 || g.rows == 64 ? 32 : 64;
    const long blocks = (long)a.N * a.H * ((a.Tq + g.rows - 1) / g.rows), tiles = (a.Tk + g.keys - 1) / g.keys;
    // Few workgroups and a long axis: split it, eight tiles at least to each (64 queries of 8 heads x 64 fp32 on 2048 keys: 31 us, with four tiles at least 21,
    // with sixteen 52; 512 of 4 x 128 fp16 on 16384: 49, 48, 53).
    g.splits = (int)max(1L, min(min((512 + blocks - 1) / max(blocks, 1L), tiles / 8), 64L));
    g.range_bytes = a.documents ? (long)a.N * tiles * 8 : 0;
    return g;
}

int krk_launch_attn_tiles(const krk_attention_args& a, const AttnTiles& g, void* scratch, hipStream_t s) {
    return a.type == KRK_TYPE_F32 ? by_width<float>(a, g, scratch, s) : a.type == KRK_TYPE_BF16 ? by_width<bf16_t>(a, g, scratch, s) : by_width<f16_t>(a, g, scratch, s);
}
