// Attention over sequence rows (krk_attention): tanh-capped scores, distance bias, document / prefix / causal / length masks, shared key heads.
//
//   s_j = scale q.k_j;  s_j = cap tanh(s_j / cap);  s_j -= slope |p - j|;  out = sum_j 2^(s'_j - m) v_j / sum_j 2^(s'_j - m),  s' = s log2 e
//
// Rows kernel: one query position of R heads that share a key head.  LE lanes share a key (16 bytes of it each), so a wave reads 64 / LE keys
// at once; every group of lanes keeps its own running maximum, sum and output and they are joined at the end.  Keys and values are read
// once per R heads: with one query position per row that is the memory bound.  A long axis is split over workgroups and joined by a second
// launch where there are few rows.  16 ragged caches of up to 8192 x 8 x 128 bf16, 32 query heads: 91 + 5 us for 355 MB = 3.7 TB/s (237 us before
// the next keys were requested ahead and the sums over lanes left LDS); R = 8 heads with two keys in flight instead of four: 289 against 406 us
// (64 x 4096, 64 heads on 8), for which four do not leave the registers.
#include "attn_seq.h"

namespace {

template <int CTRL> __device__ __forceinline__ float dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
// the sum over LE neighbouring lanes, in all of them: exchanges inside the vector registers (quads, half rows, rows, pairs of rows, halves)
template <int LE> __device__ __forceinline__ float group_sum(float v) {
    v += dpp<0xB1>(v);                                             // quad_perm 1 0 3 2
    v += dpp<0x4E>(v);                                             // quad_perm 2 3 0 1
    v += dpp<0x141>(v);                                            // row_half_mirror
    if constexpr (LE >= 16) v += dpp<0x140>(v);                    // row_mirror
    if constexpr (LE >= 32) {
        const unsigned u = __builtin_bit_cast(unsigned, v);
        const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
        v = __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
    }
    if constexpr (LE >= 64) {
        const unsigned u = __builtin_bit_cast(unsigned, v);
        const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
        v = __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
    }
    return v;
}

template <class T, int R, int LE>
__global__ __launch_bounds__(256, R == 8 ? 2 : sizeof(T) == 2 ? 3 : 1) void attn_rows_kernel(krk_attention_args a, int blocks_h, int splits, int span) {
    constexpr int V = VecOf<T>::V, KPW = 64 / LE, UK = R == 8 ? 2 : 4;
    const int rep = a.H / a.Hk;
    long item = blockIdx.x;
    const int rb = item % blocks_h; item /= blocks_h;
    const int hk = item % a.Hk; item /= a.Hk;
    const int i = item % a.Tq, n = item / a.Tq;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, grp = lane / LE, e0 = (lane % LE) * V;
    const int nv = max(0, min(V, a.E - e0));
    const int h0 = hk * rep + rb * R, nr = min(R, rep - rb * R);
    const AttnRow row = query_row(a, n, i);
    const int* docs = a.documents ? a.documents + n * a.doc_n : nullptr;
    const int doc = docs && row.limit > 0 ? docs[i] : 0;
    const float rcap = a.cap > 0.f ? 1.f / a.cap : 0.f;
    const bool fine = R == 1 && a.cap > COARSE_CAP;                // row_block has seen to it
    const float qscale = a.cap > 0.f ? a.scale : a.scale * LOG2E;

    float q[R][V], slope[R], m[R], l[R], o[R][V];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int h = h0 + (r < nr ? r : 0);
        load_vec<T, V>((const T*)a.q + n * a.q_n + i * a.q_t + h * a.q_h + e0, nv, q[r]);
#pragma unroll
        for (int v = 0; v < V; ++v) q[r][v] *= qscale, o[r][v] = 0.f;
        slope[r] = a.slopes ? a.slopes[h] * LOG2E : 0.f;
        m[r] = -INFINITY;
        l[r] = 0.f;
    }
    const T* kp = (const T*)a.k + n * a.k_n + hk * a.k_h + e0;
    const T* vp = (const T*)a.v + n * a.v_n + hk * a.v_h + e0;
    const int j0 = blockIdx.y * span, j1 = min(j0 + span, row.limit);
    typedef T Tv __attribute__((ext_vector_type(V)));
    Tv kr[UK], vr[UK];
    unsigned in = 0;                                               // which of the keys in flight are seen, a bit each
    auto fetch = [&](int jb) {                                     // nothing is loaded for a key that is not seen, whatever stands there
        in = 0;
#pragma unroll
        for (int u = 0; u < UK; ++u) {
            const int j = jb + u * KPW + grp;
            const bool see = j < j1 && (!docs || docs[j] == doc);
            kr[u] = vr[u] = (Tv)(T)0.f;
            if (!see) continue;
            in |= 1u << u;
            if (nv >= V) {
                __builtin_memcpy(&kr[u], kp + (long)j * a.k_t, sizeof(Tv));
                __builtin_memcpy(&vr[u], vp + (long)j * a.v_t, sizeof(Tv));
            } else {
#pragma unroll
                for (int v = 0; v < V; ++v)
                    if (v < nv) kr[u][v] = kp[(long)j * a.k_t + v], vr[u][v] = vp[(long)j * a.v_t + v];
            }
        }
    };
    constexpr int STEP = 4 * KPW * UK;
    int jb = j0 + wave * KPW * UK;
    if (jb < j1) fetch(jb);
    for (; jb < j1; jb += STEP) {
        Tv kc[UK], vc[UK];
        const unsigned now = in;
#pragma unroll
        for (int u = 0; u < UK; ++u) kc[u] = kr[u], vc[u] = vr[u];
        if (jb + STEP < j1) fetch(jb + STEP);                      // the next keys are in flight while these are used
        float s[UK][R];
#pragma unroll
        for (int u = 0; u < UK; ++u)
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float d = 0.f;
#pragma unroll
                for (int v = 0; v < V; ++v) d = __builtin_fmaf(q[r][v], to_f<T>(kc[u][v]), d);
                s[u][r] = group_sum<LE>(d);
            }
        if (a.cap > 0.f)
#pragma unroll
            for (int u = 0; u < UK; ++u)
#pragma unroll
                for (int r = 0; r < R; ++r) s[u][r] = (fine ? seq_cap<float>(s[u][r], a.cap, rcap) : seq_cap<T>(s[u][r], a.cap, rcap)) * LOG2E;
        if (a.slopes)
#pragma unroll
            for (int u = 0; u < UK; ++u)
#pragma unroll
                for (int r = 0; r < R; ++r) s[u][r] = __builtin_fmaf(-slope[r], fabsf((float)(row.p - (jb + u * KPW + grp))), s[u][r]);
        float top[R];
        bool move = false;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            top[r] = -INFINITY;
#pragma unroll
            for (int u = 0; u < UK; ++u) {
                s[u][r] = (now >> u) & 1u ? s[u][r] : -INFINITY;
                top[r] = fmaxf(top[r], s[u][r]);
            }
            move = move || top[r] > m[r] + 8.f;
        }
        if (__ballot(move))                                        // as in the tile kernel: the reference point moves when a score passes it by 2^8
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float nm = fmaxf(m[r], top[r]), f = __builtin_amdgcn_exp2f(m[r] - (nm == -INFINITY ? 0.f : nm));
                m[r] = nm;
                l[r] *= f;
#pragma unroll
                for (int v = 0; v < V; ++v) o[r][v] *= f;
            }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float ref = m[r] == -INFINITY ? 0.f : m[r];
#pragma unroll
            for (int u = 0; u < UK; ++u) {
                s[u][r] = __builtin_amdgcn_exp2f(s[u][r] - ref);
                l[r] += s[u][r];
            }
        }
#pragma unroll
        for (int u = 0; u < UK; ++u)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float x = to_f<T>(vc[u][v]);
#pragma unroll
                for (int r = 0; r < R; ++r) o[r][v] = __builtin_fmaf(s[u][r], x, o[r][v]);
            }
    }
    // join the groups of a wave, then the four waves
    __shared__ float wm[4][R], wl[4][R], wo[4][R][LE * V];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        float top = m[r];
#pragma unroll
        for (int x = LE; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x));
        const float f = __builtin_amdgcn_exp2f(m[r] - (top == -INFINITY ? 0.f : top));   // 0 for a group that saw nothing
        float sum = l[r] * f;
#pragma unroll
        for (int x = LE; x < 64; x <<= 1) sum += __shfl_xor(sum, x);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float t = o[r][v] * f;
#pragma unroll
            for (int x = LE; x < 64; x <<= 1) t += __shfl_xor(t, x);
            if (grp == 0) wo[wave][r][e0 + v] = t;
        }
        if (lane == 0) wm[wave][r] = top, wl[wave][r] = sum;
    }
    __syncthreads();
    const long rows = (long)a.N * a.Tq * a.H;
    for (int x = threadIdx.x; x < nr * a.E; x += 256) {
        const int r = x / a.E, e = x - r * a.E;
        float top = -INFINITY, sum = 0.f, t = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) top = fmaxf(top, wm[w][r]);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = __builtin_amdgcn_exp2f(wm[w][r] - (top == -INFINITY ? 0.f : top));
            sum = __builtin_fmaf(wl[w][r], f, sum);
            t = __builtin_fmaf(wo[w][r][e], f, t);
        }
        if (splits == 1) {
            ((T*)a.out)[n * a.o_n + i * a.o_t + (h0 + r) * a.o_h + e] = from_f<T>(sum == 0.f ? 0.f : t / sum);
        } else {
            float* ws = (float*)a.workspace;
            const long at = (((long)n * a.Tq + i) * a.H + h0 + r) * splits + blockIdx.y;
            ws[at * a.E + e] = t;
            if (e == 0) {
                float* ml = ws + rows * splits * a.E;
                ml[at * 2] = top;
                ml[at * 2 + 1] = sum;
            }
        }
    }
}

constexpr int MAX_SPLITS = 64;

// joins the splits of one row: a wave per row, lanes along the splits for their weights, along E for the sums
template <class T>
__global__ __launch_bounds__(256) void attn_join_kernel(krk_attention_args a, int splits, long rows) {
    const long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= rows) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __shared__ float weight[4][MAX_SPLITS];
    const float* ws = (const float*)a.workspace;
    const float2* ml = (const float2*)(ws + rows * splits * a.E) + row * splits;
    float top = -INFINITY, sum = 0.f;
    for (int x = lane; x < splits; x += 64) top = fmaxf(top, ml[x].x);
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x));
    const float ref = top == -INFINITY ? 0.f : top;
    for (int x = lane; x < splits; x += 64) {
        const float w = __builtin_amdgcn_exp2f(ml[x].x - ref);
        weight[wave][x] = w;
        sum = __builtin_fmaf(ml[x].y, w, sum);
    }
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) sum += __shfl_xor(sum, x);
    __builtin_amdgcn_wave_barrier();                               // a wave reads what it wrote itself
    const int h = row % a.H;
    const long it = row / a.H;
    const int i = it % a.Tq;
    const long n = it / a.Tq;
    for (int e = lane; e < a.E; e += 64) {
        float t = 0.f;
#pragma unroll 8
        for (int x = 0; x < splits; ++x) t = __builtin_fmaf(ws[(row * splits + x) * a.E + e], weight[wave][x], t);
        ((T*)a.out)[n * a.o_n + i * a.o_t + h * a.o_h + e] = from_f<T>(sum == 0.f ? 0.f : t / sum);
    }
}

// heads of a workgroup; one where 16-bit types need the finer cap, which does not leave the registers of several (R = 4: 95 -> 169 us with it)
int row_block(const krk_attention_args& a) {
    const int rep = a.H / a.Hk;
    if (a.type != KRK_TYPE_F32 && a.cap > COARSE_CAP) return 1;
    return rep >= 8 ? 8 : rep >= 4 ? 4 : rep >= 2 ? 2 : 1;
}

// workgroups along the key axis: enough for eight per CU where there are few rows, 256 keys at least for each
int split_count(const krk_attention_args& a) {
    const int rep = a.H / a.Hk, R = row_block(a);
    const long items = (long)a.N * a.Tq * a.Hk * ((rep + R - 1) / R);
    if (items <= 0 || a.Tk <= 0) return 1;
    long want = (2048 + items - 1) / items, most = (a.Tk + 255) / 256;
    return (int)max(1L, min(min(want, most), (long)MAX_SPLITS));
}

template <class T, int R, int LE>
int launch_rows(const krk_attention_args& a, hipStream_t s) {
    const int rep = a.H / a.Hk, blocks_h = (rep + R - 1) / R, splits = split_count(a);
    int span = (a.Tk + splits - 1) / splits;
    const long items = (long)a.N * a.Tq * a.Hk * blocks_h, rows = (long)a.N * a.Tq * a.H;
    if (seq_grid_too_large(items, 256)) return -4;
    hipLaunchKernelGGL((attn_rows_kernel<T, R, LE>), dim3((unsigned)items, splits), dim3(256), 0, s, a, blocks_h, splits, span);
    if (splits > 1) hipLaunchKernelGGL((attn_join_kernel<T>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, a, splits, rows);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

template <class T, int R>
int by_lanes(const krk_attention_args& a, hipStream_t s) {
    const int need = (a.E + VecOf<T>::V - 1) / VecOf<T>::V;
    if (need <= 8) return launch_rows<T, R, 8>(a, s);
    if (need <= 16) return launch_rows<T, R, 16>(a, s);
    if (need <= 32) return launch_rows<T, R, 32>(a, s);
    if constexpr (sizeof(T) == 4) return launch_rows<T, R, 64>(a, s);
    return -4;
}

template <class T>
int by_rows(const krk_attention_args& a, hipStream_t s) {
    switch (row_block(a)) {
        case 8: return by_lanes<T, 8>(a, s);
        case 4: return by_lanes<T, 4>(a, s);
        case 2: return by_lanes<T, 2>(a, s);
        default: return by_lanes<T, 1>(a, s);
    }
}

// One or two query positions read the keys as often as they are rows; more of them go to the tile kernel, which reads them once per block and query head.
// Rows here and tiles, us: 16 caches of 8192, 32 heads on 8 x 128 bf16, two queries 160 / 389, three 212 / 390, six 378 / 389, eight 494 / 391;
// 16 x 2048, 16 heads of 64 fp16 with keys of their own, two 32 / 44, four 42 / 45, six 56 / 45; 64 lines of 150, 8 x 50 fp32, two 14 / 21, three 22 / 22,
// four 24 / 22.  Heads of less than 16 bytes stay here: the tile kernel's loads are 16 bytes within a row.
bool by_tiles(const krk_attention_args& a) { return a.Tq > 2 && a.E * (a.type == KRK_TYPE_F32 ? 4 : 2) >= 16; }

long part_bytes(const krk_attention_args& a, int splits) {
    return splits == 1 ? 0 : ((long)a.N * a.Tq * a.H * splits * (a.E + 2) * (long)sizeof(float) + 15) / 16 * 16;
}

int launch_tiles(const krk_attention_args& a, hipStream_t s) {
    const AttnTiles g = krk_attn_tiles(a);
    const long rows = (long)a.N * a.Tq * a.H;
    if (int rc = krk_launch_attn_tiles(a, g, (char*)a.workspace + part_bytes(a, g.splits), s)) return rc;
    if (g.splits > 1) {
        const dim3 grid((unsigned)((rows + 3) / 4));
        if (a.type == KRK_TYPE_F32) hipLaunchKernelGGL((attn_join_kernel<float>), grid, dim3(256), 0, s, a, g.splits, rows);
        else if (a.type == KRK_TYPE_BF16) hipLaunchKernelGGL((attn_join_kernel<bf16_t>), grid, dim3(256), 0, s, a, g.splits, rows);
        else hipLaunchKernelGGL((attn_join_kernel<f16_t>), grid, dim3(256), 0, s, a, g.splits, rows);
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace

long krk_attn_workspace(const krk_attention_args& a) {
    if (!by_tiles(a)) return part_bytes(a, split_count(a));
    const AttnTiles g = krk_attn_tiles(a);
    return part_bytes(a, g.splits) + g.range_bytes;
}

int krk_launch_attention(const krk_attention_args& a, hipStream_t s) {
    if (by_tiles(a)) return launch_tiles(a, s);
    return a.type == KRK_TYPE_F32 ? by_rows<float>(a, s) : a.type == KRK_TYPE_BF16 ? by_rows<bf16_t>(a, s) : by_rows<f16_t>(a, s);
}
