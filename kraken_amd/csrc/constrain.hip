// Penalties, biases and masks on scores in front of a decoder (krk_constrain_logits).
//
// One read and one write of the scores: bound by memory (256 x 150 x 256 fp32, alphabets and a bias: 14.5 us, 5.4 TB/s, part of it from the last-level
// cache; 64 x 128000 bf16 with 1024 labels of history: 12 us, of which half is the one round of workgroups' own latency).  A workgroup owns a range of CH classes of one line and a range of its steps; it
// counts the line's history into LDS first (integers: the order of the additions does not matter), so a line's history is read once
// per class range and no count ever goes through memory.  Every operation is rounded on its own (no contraction): scores that tie before
// tie in the plain order of operations too.
#include "seq.h"

namespace {

constexpr int CH = 4096;      // classes of a workgroup: 16 KB of counters, eight workgroups (all that the waves allow) in 128 of a CU's 160 KB

// MANY: more lines than a grid has; a loop over lines in every call costs a quarter of its speed (12 -> 15.7 us)
template <class T, class I, bool MANY>
__global__ __launch_bounds__(256) void constrain_kernel(krk_constrain_args a, int tx_bits, int rows) {
#pragma clang fp contract(off)
    constexpr int V = VecOf<T>::V;
    __shared__ int count[CH];
    const int c0 = blockIdx.x * CH, c1 = min(c0 + CH, a.C);
    const bool hist = a.history != nullptr;
    int n = blockIdx.z;
    do {
        float rep = 1.f, pres = 0.f, freq = 0.f;
        if (hist) {
            rep = a.repetition ? a.repetition[n] : a.all_repetition;
            pres = a.presence ? a.presence[n] : a.all_presence;
            freq = a.frequency ? a.frequency[n] : a.all_frequency;
            for (int i = threadIdx.x; i < c1 - c0; i += 256) count[i] = 0;
            __syncthreads();
            const int L = seq_len(a.hist_lens, n, a.L);
            const I* h = (const I*)a.history + n * a.hist_n;
            for (int i = threadIdx.x; i < L; i += 256) {
                const I c = h[i];
                if (c >= c0 && c < c1) atomicAdd(&count[(int)(c - c0)], 1);
            }
            __syncthreads();
        }
        const int tx = threadIdx.x & ((1 << tx_bits) - 1), ty = threadIdx.x >> tx_bits;
        const int t1 = min((int)(blockIdx.y + 1) * rows, a.T);
        for (int t = blockIdx.y * rows + ty; t < t1; t += 256 >> tx_bits) {
            const T* in = (const T*)a.logits + n * a.l_n + t * a.l_t;
            T* out = (T*)a.out + n * a.o_n + t * a.o_t;
            const unsigned* mask = a.mask ? a.mask + n * a.mask_n + t * a.mask_t : nullptr;
            for (int c = c0 + tx * V; c < c1; c += V << tx_bits) {
                const int nv = min(V, c1 - c);
                float v[V], b[V];
                load_vec<T, V>(in + c, nv, v);
                const unsigned bits = mask ? mask[c >> 5] >> (c & 31) : ~0u;
                if (a.bias) load_vec<float, V>(a.bias + n * a.bias_n + c, nv, b);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    if (hist) {
                        const int k = j < nv ? count[c - c0 + j] : 0;
                        if (k > 0) {
                            v[j] = v[j] > 0.f ? v[j] / rep : v[j] * rep;
                            const float f = freq * (float)k;
                            v[j] = v[j] - f;
                            v[j] = v[j] - pres;
                        }
                    }
                    if (a.bias) v[j] = v[j] + b[j];
                    if (!((bits >> j) & 1u)) v[j] = -INFINITY;
                }
                store_vec<T, V>(out + c, nv, v);
            }
        }
        if constexpr (MANY) __syncthreads();      // the counters are the next line's
    } while (MANY && (n += gridDim.z) < a.N);
}

template <class T, class I>
int launch(const krk_constrain_args& a, hipStream_t s) {
    constexpr int V = VecOf<T>::V;
    const int chunks = (a.C + CH - 1) / CH, groups = (min(a.C, CH) + V - 1) / V;
    int bits = 0;
    while (bits < 8 && (1 << bits) < groups) ++bits;
    // steps of a workgroup: enough that counting the history is paid for, up to sixteen workgroups per CU
    int rows = 256 >> bits;
    while ((long)a.N * chunks * ((a.T + rows - 1) / rows) > 4096 && rows < a.T) rows *= 2;
    const int parts = (a.T + rows - 1) / rows;
    if (parts > 65535) return -4;
    const dim3 grid(chunks, parts, min(a.N, 65535));
    if (a.N > 65535) hipLaunchKernelGGL((constrain_kernel<T, I, true>), grid, dim3(256), 0, s, a, bits, rows);
    else hipLaunchKernelGGL((constrain_kernel<T, I, false>), grid, dim3(256), 0, s, a, bits, rows);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

template <class T>
int by_labels(const krk_constrain_args& a, hipStream_t s) {
    return a.hist64 ? launch<T, long>(a, s) : launch<T, int>(a, s);
}

}  // namespace

int krk_launch_constrain(const krk_constrain_args& a, hipStream_t s) {
    return a.type == KRK_TYPE_F32 ? by_labels<float>(a, s) : a.type == KRK_TYPE_BF16 ? by_labels<bf16_t>(a, s) : by_labels<f16_t>(a, s);
}
