// Short depthwise causal convolution over sequence rows, forward and reversed, with carried state (krk_causal_conv).
//
//   p_i = bias + sum_k w[d][k] x_{i-(K-1)+k}[d],   y = p or p sigmoid(p),   i in processing order over the valid steps of a row
//
// 2 K flops per element read and written: bound by memory.  A thread owns one 16-byte channel group and walks a run of steps with the
// last K-1 inputs in registers, so every input is read once (plus K-1 of them again per run); the next U steps' loads are in flight while U
// steps are computed.  Lanes of a wave lie along the channels, so a wave's access is contiguous.
// 2 x 16384 x 4096 bf16, K = 4: 110 us = 4.9 TB/s, the rate of a copy (without the loads in flight 137 us; U = 8: the same, and fp32 lines a fifth
// slower); 256 ragged lines of 150 x 400 fp32: 23 us.  One step of 8 x 800 channels: 6 us, the latency of its two dependent loads.
#include "seq.h"

namespace {

constexpr int U = 4;          // steps whose loads are in flight together

template <class T, int K>
__global__ __launch_bounds__(256) void conv_seq_kernel(krk_conv_args a, int groups, int runs, int steps) {
    constexpr int V = VecOf<T>::V, W = K - 1;
    typedef T Raw __attribute__((ext_vector_type(V)));
    const int id = blockIdx.x * 256 + threadIdx.x;
    const int run = id / groups, d0 = (id - run * groups) * V;
    if (run >= runs) return;
    const int nv = min(V, a.D - d0);
    // the kernels of V neighbouring channels lie behind one another: K vectors, put in order in the registers
    float w[K][V], b[V], flat[K * V];
#pragma unroll
    for (int k = 0; k < K; ++k)
        load_vec<T, V>((const T*)a.weight + (long)d0 * K + k * V, nv * K - k * V, *reinterpret_cast<float (*)[V]>(&flat[k * V]));
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
        for (int k = 0; k < K; ++k) w[k][j] = flat[j * K + k];
    if (a.bias) load_vec<T, V>((const T*)a.bias + d0, nv, b);
    else
#pragma unroll
        for (int j = 0; j < V; ++j) b[j] = 0.f;
    for (int n = blockIdx.y; n < a.N; n += gridDim.y) {
        const int len = seq_len(a.lens, n, a.T);
        const T* x = (const T*)a.x + n * a.x_n + d0;
        T* y = (T*)a.y + n * a.y_n + d0;
        const T* st = a.state ? (const T*)a.state + n * a.state_n + d0 : nullptr;
        // input of processing step i (i >= -W): the line, the carried state, or nothing
        auto input = [&](int i, float (&v)[V]) {
            if (i >= 0) load_vec<T, V>(x + (long)(a.reverse ? len - 1 - i : i) * a.x_t, nv, v);
            else if (st) load_vec<T, V>(st + (long)(W + i) * a.state_k, nv, v);
            else
#pragma unroll
                for (int j = 0; j < V; ++j) v[j] = 0.f;
        };
        const int i0 = run * steps, i1 = min(i0 + steps, a.T), end = min(i1, len);
        Raw next[U];
        // the next U steps, behind the end the last one again: loads without a condition, in flight while the steps before them are computed
        auto fetch = [&](int i) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int k = min(i + u, end - 1);
                next[u] = load_raw<T, V>(x + (long)(a.reverse ? len - 1 - k : k) * a.x_t, nv);
            }
        };
        if (i0 < end) fetch(i0);
        float win[W + U][V];
#pragma unroll
        for (int k = 0; k < W; ++k)
            if (i0 < len) input(i0 - W + k, win[k]);
        if (run == 0 && a.state_out) {           // every row is read before one is written: state_out may be state when T == 1
            float last[W ? W : 1][V];
#pragma unroll
            for (int k = 0; k < W; ++k) input(len - W + k, last[k]);
#pragma unroll
            for (int k = 0; k < W; ++k) store_vec<T, V>((T*)a.state_out + n * a.out_n + k * a.out_k + d0, nv, last[k]);
        }
        for (int i = i0; i < end; i += U) {
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int j = 0; j < V; ++j) win[W + u][j] = to_f<T>(next[u][j]);
            if (i + U < end) fetch(i + U);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float p[V];
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    float s = b[j];
#pragma unroll
                    for (int k = 0; k < K; ++k) s = __builtin_fmaf(w[k][j], win[u + k][j], s);
                    p[j] = a.silu ? seq_silu(s) : s;
                }
                if (i + u < end) store_vec<T, V>(y + (long)(a.reverse ? len - 1 - (i + u) : i + u) * a.y_t, nv, p);
            }
#pragma unroll
            for (int k = 0; k < W; ++k)
#pragma unroll
                for (int j = 0; j < V; ++j) win[k][j] = win[k + U][j];
        }
        const float zero[V] = {};
        for (int t = max(i0, len); t < i1; ++t) store_vec<T, V>(y + (long)t * a.y_t, nv, zero);   // padding
    }
}

template <class T, int K>
int launch(const krk_conv_args& a, hipStream_t s) {
    constexpr int V = VecOf<T>::V;
    const int groups = (a.D + V - 1) / V;
    // 32 steps per thread read 3 of 35 rows twice (K = 4); shorter runs where that would leave fewer than eight waves per SIMD
    int steps = 32;
    while (steps > U && (double)a.N * groups * ((a.T + steps - 1) / steps) < 8.0 * 64 * 1024) steps /= 2;
    const int runs = a.T > 0 ? (a.T + steps - 1) / steps : 1;     // no steps at all: one run, for the state
    const long blocks = ((long)groups * runs + 255) / 256;
    if ((long)groups * runs > 0x7fffff00L) return -4;
    hipLaunchKernelGGL((conv_seq_kernel<T, K>), dim3((unsigned)blocks, (unsigned)min(a.N, 65535)), dim3(256), 0, s, a, groups, runs, steps);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

template <class T>
int by_width(const krk_conv_args& a, hipStream_t s) {
    switch (a.K) {
        case 1: return launch<T, 1>(a, s);
        case 2: return launch<T, 2>(a, s);
        case 3: return launch<T, 3>(a, s);
        case 4: return launch<T, 4>(a, s);
        case 5: return launch<T, 5>(a, s);
        case 6: return launch<T, 6>(a, s);
        case 7: return launch<T, 7>(a, s);
        default: return launch<T, 8>(a, s);
    }
}

}  // namespace

int krk_launch_causal_conv(const krk_conv_args& a, hipStream_t s) {
    return a.type == KRK_TYPE_F32 ? by_width<float>(a, s) : a.type == KRK_TYPE_BF16 ? by_width<bf16_t>(a, s) : by_width<f16_t>(a, s);
}
