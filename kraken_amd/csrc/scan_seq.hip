// Selective state space scan over sequence rows (krk_selective_scan).
//
//   h_i = exp(s_i A) h_{i-1} + s_i x_i B_i,   y_i = C_i . h_i + skip x_i   (times z sigmoid(z)),   s_i = softplus(dt_i + bias)
//
// LP lanes share a channel, SL states each, in registers for the whole row.
#include "seq.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f;

template <class T, int LP, int SL>
__global__ __launch_bounds__(256) void scan_seq_kernel(krk_scan_args a) {
    const int id = blockIdx.x * 256 + threadIdx.x;
    const int d = id / LP, part = id % LP;
    const bool live = d < a.D;
    const int dd = live ? d : 0, s0 = part * SL, g = dd / (a.D / a.G);
    float A[SL];
#pragma unroll
    for (int j = 0; j < SL; ++j) A[j] = s0 + j < a.S ? a.A[(long)dd * a.S + s0 + j] * LOG2E : 0.f;
    const float bias = a.dt_bias ? a.dt_bias[dd] : 0.f, skip = a.skip ? a.skip[dd] : 0.f;
    for (int n = blockIdx.y; n < a.N; n += gridDim.y) {
        const int len = seq_len(a.lens, n, a.T);
        float h[SL];
#pragma unroll
        for (int j = 0; j < SL; ++j) h[j] = a.state && s0 + j < a.S ? a.state[n * a.state_n + (long)dd * a.S + s0 + j] : 0.f;
        for (int i = 0; i < len; ++i) {
            const long t = a.reverse ? len - 1 - i : i;
            const float x = to_f(((const T*)a.x)[n * a.x_n + t * a.x_t + dd]);
            float s = to_f(((const T*)a.dt)[n * a.dt_n + t * a.dt_t + dd]) + bias;
            if (a.softplus) s = seq_softplus(s);
            const T* B = (const T*)a.B + n * a.b_n + t * a.b_t + (long)g * a.S + s0;
            const T* C = (const T*)a.C + n * a.c_n + t * a.c_t + (long)g * a.S + s0;
            const float sx = s * x;
            float y = 0.f;
#pragma unroll
            for (int j = 0; j < SL; ++j) {
                const bool in = s0 + j < a.S;
                h[j] = __builtin_fmaf(__builtin_amdgcn_exp2f(s * A[j]), h[j], sx * (in ? to_f(B[j]) : 0.f));
                y = __builtin_fmaf(in ? to_f(C[j]) : 0.f, h[j], y);
            }
#pragma unroll
            for (int m = 1; m < LP; m <<= 1) y += __shfl_xor(y, m);
            y = __builtin_fmaf(skip, x, y);
            if (a.z) y *= seq_silu(to_f(((const T*)a.z)[n * a.z_n + t * a.z_t + dd]));
            if (live && part == 0) ((T*)a.y)[n * a.y_n + t * a.y_t + dd] = from_f<T>(y);
        }
        if (live && part == 0)
            for (int t = len; t < a.T; ++t) ((T*)a.y)[n * a.y_n + (long)t * a.y_t + dd] = from_f<T>(0.f);
        if (live && a.state_out)
#pragma unroll
            for (int j = 0; j < SL; ++j)
                if (s0 + j < a.S) a.state_out[n * a.out_n + (long)dd * a.S + s0 + j] = h[j];
    }
}

template <class T, int LP, int SL>
int launch(const krk_scan_args& a, hipStream_t s) {
    const long blocks = ((long)a.D * LP + 255) / 256;
    if ((long)a.D * LP > 0x7fffff00L) return -4;
    hipLaunchKernelGGL((scan_seq_kernel<T, LP, SL>), dim3((unsigned)blocks, (unsigned)min(a.N, 65535)), dim3(256), 0, s, a);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

template <class T>
int by_states(const krk_scan_args& a, hipStream_t s) {
    if (a.S <= 16) return launch<T, 1, 16>(a, s);
    if (a.S <= 64) return launch<T, 4, 16>(a, s);
    return launch<T, 16, 16>(a, s);
}

}  // namespace

long krk_scan_workspace(const krk_scan_args&) { return 0; }

int krk_launch_selective_scan(const krk_scan_args& a, hipStream_t s) {
    return a.type == KRK_TYPE_F32 ? by_states<float>(a, s) : a.type == KRK_TYPE_BF16 ? by_states<bf16_t>(a, s) : by_states<f16_t>(a, s);
}
