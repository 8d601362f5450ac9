// Selective state space scan over sequence rows (krk_selective_scan).
//
//   h_i = exp(s_i A) h_{i-1} + s_i x_i B_i,   y_i = C_i . h_i + skip x_i   (times z sigmoid(z)),   s_i = softplus(dt_i + bias)
//
// Per channel, step and state: an exponential, two products and two multiply-adds; per channel and step 6 to 16 bytes.  At 16 states the vector
// units bound it, not memory.  A lane owns a channel (LP lanes share one with more than SL states) and keeps its states and rates in
// registers for a whole row; lanes lie along the channels, so every access of a step is contiguous.  B and C, the same for all channels of a
// group, go through LDS as fp32, U steps at a time; the next U steps' inputs are in flight while U steps are computed.
// Of a step's 132 vector instructions 80 are the states' (16 of them exponentials, at half rate), so 590 cycles a wave: 256 ragged lines of
// 150 x 400 x 16 fp32 would take 40 us on evenly filled SIMDs and take 87: eight waves a row, 2048 of different lengths on 1024 SIMDs, and as a block
// holds channels of one row only, the last of the eight has none and computes all the same; blocks of 64 or 128 lanes instead of 256 make no difference.
//
// Few rows do not fill the chip with channels alone: then the time axis is cut into chunks.  One pass gives every chunk's end state from a
// zero start and the sum of its steps -- the decay over a chunk is exp(A sum) --, a second joins the chunks in order, and the main pass starts every
// chunk from its true state (1 x 8191 x 2048 x 16 bf16: 71 + 9 + 95 us; in one pass 3.6 ms).  That costs four fifths of the work again, so it is done only where a quarter of the SIMDs would idle.
#include "seq.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int U = 8;

struct ScanCut {
    int chunks, len;       // time chunks and steps of each
    float* part;           // [N][chunks - 1][D][S]: end states from a zero start, after the join the states in front of the next chunk
    float* sums;           // [N][chunks - 1][D]: sums of the steps
};

// A rate of -inf (a state that forgets at once) as the lowest number: a step of width zero, as the kernels take for one behind the end, then leaves the
// state as it is, where 0 times -inf would be no number.  Steps not computed instead, one by one at the end: lines 87 -> 97 us, long row 160 -> 167.
__device__ __forceinline__ float finite_rate(float a) { return fabsf(a) == INFINITY ? __builtin_copysignf(__FLT_MAX__, a) : a; }

// SL states of a lane, four at a time; zeros where there are none
template <int SL> __device__ __forceinline__ void load_states(const float* p, int n, float (&v)[SL]) {
#pragma unroll
    for (int j = 0; j < SL; j += 4) load_vec<float, 4>(p + j, n - j, *reinterpret_cast<float (*)[4]>(&v[j]));
}
template <int SL> __device__ __forceinline__ void store_states(float* p, int n, const float (&v)[SL]) {
#pragma unroll
    for (int j = 0; j < SL; j += 4) store_vec<float, 4>(p + j, n - j, *reinterpret_cast<const float (*)[4]>(&v[j]));
}

template <class T, int LP, int SL, bool MAIN>
__global__ __launch_bounds__(256) void scan_seq_kernel(krk_scan_args a, ScanCut cut) {
    constexpr int SP = LP * SL, NBC = (U * SP + 255) / 256;      // values of B (and of C) that a thread stages per U steps
    __shared__ __attribute__((aligned(16))) float Bs[2][U][SP], Cs[MAIN ? 2 : 1][MAIN ? U : 1][SP];
    const int per = a.D / a.G, per_block = 256 / LP, blocks_g = (per + per_block - 1) / per_block;
    const int g = blockIdx.x / blocks_g, dg = (blockIdx.x - g * blocks_g) * per_block + threadIdx.x / LP, part = threadIdx.x % LP;
    const bool live = dg < per;
    const unsigned d = g * per + (live ? dg : 0);
    const int s0 = part * SL, chunk = blockIdx.y;
    float A[SL];
    load_states(a.A + (long)d * a.S + s0, a.S - s0, A);
#pragma unroll
    for (int j = 0; j < SL; ++j) A[j] = finite_rate(A[j] * LOG2E);
    const float bias = a.dt_bias ? a.dt_bias[d] : 0.f, skip = a.skip ? a.skip[d] : 0.f;
    for (int n = blockIdx.z; n < a.N; n += gridDim.z) {
        const int len = __builtin_amdgcn_readfirstlane(seq_len(a.lens, n, a.T));
        const int i0 = chunk * cut.len, i1 = min(i0 + cut.len, len);
        const T *xp = (const T*)a.x + n * a.x_n, *dp = (const T*)a.dt + n * a.dt_n, *zp = a.z ? (const T*)a.z + n * a.z_n : nullptr;
        const T *bp = (const T*)a.B + n * a.b_n + (long)g * a.S, *cp = (const T*)a.C + n * a.c_n + (long)g * a.S;
        T* yp = (T*)a.y + n * a.y_n;
        float h[SL], sum = 0.f;
#pragma unroll
        for (int j = 0; j < SL; ++j) h[j] = 0.f;
        if (MAIN && chunk > 0) load_states(cut.part + (((long)n * (cut.chunks - 1) + chunk - 1) * a.D + d) * a.S + s0, a.S - s0, h);
        else if (MAIN && a.state) load_states(a.state + n * a.state_n + (long)d * a.S + s0, a.S - s0, h);
        T xr[U], dr[U], zr[U], br[NBC], cr[NBC];
        auto step = [&](int i) -> long { i = min(i, i1 - 1); return a.reverse ? len - 1 - i : i; };
        auto fetch = [&](int i) {                                 // steps behind the end repeat the last one; they are not computed
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const long t = step(i + u);
                xr[u] = (xp + t * a.x_t)[d];
                dr[u] = (dp + t * a.dt_t)[d];
                if (MAIN && zp) zr[u] = (zp + t * a.z_t)[d];
            }
#pragma unroll
            for (int k = 0; k < NBC; ++k) {
                const int id = threadIdx.x + 256 * k, u = min(id / SP, U - 1), j = min(id % SP, a.S - 1);
                const long t = step(i + u);
                br[k] = bp[t * a.b_t + j];
                if (MAIN) cr[k] = cp[t * a.c_t + j];
            }
        };
        auto put = [&](int i, int buf) {                          // states that do not exist and steps behind the end get B = C = 0
#pragma unroll
            for (int k = 0; k < NBC; ++k) {
                const int id = threadIdx.x + 256 * k;
                const bool is = id % SP < a.S && i + id / SP < i1;
                if (U * SP % 256 == 0 || id < U * SP) {
                    (&Bs[buf][0][0])[id] = is ? to_f(br[k]) : 0.f;
                    if (MAIN) (&Cs[buf][0][0])[id] = is ? to_f(cr[k]) : 0.f;
                }
            }
        };
        if (i0 < i1) {
            fetch(i0);
            put(i0, 0);
        }
        __syncthreads();
        int buf = 0;
        for (int i = i0; i < i1; i += U, buf ^= 1) {
            // One stretch of code for U steps, so that their LDS reads and exponentials overlap: a step behind the end has s = x = B = C = 0,
            // which leaves the states as they are.
            float x[U], w[U], y[U];
            T zc[U];
            const int left = i1 - i;
#pragma unroll
            for (int u = 0; u < U; ++u) x[u] = to_f(xr[u]), w[u] = to_f(dr[u]) + bias, zc[u] = zr[u];
            if (left > U) fetch(i + U);
            if (a.softplus)
#pragma unroll
                for (int u = 0; u < U; ++u) w[u] = seq_softplus(w[u]);
            if (left < U)
#pragma unroll
                for (int u = 0; u < U; ++u) x[u] = u < left ? x[u] : 0.f, w[u] = u < left ? w[u] : 0.f;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float wx = w[u] * x[u];
                float y0 = 0.f, y1 = 0.f;
                if (!MAIN) sum += w[u];
#pragma unroll
                for (int j = 0; j < SL; j += 4) {
                    const f32x4 b = *(const f32x4*)&Bs[buf][u][s0 + j];
                    f32x4 c = {0.f, 0.f, 0.f, 0.f};
                    if (MAIN) c = *(const f32x4*)&Cs[MAIN ? buf : 0][MAIN ? u : 0][s0 + j];
#pragma unroll
                    for (int v = 0; v < 4; ++v) {
                        h[j + v] = __builtin_fmaf(__builtin_amdgcn_exp2f(w[u] * A[j + v]), h[j + v], wx * b[v]);
                        if (MAIN) (v & 1 ? y1 : y0) = __builtin_fmaf(c[v], h[j + v], v & 1 ? y1 : y0);
                    }
                }
                if (MAIN) {
                    y[u] = y0 + y1;
#pragma unroll
                    for (int m = 1; m < LP; m <<= 1) y[u] += __shfl_xor(y[u], m);
                    y[u] = __builtin_fmaf(skip, x[u], y[u]);
                }
            }
            if (MAIN) {
                if (zp)
#pragma unroll
                    for (int u = 0; u < U; ++u) y[u] *= seq_silu(to_f(zc[u]));
                if (live && part == 0)
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (u < left) (yp + (long)(a.reverse ? len - 1 - (i + u) : i + u) * a.y_t)[d] = from_f<T>(y[u]);
            }
            if (left > U) put(i + U, buf ^ 1);
            __syncthreads();
        }
        if (!live) continue;
        if (MAIN) {
            if (part == 0)
                for (int t = max(i0, len); t < min(i0 + cut.len, a.T); ++t) (yp + (long)t * a.y_t)[d] = from_f<T>(0.f);
            if (a.state_out && chunk == max(len - 1, 0) / cut.len) store_states(a.state_out + n * a.out_n + (long)d * a.S + s0, a.S - s0, h);
        } else {
            const long at = ((long)n * (cut.chunks - 1) + chunk) * a.D + d;
            store_states(cut.part + at * a.S + s0, a.S - s0, h);
            if (part == 0) cut.sums[at] = sum;
        }
    }
}

// The states in front of every chunk: one lane per (channel, state), the chunks in order.  A chunk's factor 2^(A sum) alone may leave float32's range
// where the states do not (1e-30 under exp(6) for 20 steps, or an infinite state under a decay), so it is applied in two: a mantissa in (1/2, 1] and
// the exponent by v_ldexp, which cannot overflow or vanish unless the state itself does.
__global__ __launch_bounds__(256) void scan_join_kernel(krk_scan_args a, ScanCut cut) {
    const long id = (long)blockIdx.x * 256 + threadIdx.x, ds = (long)a.D * a.S;
    if (id >= ds) return;
    const long d = id / a.S;
    const float A = finite_rate(a.A[id] * LOG2E);
    for (int n = blockIdx.y; n < a.N; n += gridDim.y) {
        float h = a.state ? a.state[n * a.state_n + id] : 0.f;
        float* p = cut.part + (long)n * (cut.chunks - 1) * ds + id;
        const float* s = cut.sums + (long)n * (cut.chunks - 1) * a.D + d;
        constexpr int B = 16;                                     // loads in flight: the chain itself is a multiply-add a chunk
        for (int c0 = 0; c0 < cut.chunks - 1; c0 += B) {
            float e[B], q[B];
#pragma unroll
            for (int c = 0; c < B; ++c) {
                const long at = min(c0 + c, cut.chunks - 2);
                e[c] = s[at * a.D];
                q[c] = p[at * ds];
            }
#pragma unroll
            for (int c = 0; c < B; ++c)
                if (c0 + c < cut.chunks - 1) {
                    const float x = fminf(fmaxf(e[c] * A, -2000.f), 2000.f), up = ceilf(x);   // no number: q is none either
                    h = __builtin_amdgcn_ldexpf(h * __builtin_amdgcn_exp2f(x - up), (int)up) + q[c];
                    p[(c0 + c) * ds] = h;
                }
        }
    }
}

// One step of every row: four states per lane, LP lanes per channel, so that the states are read and written by whole lines; bound by them.
template <class T, int LP>
__global__ __launch_bounds__(256) void scan_step_kernel(krk_scan_args a) {
    const long id = (long)blockIdx.x * 256 + threadIdx.x;
    const int part = id % LP, s0 = part * 4, nv = min(4, a.S - s0);
    long row = id / LP;
    const bool live = row < (long)a.N * a.D;
    if (!live) row = 0;
    const int n = row / a.D, d = row - (long)n * a.D, g = d / (a.D / a.G);
    const bool on = seq_len(a.lens, n, 1) > 0;
    const float x = to_f(((const T*)a.x)[n * a.x_n + d]);
    float s = to_f(((const T*)a.dt)[n * a.dt_n + d]) + (a.dt_bias ? a.dt_bias[d] : 0.f);
    float A[4], b[4], c[4], h[4] = {0.f, 0.f, 0.f, 0.f};
    load_vec<float, 4>(a.A + (long)d * a.S + s0, nv, A);
    load_vec<T, 4>((const T*)a.B + n * a.b_n + (long)g * a.S + s0, nv, b);
    load_vec<T, 4>((const T*)a.C + n * a.c_n + (long)g * a.S + s0, nv, c);
    if (a.state) load_vec<float, 4>(a.state + n * a.state_n + (long)d * a.S + s0, nv, h);
    if (a.softplus) s = seq_softplus(s);
    float y = 0.f;
    if (on) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            h[j] = __builtin_fmaf(__builtin_amdgcn_exp2f(s * finite_rate(A[j]) * LOG2E), h[j], s * x * b[j]);
            y = __builtin_fmaf(c[j], h[j], y);
        }
    }
#pragma unroll
    for (int m = 1; m < LP; m <<= 1) y += __shfl_xor(y, m);
    if (!live) return;
    if (a.state_out) store_vec<float, 4>(a.state_out + n * a.out_n + (long)d * a.S + s0, nv, h);
    if (part) return;
    y = __builtin_fmaf(a.skip ? a.skip[d] : 0.f, x, y);
    if (a.z) y *= seq_silu(to_f(((const T*)a.z)[n * a.z_n + d]));
    ((T*)a.y)[n * a.y_n + d] = from_f<T>(on ? y : 0.f);
}

int lanes_of(int S) { return S <= 16 ? 1 : S <= 64 ? 4 : 16; }

// Chunks of the time axis: none while the channels give one wave per SIMD or the rows are short; else enough for two waves each, 16 steps at least
// (1 x 1000 x 500 x 16: 35 us against 43 with 32 and 63 with 64 steps at least).  Cut and whole, lines of 150 x 400 fp32: 32 of them 49 / 66 us, 64 58 / 67,
// 96 85 / 67, 128 93 / 67; lines of 150 x 64: 64 of them 41 / 65, 128 64 / 65, 256 88 / 66; rows of 1000 x 512: 64 of them 289 / 413, 96 428 / 428.
// The rule counts channels, not the waves launched, which on narrow rows are up to four times as many.
void cut_time(const krk_scan_args& a, ScanCut& c) {
    const long waves = (long)a.N * a.D * lanes_of(a.S) / 64 + 1;
    long chunks = waves > 768 ? 1 : min((long)a.T / 16, 2048 / waves);
    chunks = max(1L, min(chunks, 1024L));
    c.len = a.T > 0 ? (int)((a.T + chunks - 1) / chunks) : 1;
    c.chunks = a.T > 0 ? (a.T + c.len - 1) / c.len : 1;
}

template <class T, int LP, int SL>
int launch(const krk_scan_args& a, hipStream_t s) {
    ScanCut c;
    cut_time(a, c);
    const long states = (long)a.N * (c.chunks - 1) * a.D;
    c.part = (float*)a.workspace;
    c.sums = c.part + states * a.S;
    const int per_block = 256 / LP;
    const long blocks = (long)a.G * ((a.D / a.G + per_block - 1) / per_block);
    const unsigned rows = (unsigned)min(a.N, 65535);
    if (seq_grid_too_large(blocks, 256)) return -4;
    if (c.chunks > 1) {
        hipLaunchKernelGGL((scan_seq_kernel<T, LP, SL, false>), dim3((unsigned)blocks, c.chunks - 1, rows), dim3(256), 0, s, a, c);
        hipLaunchKernelGGL(scan_join_kernel, dim3((unsigned)(((long)a.D * a.S + 255) / 256), rows), dim3(256), 0, s, a, c);
    }
    hipLaunchKernelGGL((scan_seq_kernel<T, LP, SL, true>), dim3((unsigned)blocks, c.chunks, rows), dim3(256), 0, s, a, c);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

template <class T, int LP>
int launch_step(const krk_scan_args& a, hipStream_t s) {
    const long blocks = ((long)a.N * a.D * LP + 255) / 256;
    if (seq_grid_too_large(blocks, 256)) return -4;
    hipLaunchKernelGGL((scan_step_kernel<T, LP>), dim3((unsigned)blocks), dim3(256), 0, s, a);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

template <class T>
int by_states(const krk_scan_args& a, hipStream_t s) {
    if (a.T == 1) {
        if (a.S <= 4) return launch_step<T, 1>(a, s);
        if (a.S <= 8) return launch_step<T, 2>(a, s);
        if (a.S <= 16) return launch_step<T, 4>(a, s);
        if (a.S <= 64) return launch_step<T, 16>(a, s);
        return launch_step<T, 64>(a, s);
    }
    if (a.S <= 8) return launch<T, 1, 8>(a, s);
    if (a.S <= 16) return launch<T, 1, 16>(a, s);
    if (a.S <= 64) return launch<T, 4, 16>(a, s);
    return launch<T, 16, 16>(a, s);
}

}  // namespace

long krk_scan_workspace(const krk_scan_args& a) {
    ScanCut c;
    cut_time(a, c);
    return c.chunks > 1 ? (long)a.N * (c.chunks - 1) * a.D * (a.S + 1) * (long)sizeof(float) : 0;
}

int krk_launch_selective_scan(const krk_scan_args& a, hipStream_t s) {
    return a.type == KRK_TYPE_F32 ? by_states<float>(a, s) : a.type == KRK_TYPE_BF16 ? by_states<bf16_t>(a, s) : by_states<f16_t>(a, s);
}
