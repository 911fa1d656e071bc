// The 8-bit integer linear layer: rows of int8 codes with one f32 scale a row (k_rmsnorm_i8, k_quant_i8), and the
// product of two such matrices (k_gemm_i8).
//
//   row quantiser   a = max_i |t_i|, q_i = rint(t_i * (127 / a)) in -127..127, scale = a / 127: q_i * scale ~ t_i
//   RMS norm        s = x + delta, rounded to x's type and stored; t = s * g; r = 1 / sqrt(mean(s^2) + eps);
//                   the codes of t, scale = a * r / 127: the row factor r cancels in the codes, so it enters the
//                   scale alone and a row needs one pass: sum of squares and maximum together
//   product         C[m, n] = epilogue(acc * rowscale[m] * colscale[n] + bias[n]), acc = sum_k A[m, k] W[n, k] in
//                   int32: exact, so the order of the sum, a split of K and the choice of kernel change no bit
//
// Rows with nothing to scale: a < 2^-120 (127 / a would overflow) gives scale 0 and codes 0. A row that holds a NaN
// or an infinity, or whose sum of squares leaves f32, gives scale NaN and codes 0, so that what is computed from it
// is NaN and not a plausible number.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "gemm.cuh"

namespace mf {

constexpr float kI8Tiny = 7.52316385e-37f;   // 2^-120

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// A row's scale and the factor of its codes from the bits of max |t| (as an integer: a NaN is above an infinity is
// above every number) and, for the norm, r = 1 / sqrt(mean(s^2) + eps), 1 otherwise.
struct RowScale {
    float scale, inv;
};
__device__ __forceinline__ RowScale row_scale(uint32_t amax_bits, float r)
{
    const float a = __uint_as_float(amax_bits);
    if (amax_bits >= 0x7F800000u || !(r > 0.f)) return {__uint_as_float(0x7FC00000u), 0.f};
    if (a < kI8Tiny) return {0.f, 0.f};
    return {__fdiv_rn(a * r, 127.f), __fdiv_rn(127.f, a)};
}

// The code of t. A row without a scale (inv 0) has codes 0, whatever t is.
__device__ __forceinline__ int code_of(float t, float inv) { return inv == 0.f ? 0 : __float2int_rn(t * inv); }

// One block a row; D any, every element by itself.
template <typename XT, typename DT, bool NORM>
__global__ void __launch_bounds__(256) rows_i8_kernel(const XT* __restrict__ x, const DT* __restrict__ delta,
                                                      const float* __restrict__ g, XT* out, int8_t* __restrict__ q,
                                                      float* __restrict__ scale, int D, long long ldx, long long ldd,
                                                      long long ldo, long long ldq, float eps)
{
    griddep_wait();
    griddep_launch();
    __shared__ float s_sum[8];
    __shared__ uint32_t s_max[8];
    const size_t row = blockIdx.x;
    auto value = [&](int i) {
        float s = to_f32(x[row * ldx + i]);
        if (delta) s = to_f32(from_f32<XT>(s + to_f32(delta[row * ldd + i])));
        return s;
    };
    float ss = 0.f;
    uint32_t mx = 0;
    for (int i = threadIdx.x; i < D; i += 256) {
        const float s = value(i);
        ss += s * s;
        mx = max(mx, __float_as_uint(NORM ? s * g[i] : s) & 0x7FFFFFFFu);
    }
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    mx = __reduce_max_sync(0xffffffffu, mx);
    if ((threadIdx.x & 31) == 0) {
        s_sum[threadIdx.x >> 5] = ss;
        s_max[threadIdx.x >> 5] = mx;
    }
    __syncthreads();
    ss = 0.f;
    mx = 0;
    for (int w = 0; w < 8; ++w) {
        ss += s_sum[w];
        mx = max(mx, s_max[w]);
    }
    const RowScale rs = row_scale(mx, NORM ? rsqrtf(ss / D + eps) : 1.f);
    for (int i = threadIdx.x; i < D; i += 256) {
        const float s = value(i);
        if (delta) out[row * ldo + i] = from_f32<XT>(s);
        q[row * ldq + i] = static_cast<int8_t>(code_of(NORM ? s * g[i] : s, rs.inv));
    }
    if (threadIdx.x == 0) scale[row] = rs.scale;
}

// One thread an output, 16 x 16 outputs a block, K by 64 codes through shared memory.
template <typename TO, int EPI>
__global__ void __launch_bounds__(256) gemm_i8_simple_kernel(const int8_t* __restrict__ A, const int8_t* __restrict__ W,
                                                             const float* __restrict__ rowscale,
                                                             const float* __restrict__ colscale,
                                                             const float* __restrict__ bias, TO* C, int M, int N, int K,
                                                             long long lda, long long ldw, long long ldc)
{
    griddep_wait();
    griddep_launch();
    __shared__ int sa[16][17], sw[16][17];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const long long m0 = (long long)blockIdx.y * 16, n0 = (long long)blockIdx.x * 16;
    auto word = [&](const int8_t* p, long long ld, long long r, long long rows, int k) {
        uint32_t w = 0;
        if (r < rows)
            for (int b = 0; b < 4; ++b)
                if (k + b < K) w |= (uint32_t)(uint8_t)p[r * ld + k + b] << (8 * b);
        return (int)w;
    };
    int acc = 0;
    for (int k0 = 0; k0 < K; k0 += 64) {
        sa[ty][tx] = word(A, lda, m0 + ty, M, k0 + 4 * tx);
        sw[ty][tx] = word(W, ldw, n0 + ty, N, k0 + 4 * tx);
        __syncthreads();
        for (int j = 0; j < 16; ++j) acc = __dp4a(sa[ty][j], sw[tx][j], acc);
        __syncthreads();
    }
    const long long m = m0 + ty, n = n0 + tx;
    if (m >= M || n >= N) return;
    float v = i8_value(acc, rowscale[m], colscale[n], bias ? bias[n] : 0.f);
    if constexpr (EPI == kEpiBiasGelu) v = gelu_pair<false, true>(pk2(v, v), GeluK(1.0f)).x;
    if constexpr (EPI == kEpiResidual) v += C[m * ldc + n];
    C[m * ldc + n] = from_f32<TO>(v);
}

}  // namespace mf
