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

#include "trunk.cuh"

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

// The arguments of the row kernels (pitches in elements). delta and out nullptr: nothing is added or stored.
struct RowsI8 {
    const void *x, *delta;
    const float* g;          // the norm only
    void* out;
    int8_t* q;
    float* scale;
    int M, D;
    long long ldx, ldd, ldo, ldq;
    float eps;
};

// 8 elements as they lie in memory, so that all of a thread's loads are on their way before the first is converted.
template <typename T> struct Raw8 {
    uint4 w;
    __device__ __forceinline__ void load(const T* p) { w = __ldg(reinterpret_cast<const uint4*>(p)); }   // on 16 bytes
    __device__ __forceinline__ void zero() { w = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void get(float (&v)[8]) const
    {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same<T, __half>::value) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
                v[2 * i] = f.x, v[2 * i + 1] = f.y;
            } else {
                v[2 * i] = bf16_lo(u[i]), v[2 * i + 1] = bf16_hi(u[i]);
            }
        }
    }
};
template <> struct Raw8<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p)
    {
        a = __ldg(reinterpret_cast<const float4*>(p));
        b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    }
    __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
    __device__ __forceinline__ void get(float (&v)[8]) const
    {
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    }
};
__device__ __forceinline__ void store8(float* p, const float (&v)[8])
{
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float (&v)[8])
{
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
}

// The code of t as the low byte of t * inv + 1.5 * 2^23, whose sum is rounded to a whole number, ties to even: one
// instruction where a conversion to an integer runs at a quarter of the rate. |t * inv| < 127.001.
__device__ __forceinline__ uint32_t code_byte(float t, float inv) { return __float_as_uint(fmaf(t, inv, 12582912.f)); }
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d, float inv)
{
    return __byte_perm(__byte_perm(code_byte(a, inv), code_byte(b, inv), 0x0040),
                       __byte_perm(code_byte(c, inv), code_byte(d, inv), 0x0040), 0x5410);
}

// L threads hold a row in registers (8, 16 or 32 of a warp, or a block, L = 0), 8 V elements a thread, so x and delta
// are read and out, q and scale written once: bound by HBM from about a thousand rows. VEC: neighbouring elements 8 at a
// time (D a multiple of 8, every row of every operand begins on 16 bytes, q's on 8); else element by element.
template <typename XT, typename DT, bool NORM, bool VEC, int L, int V>
__global__ void __launch_bounds__(L ? 256 : 1024) rows_i8_kernel(const RowsI8 a)
{
    griddep_wait();
    griddep_launch();
    const int T = L ? L : blockDim.x;
    const int t = L ? threadIdx.x & (L - 1) : threadIdx.x;
    const size_t row = L ? ((size_t)blockIdx.x * blockDim.x + threadIdx.x) / (L ? L : 1) : blockIdx.x;
    // a warp that holds a row at all goes on as a whole, its threads without one with no elements
    if (L && row - (threadIdx.x & 31) / (L ? L : 1) >= (size_t)a.M) return;
    const int D = row < (size_t)a.M ? a.D : 0;
    const XT* __restrict__ x = static_cast<const XT*>(a.x) + row * a.ldx;
    const DT* __restrict__ delta = static_cast<const DT*>(a.delta) + row * a.ldd;
    XT* out = static_cast<XT*>(a.out) + row * a.ldo;
    int8_t* q = a.q + row * a.ldq;
    const bool add = NORM && a.delta;
    // element j of vector v of this thread
    auto at = [&](int v, int j) { return VEC ? 8 * (t + T * v) + j : t + T * (8 * v + j); };

    float s[V][8], d[V][8];
    if constexpr (VEC) {
        Raw8<XT> rx[V];
        Raw8<DT> rd[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            rx[v].zero();
            if (at(v, 0) < D) rx[v].load(x + at(v, 0));
        }
        if (add) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                rd[v].zero();
                if (at(v, 0) < D) rd[v].load(delta + at(v, 0));
            }
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
            rx[v].get(s[v]);
            if (add) rd[v].get(d[v]);
        }
    } else {
        XT rx[V][8];
        DT rd[V][8];
#pragma unroll
        for (int v = 0; v < V; ++v) {
#pragma unroll
            for (int j = 0; j < 8; ++j) rx[v][j] = at(v, j) < D ? x[at(v, j)] : from_f32<XT>(0.f);
        }
        if (add) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
#pragma unroll
                for (int j = 0; j < 8; ++j) rd[v][j] = at(v, j) < D ? delta[at(v, j)] : from_f32<DT>(0.f);
            }
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                s[v][j] = to_f32(rx[v][j]);
                if (add) d[v][j] = to_f32(rd[v][j]);
            }
        }
    }
    if (add) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
#pragma unroll
            for (int j = 0; j < 8; ++j) s[v][j] = to_f32(from_f32<XT>(s[v][j] + d[v][j]));
            if constexpr (VEC) {
                if (at(v, 0) < D) store8(out + at(v, 0), s[v]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (at(v, j) < D) out[at(v, j)] = from_f32<XT>(s[v][j]);
            }
        }
    }
    float ss = 0.f;
    uint32_t mx = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        if constexpr (NORM) {
            float g[8];
            if constexpr (VEC) {
                Raw8<float> rg;
                rg.zero();
                if (at(v, 0) < D) rg.load(a.g + at(v, 0));
                rg.get(g);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) g[j] = at(v, j) < D ? __ldg(a.g + at(v, j)) : 0.f;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                ss = fmaf(s[v][j], s[v][j], ss);
                s[v][j] *= g[j];
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) mx = max(mx, __float_as_uint(s[v][j]) & 0x7FFFFFFFu);
    }
    if constexpr (L == 8 || L == 16) {
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) {
            if constexpr (NORM) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        }
    } else {
        if constexpr (NORM) ss = warp_sum(ss);
        mx = __reduce_max_sync(0xffffffffu, mx);
    }
    if constexpr (L == 0) {
        __shared__ float s_sum[32];
        __shared__ uint32_t s_max[32];
        if ((t & 31) == 0) {
            s_sum[t >> 5] = ss;
            s_max[t >> 5] = mx;
        }
        __syncthreads();
        // every warp reduces the warps' values for itself
        const int w = t & 31;
        ss = w < T / 32 ? s_sum[w] : 0.f;
        mx = w < T / 32 ? s_max[w] : 0u;
        if constexpr (NORM) ss = warp_sum(ss);
        mx = __reduce_max_sync(0xffffffffu, mx);
    }
    const RowScale rs = row_scale(mx, NORM ? rsqrtf(ss / static_cast<float>(a.D) + a.eps) : 1.f);
    if (t == 0 && D) a.scale[row] = rs.scale;
    const uint32_t live = rs.inv == 0.f ? 0u : 0xFFFFFFFFu;   // a row without a scale has codes 0, whatever it holds
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const uint32_t lo = codes4(s[v][0], s[v][1], s[v][2], s[v][3], rs.inv) & live;
        const uint32_t hi = codes4(s[v][4], s[v][5], s[v][6], s[v][7], rs.inv) & live;
        if constexpr (VEC) {
            if (at(v, 0) < D) *reinterpret_cast<uint2*>(q + at(v, 0)) = make_uint2(lo, hi);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (at(v, j) < D) q[at(v, j)] = static_cast<int8_t>((j < 4 ? lo : hi) >> (8 * (j & 3)));
        }
    }
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
