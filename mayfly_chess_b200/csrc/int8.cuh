// The 8-bit integer linear layer: rows of int8 codes with one f32 scale a row (k_rmsnorm_i8, k_quant_i8), and the
// product of two such matrices (k_gemm_i8).
//
//   row quantiser   a = max_i |t_i|, q_i = rint(127 t_i / a) in -127..127, scale = a / 127: q_i * scale ~ t_i
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
// above every number) and, for the norm, r = 1 / sqrt(mean(s^2) + eps), 1 otherwise. The factor is 127 / a: UP, rounded
// up; else inv + rest, its rounding to f32 and what that leaves (codes2 says which is for whom).
struct RowScale {
    float scale, inv, rest;
};
template <bool UP> __device__ __forceinline__ RowScale row_scale(uint32_t amax_bits, float r)
{
    const float a = __uint_as_float(amax_bits);
    if (amax_bits >= 0x7F800000u || !(r > 0.f)) return {__uint_as_float(0x7FC00000u), 0.f, 0.f};
    if (a < kI8Tiny) return {0.f, 0.f, 0.f};
    const float scale = __fdiv_rn(a * r, 127.f);
    if constexpr (UP) return {scale, __fdiv_ru(127.f, a), 0.f};
    const float inv = __fdiv_rn(127.f, a);
    return {scale, inv, __fdiv_rn(fmaf(-inv, a, 127.f), a)};
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
// RO: nothing writes them while the kernel runs (the read-only path).
template <typename T> struct Raw8 {
    uint4 w;
    template <bool RO> __device__ __forceinline__ void load(const T* p)   // on 16 bytes
    {
        const uint4* u = reinterpret_cast<const uint4*>(p);
        w = RO ? __ldg(u) : *u;
    }
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
    template <bool RO> __device__ __forceinline__ void load(const float* p)
    {
        const float4* u = reinterpret_cast<const float4*>(p);
        a = RO ? __ldg(u) : u[0];
        b = RO ? __ldg(u + 1) : u[1];
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

// The codes of two values t, each the low byte of v + 1.5 * 2^23, whose sum is rounded to a whole number, ties to even:
// one instruction where a conversion to an integer runs at a quarter of the rate. v is the quotient 127 t / a rounded
// to f32 once, |v| <= 127: a product with the rounded factor alone misses the ties (t = a / 2 is 63.5 steps, whatever a
// is; 1.3e-5 of the codes of bf16 rows of 2,048, 2.0e-5 of f16).
//   UP      bf16 values: t * inv + 1.5 * 2^23 in one fused step. With t = T 2^i, a = A 2^j, T and A < 256, the quotient
//           is a tie only for t = a / 2, where inv >= 127 / a gives 64, the even code, and for A = 254, where inv is
//           exact; it is at least 2^(i-j-9) away from every tie otherwise, and off by less than 2^(i-j-15)
//   else    t * inv + t * rest. PAIRED: two values an instruction. 33,280 x 2,048 f16 quantised 32.0 us, one at a time
//           34.7, with inv alone 30.8; but 20,871 x 727 f16, element by element in a warp, 15.0 and 12.2
template <bool UP, bool PAIRED> __device__ __forceinline__ uint2 codes2(float t, float u, const RowScale& rs)
{
    constexpr float kRound = 12582912.f;
    if constexpr (UP) {
        return make_uint2(__float_as_uint(fmaf(t, rs.inv, kRound)), __float_as_uint(fmaf(u, rs.inv, kRound)));
    } else if constexpr (PAIRED) {
        const uint64_t t2 = pk2(t, u), low = mul2(t2, pk2(rs.rest, rs.rest));
        const float2 v = upk2(add2(fma2(t2, pk2(rs.inv, rs.inv), low), pk2(kRound, kRound)));
        return make_uint2(__float_as_uint(v.x), __float_as_uint(v.y));
    } else {
        return make_uint2(__float_as_uint(__fadd_rn(fmaf(t, rs.inv, __fmul_rn(t, rs.rest)), kRound)),
                          __float_as_uint(__fadd_rn(fmaf(u, rs.inv, __fmul_rn(u, rs.rest)), kRound)));
    }
}
template <bool UP, bool PAIRED> __device__ __forceinline__ uint32_t codes4(const float* t, const RowScale& rs)
{
    const uint2 a = codes2<UP, PAIRED>(t[0], t[1], rs), b = codes2<UP, PAIRED>(t[2], t[3], rs);
    return __byte_perm(__byte_perm(a.x, a.y, 0x0040), __byte_perm(b.x, b.y, 0x0040), 0x5410);
}

// L threads hold a row in registers (8, 16 or 32 of a warp, or a block, L = 0), 8 V elements a thread, so x and delta
// are read and out, q and scale written once: bound by HBM from about a thousand rows (norm 66,560 x 1,024, f32 + bf16:
// 110 us, 6.8 TB/s; quantiser 66,560 x 2,048 bf16: 59 us, 6.9 TB/s). VEC: neighbouring elements 8 at a
// time (D a multiple of 8, every row of every operand begins on 16 bytes, q's on 8); else element by element.
template <typename XT, typename DT, bool NORM, bool VEC, int L, int V>
__global__ void __launch_bounds__(L ? 128 : 1024) rows_i8_kernel(const RowsI8 a)
{
    griddep_wait();
    griddep_launch();
    const int T = L ? L : blockDim.x;
    const int t = L ? threadIdx.x & (L - 1) : threadIdx.x;
    const size_t row = L ? ((size_t)blockIdx.x * blockDim.x + threadIdx.x) / (L ? L : 1) : blockIdx.x;
    // a warp that holds a row at all goes on as a whole, its threads without one with no elements
    if (L && row - (threadIdx.x & 31) / (L ? L : 1) >= (size_t)a.M) return;
    const int D = row < (size_t)a.M ? a.D : 0;
    // This thread's first element, and the elements from there to the row's end: element j of vector v lies at(v, j)
    // further on. Element by element a warp (or the part of it that has the row) has its neighbours, so that the
    // distances are constants: what such a row costs is instructions.
    const int e0 = VEC ? 8 * t : L ? t : (t >> 5) * 256 * V + (t & 31);
    const int left = D - e0;
    auto at = [&](int v, int j) { return VEC ? 8 * T * v + j : (L ? L : 32) * (8 * v + j); };
    // the norm's out may be x or delta: ordinary loads, all of a thread's ahead of its first store
    const XT* x = static_cast<const XT*>(a.x) + row * a.ldx + e0;
    const DT* delta = static_cast<const DT*>(a.delta) + row * a.ldd + e0;
    const float* __restrict__ gp = NORM ? a.g + e0 : nullptr;
    XT* out = static_cast<XT*>(a.out) + row * a.ldo + e0;
    int8_t* q = a.q + row * a.ldq + e0;
    const bool add = NORM && a.delta;

    float s[V][8], d[V][8];
    if constexpr (VEC) {
        Raw8<XT> rx[V];
        Raw8<DT> rd[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            rx[v].zero();
            if (at(v, 0) < left) rx[v].template load<!NORM>(x + at(v, 0));
        }
        if (add) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                rd[v].zero();
                if (at(v, 0) < left) rd[v].template load<false>(delta + at(v, 0));
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
            for (int j = 0; j < 8; ++j) rx[v][j] = at(v, j) < left ? x[at(v, j)] : from_f32<XT>(0.f);
        }
        if (add) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
#pragma unroll
                for (int j = 0; j < 8; ++j) rd[v][j] = at(v, j) < left ? delta[at(v, j)] : from_f32<DT>(0.f);
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
                if (at(v, 0) < left) store8(out + at(v, 0), s[v]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (at(v, j) < left) out[at(v, j)] = from_f32<XT>(s[v][j]);
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
                if (at(v, 0) < left) rg.template load<true>(gp + at(v, 0));
                rg.get(g);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) g[j] = at(v, j) < left ? __ldg(gp + at(v, j)) : 0.f;
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
    constexpr bool UP = !NORM && std::is_same<XT, __nv_bfloat16>::value, PAIRED = NORM || VEC || L == 0;
    const RowScale rs = row_scale<UP>(mx, NORM ? rsqrtf(ss / static_cast<float>(a.D) + a.eps) : 1.f);
    if (t == 0 && D) a.scale[row] = rs.scale;
    if (rs.inv == 0.f) {   // a row without a scale has codes 0, whatever it holds
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int j = 0; j < 8; ++j) s[v][j] = 0.f;
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
        if constexpr (VEC) {
            if (at(v, 0) < left)
                *reinterpret_cast<uint2*>(q + at(v, 0)) =
                    make_uint2(codes4<UP, PAIRED>(s[v], rs), codes4<UP, PAIRED>(s[v] + 4, rs));
        } else {
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const uint2 c = codes2<UP, PAIRED>(s[v][j], s[v][j + 1], rs);
                if (at(v, j) < left) q[at(v, j)] = static_cast<int8_t>(c.x);
                if (at(v, j + 1) < left) q[at(v, j + 1)] = static_cast<int8_t>(c.y);
            }
        }
    }
}

// The value of an accumulator before GELU or a residual's addition, a rounding a step and the same in every kernel, so
// that they agree to the bit.
__device__ __forceinline__ float i8_value(int acc, float rowscale, float colscale, float bias)
{
    return fmaf(__fmul_rn(__int2float_rn(acc), rowscale), colscale, bias);
}

// The outputs and vectors of a product.
struct I8Out {
    const float *rowscale, *colscale, *bias;
    void* C;
    long long ldc;
    int M, N, K, n_tiles;
    int direct;              // the pair kernel: C's rows are not whole 16-byte units, plain stores
    int stall;               // the split kernel: a cluster's last CTA loads nothing, so that its waits run out
};

// ------------------------------------------------------------------------------------------------ many rows
// 256 x 256 tiles on CTA pairs (tcgen05.mma.cta_group::2, kind::i8), persistent: each CTA holds 128 rows of A, 128 of the
// 256 rows of W and 128 x 256 accumulators, two of them, so that a tile's epilogue runs under the next tile's products.
// At the full rate of the products the operands' arrival takes half of shared memory's 128 bytes a cycle and their
// reading the other half, and the epilogue's staging comes on top. So a pair takes neighbouring tiles, W's blocks
// fastest, and keeps its rows of A in shared memory over all of them where they fit (K <= 1,024): only W then streams.
// What paced the products before was their issue: by one lane of a diverged warp, with two commits a stage, 187 cycles an
// instruction; from a converged warp with one commit to both CTAs 128 to 140 (66,560 x 2,048 x 1,024: 131 -> 113 us).
// What bounds it now: 8,192^3 keeps the tensor cores busy 92% of their cycles (2,600 TOP/s); the 1,000 W cap, which takes
// the clock from 1.97 to about 1.4 GHz in a long run (66,560 x 2,048 x 1,024 there 133 us, with GELU 156; cool 111 and
// 131); and with GELU the epilogue's instructions (7,900 cycles a tile, 6,100 without it, 4,096 of products).
// Roles: warp 0 TMA loads, warp 1 tensor memory and the products (leader CTA), warps 2..17 the epilogue.
struct I8PairCfg {
    static constexpr int SLOTS = 11;                     // of 128 rows x 128 bytes
    static constexpr uint32_t SLOT = 128 * 128;
    static constexpr int MAX_A = 8, RING = 5;            // blocks of A that stay; stages of both where they do not
    static constexpr int MAX_B = 8;
    static constexpr int GROUPS = 4, COLS = 64;          // epilogue groups of 4 warps, columns of a tile each
    static constexpr uint32_t STAGE = 32 * 64;           // a warp's staging: 32 rows x 64 bytes
    static constexpr size_t SMEM = 1024 + SLOTS * SLOT + 4 * GROUPS * STAGE + GROUPS * 2 * 2 * COLS * 4 + 512;
    static constexpr int THREADS = 64 + 128 * GROUPS;
};

// A warp owns 32 rows of the tile and COLS neighbouring columns: it converts them from tensor memory into its own
// staging chunk, and its lane 0 stores the chunk (for the residual: adds it at L2) by TMA, so that the warps of a group
// meet once a tile and not at every chunk; where C does not suit TMA, the warp stores the chunk row by row. The group's
// column scales and bias of a tile are read by its 128 threads a tile ahead and passed through shared memory: each is
// read once from L2, and an aligned float4 serves a warp.
template <typename TO, int EPI, typename OriginFn, typename ReleaseFn>
__device__ __forceinline__ void i8_pair_epilogue(const CUtensorMap* tmC, const I8Out& p, uint8_t* stages, float* vecs,
                                                 volatile uint32_t* epi_ok, uint64_t* tfull, uint32_t tmem_base,
                                                 int tiles, OriginFn origin, ReleaseFn release, uint32_t* err)
{
    using C = I8PairCfg;
    griddep_wait();
    constexpr int COLS = C::COLS, CHUNK = 64 / sizeof(TO);   // columns of a 64-byte row of staging
    constexpr int LD = CHUNK < 32 ? CHUNK : 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int grp = (warp - 2) >> 2, gtid = (int)threadIdx.x - 64 - 128 * grp;
    const int quarter = warp & 3;
    const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(grp * COLS);
    uint8_t* const stage = stages + (grp * 4 + quarter) * C::STAGE;
    float* const svec = vecs + grp * 2 * 2 * COLS;

    float next = 0.f, next_rs = 0.f;
    auto read_ahead = [&](int it) {
        if (it >= tiles) return;
        const int2 o = origin(it);                           // row, column
        const int n = o.y + grp * COLS + (gtid & (COLS - 1)), r = o.x + quarter * 32 + lane;
        const float* src = gtid < COLS ? p.colscale : p.bias;
        next = src && n < p.N ? __ldg(src + n) : 0.f;
        next_rs = r < p.M ? __ldg(p.rowscale + r) : 0.f;
    };
    read_ahead(0);

    int acc = 0;
    uint32_t acc_phase = 0;
    for (int it = 0; it < tiles; ++it) {
        const int2 o = origin(it);
        const int row0 = o.x + quarter * 32, col0 = o.y + grp * COLS;
        float* sv = svec + (it & 1) * 2 * COLS;              // the other half is still read by this group's slower warps
        sv[gtid] = next;
        const uint64_t rs2 = pk2(next_rs, next_rs);
        // the group's one decision; the word of the tile before may still be read by its slower warps
        volatile uint32_t* const go = epi_ok + (it & 1) * C::GROUPS + grp;
        if (gtid == 0) *go = mbar_wait(&tfull[acc], acc_phase, err, kErrTmemFull) ? 1u : 0u;
        named_barrier(1 + grp, 128);
        if (!*go) break;
        tc_fence_after();
        read_ahead(it + 1);
        const uint32_t t_acc = t_lane + static_cast<uint32_t>(acc * 256);
#pragma unroll 1
        for (int c = 0; c < COLS; c += CHUNK) {
            uint32_t a[LD], q[16];
            if constexpr (LD == 32) tmem_ld_32x32b_x32(t_acc + static_cast<uint32_t>(c), a);
            else tmem_ld_32x32b_x16(t_acc + static_cast<uint32_t>(c), a);
            tmem_ld_wait(a);
            if (c == COLS - CHUNK) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) release(acc);
            }
#pragma unroll
            for (int i = 0; i < LD; i += 4) {
                const float4 sc = *reinterpret_cast<const float4*>(sv + c + i);
                const float4 b = *reinterpret_cast<const float4*>(sv + COLS + c + i);
                const uint64_t lo = fma2(mul2(pk2(__int2float_rn((int)a[i]), __int2float_rn((int)a[i + 1])), rs2),
                                         pk2(sc.x, sc.y), pk2(b.x, b.y));
                const uint64_t hi = fma2(mul2(pk2(__int2float_rn((int)a[i + 2]), __int2float_rn((int)a[i + 3])), rs2),
                                         pk2(sc.z, sc.w), pk2(b.z, b.w));
                float2 x, y;
                if constexpr (EPI == kEpiBiasGelu) {
                    x = gelu_pair<false, true>(lo, GeluK(1.0f));
                    y = gelu_pair<false, true>(hi, GeluK(1.0f));
                } else {
                    x = upk2(lo);
                    y = upk2(hi);
                }
                if constexpr (sizeof(TO) == 2) {
                    q[i / 2] = pack2<TO>(x.x, x.y);
                    q[i / 2 + 1] = pack2<TO>(y.x, y.y);
                } else {
                    q[i] = __float_as_uint(x.x);
                    q[i + 1] = __float_as_uint(x.y);
                    q[i + 2] = __float_as_uint(y.x);
                    q[i + 3] = __float_as_uint(y.y);
                }
            }
            if (lane == 0) bulk_wait_read<0>();              // the last store out of this chunk has read it
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *reinterpret_cast<uint4*>(stage + swz<64>(lane, j)) =
                    make_uint4(q[4 * j], q[4 * j + 1], q[4 * j + 2], q[4 * j + 3]);
            if (p.direct) {
                // the warp's 32 x CHUNK values row by row, a row's columns by neighbouring lanes; a residual is added at L2,
                // once an element (27,690 x 2,993 x 848: 207 us, 255 where the warp reads, adds and writes)
                __syncwarp();
                constexpr int RPI = 32 / CHUNK;              // rows an instruction
                const int cc = lane % CHUNK, n = col0 + c + cc, first = lane / CHUNK;
                const int rows = n < p.N ? p.M - row0 : 0;
                TO* cp = static_cast<TO*>(p.C) + (size_t)(row0 + first) * p.ldc + n;
                const size_t step = RPI * (size_t)p.ldc;
#pragma unroll 1
                for (int i = 0; i < 32; i += 8 * RPI, cp += 8 * step) {
                    TO v[8];
#pragma unroll
                    for (int u = 0; u < 8; ++u) {
                        const int r = i + u * RPI + first;
                        v[u] = *reinterpret_cast<const TO*>(stage + swz<64>(r, cc * (int)sizeof(TO) / 16) +
                                                            cc * (int)sizeof(TO) % 16);
                    }
#pragma unroll
                    for (int u = 0; u < 8; ++u)
                        if (i + u * RPI + first < rows) {
                            if constexpr (EPI == kEpiResidual) atomicAdd(cp + u * step, v[u]);
                            else cp[u * step] = v[u];
                        }
                }
                __syncwarp();                                // read, before the next chunk overwrites it
                continue;
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0 && row0 < p.M) {
                if constexpr (EPI == kEpiResidual) tma_reduce_add_2d(tmC, stage, col0 + c, row0);
                else tma_store_2d(tmC, stage, col0 + c, row0);
                bulk_commit();
            }
        }
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1u;
    }
    if (lane == 0) bulk_wait_all();
}

template <typename TO, int EPI>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(I8PairCfg::THREADS, 1)
gemm_i8_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW,
                    const __grid_constant__ CUtensorMap tmC, const I8Out p, uint32_t* err)
{
    using C = I8PairCfg;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* const slots = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* const stages = slots + C::SLOTS * C::SLOT;
    float* const vecs = reinterpret_cast<float*>(stages + 4 * C::GROUPS * C::STAGE);
    uint64_t* const full_a = reinterpret_cast<uint64_t*>(vecs + C::GROUPS * 2 * 2 * C::COLS);
    uint64_t* const empty_a = full_a + C::MAX_A;
    uint64_t* const full_b = empty_a + C::MAX_A;
    uint64_t* const empty_b = full_b + C::MAX_B;
    uint64_t* const tfull = empty_b + C::MAX_B;
    uint64_t* const tempty = tfull + 2;
    uint64_t* const mma_done = tempty + 2;
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(mma_done + 1);
    volatile uint32_t* const epi_ok = tmem_slot + 1;   // [2][GROUPS]

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const bool lead = rank == 0;
    const int pair = (int)blockIdx.x >> 1, pairs = (int)gridDim.x >> 1;
    const long long all = (long long)((p.M + 255) / 256) * p.n_tiles;
    const int lo = static_cast<int>(all * pair / pairs), hi = static_cast<int>(all * (pair + 1) / pairs);
    const int blocks = (p.K + 127) / 128;
    // A's blocks stay over a row of tiles, in slots of their own; else both operands go round a ring
    const bool stay = blocks <= C::MAX_A;
    const int na = stay ? blocks : C::RING;
    const int nb = stay ? (C::SLOTS - na < C::MAX_B ? C::SLOTS - na : C::MAX_B) : C::RING;

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::MAX_A; ++s) {
            mbar_init(&full_a[s], 1);
            mbar_init(&empty_a[s], 1);
        }
        for (int s = 0; s < C::MAX_B; ++s) {
            mbar_init(&full_b[s], 1);
            mbar_init(&empty_b[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&tfull[b], 1);
            mbar_init(&tempty[b], 2 * 4 * C::GROUPS);   // the epilogue warps of both CTAs
        }
        mbar_init(mma_done, 1);
        fence_barrier_init();
        tma_prefetch_desc(&tmA);
        tma_prefetch_desc(&tmW);
        if (!p.direct) tma_prefetch_desc(&tmC);
    }
    if (warp == 1) {
        tmem_alloc_pair(tmem_slot, 512);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    cluster_sync();   // both CTAs' barriers exist before either signals the other's
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    if (threadIdx.x == 0) griddep_launch();

    if (warp == 0) {
        if (lane == 0) {
            griddep_wait();
            int sa = 0, sb = 0;
            uint32_t pha = 0, phb = 0;                  // parities of the rounds of A's and W's slots
            uint32_t used_a = 0, par_a = 0, used_b = 0, par_b = 0;   // slots loaded, and the parity of their last load
            bool ok = true;
            for (int tile = lo; tile < hi && ok; ++tile) {
                const int n_blk = tile % p.n_tiles;
                const int a_row = tile / p.n_tiles * 256 + (int)rank * 128, b_row = n_blk * 256 + (int)rank * 128;
                const bool fresh = stay && (tile == lo || n_blk == 0);
                for (int kb = 0; kb < blocks; ++kb) {
                    if (fresh) {
                        if (!(ok = mbar_wait(&empty_a[sa], pha ^ 1u, err, kErrSmemEmpty))) break;
                        if (lead) mbar_arrive_expect_tx(&full_a[sa], 2 * C::SLOT);
                        tma_load_2d_pair(slots + sa * C::SLOT, &tmA, mapa_shared(smem_u32(&full_a[sa]), 0), kb * 128, a_row);
                        used_a |= 1u << sa;
                        par_a = (par_a & ~(1u << sa)) | (pha << sa);
                        if (++sa == na) sa = 0, pha ^= 1u;
                    }
                    if (!(ok = mbar_wait(&empty_b[sb], phb ^ 1u, err, kErrSmemEmpty))) break;
                    if (lead) mbar_arrive_expect_tx(&full_b[sb], (stay ? 2 : 4) * C::SLOT);
                    const uint32_t full = mapa_shared(smem_u32(&full_b[sb]), 0);
                    if (!stay) tma_load_2d_pair(slots + sb * C::SLOT, &tmA, full, kb * 128, a_row);
                    tma_load_2d_pair(slots + (na + sb) * C::SLOT, &tmW, full, kb * 128, b_row);
                    used_b |= 1u << sb;
                    par_b = (par_b & ~(1u << sb)) | (phb << sb);
                    if (++sb == nb) sb = 0, phb ^= 1u;
                }
            }
            // this CTA's copies have landed before it can leave: the leader sees them on its `full` barriers, the other
            // CTA on its `empty` ones (a slot is released only after both halves landed and were read)
            for (int s = 0; s < C::MAX_A; ++s)
                if (used_a >> s & 1) mbar_wait(lead ? &full_a[s] : &empty_a[s], par_a >> s & 1, err, kErrTmaFull);
            for (int s = 0; s < C::MAX_B; ++s)
                if (used_b >> s & 1) mbar_wait(lead ? &full_b[s] : &empty_b[s], par_b >> s & 1, err, kErrTmaFull);
        }
    } else if (warp == 1) {
        if (lead) {
            // The whole warp walks the loop and one lane issues, so that stages and descriptors stay in uniform
            // registers: issuing is what paces the products otherwise.
            constexpr uint32_t idesc = idesc_i8(256, 256);
            const uint64_t desc0 = sdesc_sw128(smem_u32(slots));
            int sb = 0;
            uint32_t pha = 0, phb = 0;
            int acc = 0, n_blk = lo % p.n_tiles;
            uint32_t acc_phase = 0;
            bool ok = true;
            for (int tile = lo; tile < hi; ++tile) {
                if (!__all_sync(0xffffffffu, mbar_wait(&tempty[acc], acc_phase ^ 1u, err, kErrTmemEmpty))) break;
                tc_fence_after();
                const bool fresh = stay && (tile == lo || n_blk == 0);
                const bool last = stay && (tile == hi - 1 || n_blk == p.n_tiles - 1);
                const uint32_t d = tmem_base + static_cast<uint32_t>(acc * 256);
                for (int kb = 0; kb < blocks; ++kb) {
                    ok = !fresh || mbar_wait(&full_a[kb], pha, err, kErrTmaFull);
                    ok = mbar_wait(&full_b[sb], phb, err, kErrTmaFull) && ok;
                    if (!(ok = __all_sync(0xffffffffu, ok))) break;
                    tc_fence_after();
                    // a slot is SLOT / 16 steps of a descriptor's address, an instruction's 32 bytes of K two
                    const uint64_t a = desc0 + static_cast<uint32_t>((stay ? kb : sb) * (int)(C::SLOT / 16));
                    const uint64_t w = desc0 + static_cast<uint32_t>((na + sb) * (int)(C::SLOT / 16));
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) umma_i8_pair(d, a + 2 * k, w + 2 * k, idesc, (kb | k) != 0 ? 1u : 0u);
                        umma_commit_pair_both(&empty_b[sb]);
                        if (last) umma_commit_pair_both(&empty_a[kb]);
                        if (kb == blocks - 1) umma_commit_pair_both(&tfull[acc]);
                    }
                    __syncwarp();
                    if (++sb == nb) sb = 0, phb ^= 1u;
                }
                if (!ok) break;
                if (last) pha ^= 1u;
                if (++n_blk == p.n_tiles) n_blk = 0;
                acc ^= 1;
                if (acc == 0) acc_phase ^= 1u;
            }
            // every product issued has completed (both CTAs' tensor memory) before either frees it
            if (elect_one()) umma_commit_pair(smem_u32(mma_done));
            __syncwarp();
            mbar_wait(mma_done, 0, err, kErrTmemFull);
        }
    } else {
        const uint32_t tempty0 = mapa_shared(smem_u32(&tempty[0]), 0), tempty1 = mapa_shared(smem_u32(&tempty[1]), 0);
        i8_pair_epilogue<TO, EPI>(
            &tmC, p, stages, vecs, epi_ok, tfull, tmem_base, hi - lo,
            [&](int it) {
                return make_int2((lo + it) / p.n_tiles * 256 + (int)rank * 128, (lo + it) % p.n_tiles * 256);
            },
            [&](int acc) { mbar_arrive_cluster_tmem(acc ? tempty1 : tempty0); }, err);
    }

    __syncwarp();
    tc_fence_before();
    cluster_sync();   // the leader's products are done and no CTA signals the other any more
    tc_fence_after();
    if (warp == 1) tmem_dealloc_pair(tmem_base, 512);
}

// ------------------------------------------------------------------------------------------------ few rows
// The product for few rows of A. The weight takes the 128 lanes of the tensor-core instruction (M = 128 rows of W) and the
// tokens its columns (N = TN rows of A), so that a few tokens waste little and a thread of the epilogue owns an output
// channel: its column scale and bias stay in two registers, and a warp stores 32 neighbouring channels of a row, wherever
// the row begins. K is split over a cluster of S CTAs, which fills the GPU where the tiles alone do not: each CTA leaves
// its exact int32 partial sums in its shared memory and sums a share of the tokens over the cluster through distributed
// shared memory, without a workspace; where a CTA of the cluster has given up on a wait, none stores. Bound by
// what W takes from HBM plus about 5 us (start, first bytes, exchange): 16 x 32,768 x 8,192 43.8 us (6.1 TB/s),
// 16 x 8,192 x 8,192 15.4 us, out of L2 9.7 us; 1 x 8,324 x 1,024 4.3 us; 777 x 1,001 x 1,000 added in place 6.7 us (7.9
// where it reads, adds and writes).
template <int TN> struct I8SplitCfg {
    static constexpr uint32_t W_BYTES = 128 * 128, A_BYTES = TN * 128, STAGE_BYTES = W_BYTES + A_BYTES;
    static constexpr int STAGES = TN == 128 ? 3 : TN == 64 ? 4 : 5;   // two CTAs an SM
    static constexpr uint32_t TMEM_COLS = TN < 32 ? 32 : TN;
    static constexpr size_t SMEM = 1024 + STAGES * STAGE_BYTES + 4 * (TN + 4) + 16 * STAGES + 32;
    static constexpr int GROUPS = 4;                                  // of 4 epilogue warps, TN / 4 tokens each
    static constexpr int THREADS = 64 + 128 * GROUPS;
    static_assert(STAGES * STAGE_BYTES >= 4 * 128 * TN, "the partial sums lie where the stages were");
};

template <typename TO, int EPI, int TN>
__global__ void __launch_bounds__(I8SplitCfg<TN>::THREADS, 2)
gemm_i8_split_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW, const I8Out p,
                     uint32_t* err)
{
    using C = I8SplitCfg<TN>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* const sW = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* const sA = sW + C::STAGES * C::W_BYTES;
    float* const s_rowscale = reinterpret_cast<float*>(sA + C::STAGES * C::A_BYTES);
    uint64_t* const full = reinterpret_cast<uint64_t*>(s_rowscale + TN + 4);   // put2 may look one behind TN
    uint64_t* const empty = full + C::STAGES;
    uint64_t* const done = empty + C::STAGES;      // every MMA of this CTA has completed
    uint64_t* const drained = done + 1;            // those of a CTA that gave up have
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
    uint32_t* const s_ok = tmem_slot + 1;          // this CTA's partial sums are all there

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t S = cluster_nctarank(), rank = cluster_ctarank();
    const int tile = blockIdx.x / S;
    const int n0 = tile % p.n_tiles * 128, m0 = tile / p.n_tiles * TN;
    // this CTA's 128-byte blocks of K (at least one: S is no more than there are)
    const int blocks = (p.K + 127) / 128;
    const int kb0 = static_cast<int>((long long)blocks * rank / S), kb1 = static_cast<int>((long long)blocks * (rank + 1) / S);

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(done, 1);
        mbar_init(drained, 1);
        *s_ok = 1u;
        fence_barrier_init();
        tma_prefetch_desc(&tmA);
        tma_prefetch_desc(&tmW);
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, C::TMEM_COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    if (threadIdx.x == 0) griddep_launch();

    // the epilogue: this thread's channel, its group's share of a tile's or a rank's tokens
    const int n_in = (warp & 3) * 32 + lane, n = n0 + n_in, grp = (warp - 2) >> 2;
    const int tokens = p.M - m0 < TN ? p.M - m0 : TN;
    const bool in = n < p.N;
    float cs = 0.f, bias = 0.f;
    bool ok = true;
    TO* const c = static_cast<TO*>(p.C) + (size_t)m0 * p.ldc + n;
    // the outputs of tokens t and u from their accumulators; a token outside [0, end) is computed and not stored
    const auto put2 = [&](int acc_t, int t, int acc_u, int u, int end) {
        float2 v = make_float2(i8_value(acc_t, s_rowscale[t], cs, bias), i8_value(acc_u, s_rowscale[u], cs, bias));
        if constexpr (EPI == kEpiBiasGelu) v = gelu_pair<false, true>(pk2(v.x, v.y), GeluK(1.0f));
        TO *ct = c + (size_t)t * p.ldc, *cu = c + (size_t)u * p.ldc;
        if constexpr (EPI == kEpiResidual) {   // added at L2, once an element: nothing waits for the old value
            if (t < end) atomicAdd(ct, v.x);
            if (u < end) atomicAdd(cu, v.y);
        } else {
            if (t < end) *ct = from_f32<TO>(v.x);
            if (u < end) *cu = from_f32<TO>(v.y);
        }
    };
    int* const part = reinterpret_cast<int*>(sW);                  // [tokens][128] partial sums

    if (warp == 0) {
        if (lane == 0) {
            griddep_wait();
            int stage = 0;
            uint32_t phase = 0;
            int kb = kb0;
            for (; kb < (p.stall && rank == S - 1 ? kb0 : kb1); ++kb) {
                if (!mbar_wait(&empty[stage], phase ^ 1u, err, kErrSmemEmpty)) break;
                mbar_arrive_expect_tx(&full[stage], C::STAGE_BYTES);
                tma_load_2d(sW + stage * C::W_BYTES, &tmW, &full[stage], kb * 128, n0);
                tma_load_2d(sA + stage * C::A_BYTES, &tmA, &full[stage], kb * 128, m0);
                if (++stage == C::STAGES) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
            // every copy that was started has landed before the CTA can leave: the last ones, stage by stage
            const int issued = kb - kb0;
            for (int i = issued > C::STAGES ? issued - C::STAGES : 0; i < issued; ++i)
                mbar_wait(&full[i % C::STAGES], (i / C::STAGES) & 1, err, kErrTmaFull);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t idesc = idesc_i8(128, TN);
            int stage = 0;
            uint32_t phase = 0;
            int kb = kb0;
            for (; kb < kb1; ++kb) {
                if (!mbar_wait(&full[stage], phase, err, kErrTmaFull)) break;
                tc_fence_after();
                const uint32_t w = smem_u32(sW + stage * C::W_BYTES), a = smem_u32(sA + stage * C::A_BYTES);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    umma_i8(tmem, sdesc_sw128(w + 32u * k), sdesc_sw128(a + 32u * k), idesc,
                            kb != kb0 || k != 0 ? 1u : 0u);
                umma_commit(&empty[stage]);
                if (++stage == C::STAGES) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
            // a sum that stopped short is never called done: the epilogue's wait runs out too
            uint64_t* const end = kb == kb1 ? done : drained;
            umma_commit(end);
            mbar_wait(end, 0, err, kErrTmemFull);
        }
    } else {
        griddep_wait();
        const int e = threadIdx.x - 64;
        if (e < TN) s_rowscale[e] = e < tokens ? __ldg(p.rowscale + m0 + e) : 0.f;
        if (in) {
            cs = __ldg(p.colscale + n);
            if (p.bias) bias = __ldg(p.bias + n);
        }
        named_barrier(1, 128 * C::GROUPS);
        ok = __all_sync(0xffffffffu, mbar_wait(done, 0, err, kErrTmemFull));
        if (!ok) *s_ok = 0u;
        tc_fence_after();
        constexpr int SHARE = TN / C::GROUPS, LD = SHARE < 16 ? SHARE : 16;
        const uint32_t t_lane = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
#pragma unroll 1
        for (int t0 = grp * SHARE; ok && t0 < (grp + 1) * SHARE && t0 < tokens; t0 += LD) {
            uint32_t a[LD];
            if constexpr (LD == 4) tmem_ld_32x32b_x4(t_lane + static_cast<uint32_t>(t0), a);
            else if constexpr (LD == 8) tmem_ld_32x32b_x8(t_lane + static_cast<uint32_t>(t0), a);
            else tmem_ld_32x32b_x16(t_lane + static_cast<uint32_t>(t0), a);
            tmem_ld_wait(a);
            if (S > 1) {
#pragma unroll
                for (int i = 0; i < LD; ++i) part[(t0 + i) * 128 + n_in] = static_cast<int>(a[i]);
            } else if (in) {
#pragma unroll
                for (int i = 0; i < LD; i += 2)
                    put2(static_cast<int>(a[i]), t0 + i, static_cast<int>(a[i + 1]), t0 + i + 1, tokens);
            }
        }
    }

    __syncwarp();
    if (S > 1) {
        cluster_sync();            // every CTA's partial sums are written
        // this CTA's share of the tokens, its groups' tokens neighbouring pairs
        const int ta = static_cast<int>(tokens * rank / S), tb = static_cast<int>(tokens * (rank + 1) / S);
        if (warp >= 2) {
            // A sum that lacks a CTA's part is not stored: lane r reads whether CTA r's is there, the sums' own loads
            // under way (16 x 8,192 x 8,192 9.62 us, 9.54 without; every lane reading all words before them 9.84).
            const uint32_t there = lane < static_cast<int>(S) ? ld_cluster(mapa_shared(smem_u32(s_ok), lane)) : 1u;
            const uint32_t mine = smem_u32(part) + 4u * static_cast<uint32_t>(n_in);
            for (int t = ta + 2 * grp; t < tb; t += 2 * C::GROUPS) {
                const int u = t + 1 < TN ? t + 1 : t;     // in the buffer, if not in the share
                int x = 0, y = 0;
#pragma unroll
                for (uint32_t r = 0; r < 8; ++r) {
                    if (r < S) {
                        const uint32_t from = mapa_shared(mine, r);
                        x += static_cast<int>(ld_cluster(from + 512u * static_cast<uint32_t>(t)));
                        y += static_cast<int>(ld_cluster(from + 512u * static_cast<uint32_t>(u)));
                    }
                }
                const bool all = __all_sync(0xffffffffu, there);
                if (in) put2(x, t, y, t + 1, all ? tb : 0);
            }
        }
        __syncwarp();
        cluster_sync();            // no CTA reads another's shared memory any more
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_dealloc(tmem, C::TMEM_COLS);
}

}  // namespace mf
