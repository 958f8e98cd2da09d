// qtts_int8.hip - the 8-bit integer path: rows quantised with one scale each (alone, or behind the residual addition and
// RMSNorm), int8 weight packing, and the product of int8 rows with int8 weights on the int8 matrix instructions, plain
// or with the SwiGLU epilogue.  An extension: the reference has bf16 only.
//
//   s_m = max(max_k |y_mk| / 127, 2^-126)      q_mk = rint(y_mk / s_m)            |q| <= 127      (quotients in fp32)
//   out_mn = bf16(xs_m * ws_n * sum_k q_mk w_nk [+ bias_n] [+ residual_mn])
//
// The sum is exact: |q w| <= 2^14, so int32 holds K <= 131071 of them whatever the order of the additions - the same
// result for every tile shape and every split of K, which is why the launch is free to choose both by speed alone.
// Everything after the sum is fp32 with one rounding to bf16 at the store.
#include "qtts_common.h"
#include <type_traits>

typedef int int4_t __attribute__((ext_vector_type(4)));

static constexpr int I8_MAX_K = 131071;            // int32 holds the sum of this many products of two int8 values
static constexpr int I8_MAX_ROWS = 0x7f800000;     // row numbers a launch's rounding up passes still fit an int
static constexpr int I8_MAX_N = 0x3ffffff;
static constexpr float I8_TINY = 0x1p-126f;        // smallest scale: its reciprocal is finite, rows of zeros stay zeros

__host__ __device__ static inline int ceil_div(int a, int b) { return (a - 1) / b + 1; }       // a, b > 0

// ------------------------------------------------------------------ rows -> int8
struct RowsI8Args {
    const bf16_t *x; int ldx;
    const bf16_t *delta; int ldd;
    const bf16_t *w; float eps;
    bf16_t *sum; int lds;
    int8_t *q; int ldq;
    float *scales;
    int M, K;
};

// bf16 rows may start anywhere: the hardware takes 16- and 8-byte requests at any address, and these types say so.
typedef u32x4_t u32x4_any __attribute__((aligned(2)));
typedef unsigned int u32x2_t __attribute__((ext_vector_type(2)));
typedef u32x2_t u32x2_any __attribute__((aligned(2)));

// 8 columns from k0 on of a row; columns behind the last are zeros.
__device__ __forceinline__ uint4 load8(const bf16_t *row, int k0, int K) {
    Frag f;
    if (k0 + 8 <= K) f.n = *reinterpret_cast<const u32x4_any *>(row + k0);
    else {
#pragma unroll
        for (int j = 0; j < 8; ++j) f.h[j] = k0 + j < K ? row[k0 + j] : (bf16_t)0;
    }
    return f.u;
}
__device__ __forceinline__ void store8(bf16_t *row, int k0, int K, uint4 v) {
    Frag f;
    f.u = v;
    if (k0 + 8 <= K) { *reinterpret_cast<u32x4_any *>(row + k0) = f.n; return; }
#pragma unroll
    for (int j = 0; j < 8; ++j) if (k0 + j < K) row[k0 + j] = f.h[j];
}

// Four values of at most 127.5 in magnitude, rounded to the nearest integer (ties to even) and packed: 1.5 * 2^23 + v has
// the integer in its low bits, in two's complement.
__device__ __forceinline__ uint32_t pack4_i8(float a, float b, float c, float d) {
    const float magic = 12582912.0f;
    const uint32_t ua = __float_as_uint(a + magic), ub = __float_as_uint(b + magic);
    const uint32_t uc = __float_as_uint(c + magic), ud = __float_as_uint(d + magic);
    const uint32_t lo = __builtin_amdgcn_perm(ub, ua, 0x0c0c0400), hi = __builtin_amdgcn_perm(ud, uc, 0x0c0c0400);
    return lo | (hi << 16);
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    v = max(v, dpp_u32<0xB1>(v));          // as row16_sum
    v = max(v, dpp_u32<0x4E>(v));
    v = max(v, dpp_u32<0x141>(v));
    v = max(v, dpp_u32<0x140>(v));
    v = max(v, (uint32_t)__shfl_xor((int)v, 16));
    return max(v, (uint32_t)__shfl_xor((int)v, 32));
}
// The largest magnitude of eight values and top; a NaN is larger than every number and stays.
__device__ __forceinline__ float magnitude(float top, const float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; j += 2)
        top = __builtin_elementwise_maximum(__builtin_elementwise_maximum(__builtin_fabsf(v[j]), __builtin_fabsf(v[j + 1])), top);
    return top;
}
// A row's scale from the bits of its largest magnitude.  NaN and infinity stay: the whole row then stands for NaN.
__device__ __forceinline__ float i8_scale(uint32_t top) {
    const float s = __uint_as_float(top) / 127.0f;
    return s < I8_TINY ? I8_TINY : s;
}
// a / b in fp32 with inv, the reciprocal of b rounded to nearest: the product is off by 1.5 units in the last place at most, and
// the step of Markstein (IBM J. Res. Dev. 34, 1990) adds what is left of a, which a fused multiply-add gives (nearly) without
// error.  For bf16 a and b = RN(bf16 / 127) >= 2^-100, all there is to quantising bf16 rows, it is the rounded quotient for every
// pair of mantissas; otherwise it is that but for last bits decided by less than 2^-22 of a unit.  The product alone puts
// 127 * (1/2), the half of a row's maximum, on the other side of 63.5 for some maxima.
__device__ __forceinline__ float quotient(float a, float b, float inv) {
    const float q = a * inv;
    return __builtin_fmaf(__builtin_fmaf(-q, b, a), inv, q);
}
// What a row's values are divided by, with its reciprocal.  Rows that are not finite stand for zeros, and with a very small scale
// up keeps what is left of a value a normal number: both are rare, the same in the whole wave, and behind one scalar branch.
struct I8Div { float s, inv, up; bool rare; };
__device__ __forceinline__ I8Div i8_div(uint32_t top, float s) {
    I8Div d;
    d.up = top >= 0x7f800000u ? 0.f : s < 0x1p-100f ? 0x1p100f : 1.0f;
    d.s = d.up == 0.f ? 1.0f : s * d.up;
    d.inv = 1.0f / d.s;
    d.rare = __builtin_amdgcn_readfirstlane(__float_as_uint(d.up)) != 0x3f800000u;
    return d;
}
// RMSNorm's h / root * w with rstd = 1 / root.  The root is infinite where the mean is: h / root is 0 then (NaN for an infinite h).
__device__ __forceinline__ float i8_normed(float h, float root, float rstd, float w) { return quotient(h, root, rstd) * w; }
__device__ __forceinline__ float i8_root(float mean_eps, float &rstd) {
    const float root = sqrtf(mean_eps);
    rstd = 1.0f / root;
    return rstd == 0.f ? 0.f : root;
}
// Eight columns from k0 on.
__device__ __forceinline__ void store8_i8(int8_t *row, int k0, int K, float (&v)[8], const I8Div &d) {
    if (d.rare) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = d.up != 0.f ? v[j] * d.up : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = quotient(v[j], d.s, d.inv);
    const uint2 p = make_uint2(pack4_i8(v[0], v[1], v[2], v[3]), pack4_i8(v[4], v[5], v[6], v[7]));
    if (k0 + 8 <= K) *reinterpret_cast<uint2 *>(row + k0) = p;
    else
        for (int j = 0; j < K - k0; ++j) row[k0 + j] = (int8_t)((j < 4 ? p.x >> (8 * j) : p.y >> (8 * (j - 4))) & 0xff);
}

// A row per T = 64 * W threads, R rows a workgroup; thread t of a row holds the 8-column chunks t, t + T, ... (CH of them) as
// bf16 across both reductions, so x, delta and the weights are read once and nothing is read back.  All of a thread's
// requests go out before its first store: sum may be x or delta, and a load behind a store that may alias waits for it.
// Few rows are bound by the chain request - sum of squares - maximum - store (8 rows of 2048 with delta 3.2 us, an empty launch
// 2.3), many by memory and, without delta, by arithmetic too: 16384 x 2048 with delta 39.5 us, 5.9 TB/s (a large copy reaches
// 4.9-5.4), without 24.3 us, 4.1 TB/s (23.0 with products in the quotients' place); 8192 x 6144 quantised alone 26.7 us, 5.7 TB/s.
template <int W, int R, int CH, bool NORM>
__global__ __launch_bounds__(W * R * 64) void rows_int8_kernel(RowsI8Args a) {
    constexpr int T = W * 64;
    static_assert(W == 1 || R == 1, "one row a workgroup, or one wave a row");
    __shared__ float red_f[W * CH];
    __shared__ uint32_t red_u[W];
    const int t = threadIdx.x % T;
    for (int m = blockIdx.x * R + threadIdx.x / T; m < a.M; m += gridDim.x * R) {
        const bf16_t *xr = a.x + (size_t)m * a.ldx;
        const uint4 zero = make_uint4(0, 0, 0, 0);
        Frag h[CH], wv[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int k0 = (c * T + t) * 8;
            h[c].u = k0 < a.K ? load8(xr, k0, a.K) : zero;
        }
        if (NORM) {
            Frag d[CH];
            if (a.delta) {
                const bf16_t *dr = a.delta + (size_t)m * a.ldd;
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    const int k0 = (c * T + t) * 8;
                    d[c].u = k0 < a.K ? load8(dr, k0, a.K) : zero;
                }
            }
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int k0 = (c * T + t) * 8;
                wv[c].u = k0 < a.K ? load8(a.w, k0, a.K) : zero;
            }
            if (a.delta) {
                bf16_t *sr = a.sum + (size_t)m * a.lds;
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    const int k0 = (c * T + t) * 8;
#pragma unroll
                    for (int j = 0; j < 8; ++j) h[c].h[j] = f2bf(bf2f(h[c].h[j]) + bf2f(d[c].h[j]));
                    if (k0 < a.K) store8(sr, k0, a.K, h[c].u);
                }
            }
        }
        float root = 1.0f, rstd = 1.0f;
        if (NORM) {
            // Squares are added up per 512 columns (a chunk's 8, then the 64 lanes of a wave), then in the order of the columns:
            // the same sum, and the same row, whatever number of threads the launch chose.
            float part[CH], ss = 0.f;
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                part[c] = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) { const float v = bf2f(h[c].h[j]); part[c] = __builtin_fmaf(v, v, part[c]); }
                part[c] = row16_sum(part[c]);
                part[c] += __shfl_xor(part[c], 16);
                part[c] += __shfl_xor(part[c], 32);
            }
            if (W > 1) {
                if ((t & 63) == 0) {
#pragma unroll
                    for (int c = 0; c < CH; ++c) red_f[c * W + (t >> 6)] = part[c];
                }
                __syncthreads();
#pragma unroll
                for (int i = 0; i < W * CH; ++i) ss += red_f[i];
            } else {
#pragma unroll
                for (int c = 0; c < CH; ++c) ss += part[c];
            }
            root = i8_root(ss / (float)a.K + a.eps, rstd);
        }
        // across lanes the maximum is one of integers, over the numbers' bits: a NaN is above every number and stays.  Columns
        // behind the last are zeros (not where the root is 0 or NaN: then the row is not finite whatever they are)
        float largest = 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[j] = bf2f(h[c].h[j]);
                if (NORM) v[j] = i8_normed(v[j], root, rstd, bf2f(wv[c].h[j]));
            }
            largest = magnitude(largest, v);
        }
        uint32_t top = __float_as_uint(largest) & 0x7fffffffu;
        top = wave_max(top);
        if (W > 1) {
            if ((t & 63) == 0) red_u[t >> 6] = top;
            __syncthreads();
            top = 0;
#pragma unroll
            for (int i = 0; i < W; ++i) top = max(top, red_u[i]);
            if (m + gridDim.x < (unsigned)a.M) __syncthreads();      // the next row writes red_* again
        }
        const float s = i8_scale(top);
        const I8Div by = i8_div(top, s);
        if (t == 0) a.scales[m] = s;
        int8_t *qr = a.q + (size_t)m * a.ldq;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int k0 = (c * T + t) * 8;
            if (k0 >= a.K) continue;
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[j] = bf2f(h[c].h[j]);
                if (NORM) v[j] = i8_normed(v[j], root, rstd, bf2f(wv[c].h[j]));
            }
            store8_i8(qr, k0, a.K, v, by);
        }
    }
}

// Rows too long for registers: three walks over the row, the second and third of them out of L2 - h is read back from where
// the first walk wrote it (sum), or from x.  Bound by those walks' latencies, a workgroup a row: 300 rows of 40000 columns 12 us
// quantised, 32 us with norm and delta (floor 9 and 18 with the launch; the form above, whose chunks such rows push out of the registers: 94 us).
template <bool NORM>
__global__ __launch_bounds__(1024) void rows_int8_long_kernel(RowsI8Args a) {
    __shared__ float red_f[16];
    __shared__ uint32_t red_u[16];
    const int t = threadIdx.x;
    for (int m = blockIdx.x; m < a.M; m += gridDim.x) {
        const bf16_t *xr = a.x + (size_t)m * a.ldx, *hr = xr;
        float root = 1.0f, rstd = 1.0f;
        if (NORM) {
            float ss = 0.f;
            const bf16_t *dr = a.delta ? a.delta + (size_t)m * a.ldd : nullptr;
            bf16_t *sr = a.delta ? a.sum + (size_t)m * a.lds : nullptr;
#pragma unroll 2
            for (int k0 = t * 8; k0 < a.K; k0 += 8192) {
                Frag h, d;
                h.u = load8(xr, k0, a.K);
                if (dr) {
                    d.u = load8(dr, k0, a.K);
#pragma unroll
                    for (int j = 0; j < 8; ++j) h.h[j] = f2bf(bf2f(h.h[j]) + bf2f(d.h[j]));
                    store8(sr, k0, a.K, h.u);
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) { const float v = bf2f(h.h[j]); ss += v * v; }
            }
            if (dr) hr = sr;
            ss = row16_sum(ss);
            ss += __shfl_xor(ss, 16);
            ss += __shfl_xor(ss, 32);
            if ((t & 63) == 0) red_f[t >> 6] = ss;
            __syncthreads();
            ss = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) ss += red_f[i];
            root = i8_root(ss / (float)a.K + a.eps, rstd);
        }
        auto chunk = [&](int k0, float (&v)[8]) {
            Frag h, w;
            h.u = load8(hr, k0, a.K);
            if (NORM) w.u = load8(a.w, k0, a.K);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[j] = bf2f(h.h[j]);
                if (NORM) v[j] = i8_normed(v[j], root, rstd, bf2f(w.h[j]));
            }
        };
        float largest = 0.f;
#pragma unroll 4
        for (int k0 = t * 8; k0 < a.K; k0 += 8192) {
            float v[8];
            chunk(k0, v);
            largest = magnitude(largest, v);
        }
        uint32_t top = wave_max(__float_as_uint(largest) & 0x7fffffffu);
        if ((t & 63) == 0) red_u[t >> 6] = top;
        __syncthreads();
        top = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) top = max(top, red_u[i]);
        if (m + gridDim.x < (unsigned)a.M) __syncthreads();          // the next row writes red_* again
        const float s = i8_scale(top);
        const I8Div by = i8_div(top, s);
        if (t == 0) a.scales[m] = s;
        int8_t *qr = a.q + (size_t)m * a.ldq;
#pragma unroll 4
        for (int k0 = t * 8; k0 < a.K; k0 += 8192) {
            float v[8];
            chunk(k0, v);
            store8_i8(qr, k0, a.K, v, by);
        }
    }
}

// Threads per row.  Few rows: as many as leave a chunk or two each, the launch is a chain of latencies (8 rows of 6144, with
// delta: 3.9 us with 512 threads, 4.5 with 256).  Many rows: fewer waves a row and more rows in flight (8192 rows of 6144 with
// delta: 67 us, 5.3 TB/s, with 256 threads, 72 with 512; 16384 of 2048: 39.4 us with 128, 41.8 with 256, 56 with 512; 16384 of
// 256: 9.9 us with a wave, 14 with 128 threads, 23 with 256).
template <bool NORM>
static void launch_rows_int8(const RowsI8Args &a, hipStream_t s) {
#define QTTS_ROWS_I8(W, R, CH, WHEN) if (a.K <= W * 64 * 8 * CH && (WHEN)) { \
        const dim3 grid(std::min(ceil_div(a.M, R), 1 << 20));       /* rows beyond that in turns: a launch takes fewer than 2^32 threads */ \
        hipLaunchKernelGGL((rows_int8_kernel<W, R, CH, NORM>), grid, dim3(W * R * 64), 0, s, a); return; }
    QTTS_ROWS_I8(1, 4, 1, true)              // up to 512 columns
    QTTS_ROWS_I8(2, 1, 1, true)              // 1024
    QTTS_ROWS_I8(2, 1, 2, a.M >= 4096)       // 2048
    QTTS_ROWS_I8(4, 1, 1, true)
    QTTS_ROWS_I8(4, 1, 2, a.M >= 2048)       // 4096
    QTTS_ROWS_I8(8, 1, 1, true)
    QTTS_ROWS_I8(4, 1, 3, a.M >= 2048)       // 6144
    QTTS_ROWS_I8(8, 1, 2, true)              // 8192
    QTTS_ROWS_I8(16, 1, 2, true)             // 16384
    hipLaunchKernelGGL((rows_int8_long_kernel<NORM>), dim3(std::min(a.M, 1 << 20)), dim3(1024), 0, s, a);
#undef QTTS_ROWS_I8
}

extern "C" int qtts_quantize_int8(const void *x, int ldx, void *q, int ldq, float *scales, int M, int K, qtts_stream_t stream) {
    QCHECK(x && q && scales, "quantize_int8: null pointer");
    QCHECK(M > 0 && M <= I8_MAX_ROWS && K > 0 && K <= I8_MAX_K, "quantize_int8: bad shape M=%d K=%d (M <= %d, K <= %d)", M, K, I8_MAX_ROWS, I8_MAX_K);
    QCHECK(ldx >= K && ldq >= K && ldq % 16 == 0, "quantize_int8: row strides ldx=%d ldq=%d (need ldx >= K, ldq >= K, ldq %% 16 == 0)", ldx, ldq);
    QCHECK(((uintptr_t)x & 1) == 0 && ((uintptr_t)q & 15) == 0 && ((uintptr_t)scales & 3) == 0, "quantize_int8: misaligned pointer");
    RowsI8Args a{};
    a.x = (const bf16_t *)x; a.ldx = ldx; a.q = (int8_t *)q; a.ldq = ldq; a.scales = scales; a.M = M; a.K = K;
    launch_rows_int8<false>(a, (hipStream_t)stream);
    QLAUNCH();
    return QTTS_OK;
}

extern "C" int qtts_rmsnorm_int8(const void *x, int ldx, const void *delta, int ldd, const void *w, float eps, void *sum, int lds,
                                 void *q, int ldq, float *scales, int M, int H, qtts_stream_t stream) {
    QCHECK(x && w && q && scales, "rmsnorm_int8: null pointer");
    QCHECK(!delta == !sum, "rmsnorm_int8: delta and sum come together");
    QCHECK(M > 0 && M <= I8_MAX_ROWS && H > 0 && H <= I8_MAX_K, "rmsnorm_int8: bad shape M=%d H=%d (M <= %d, H <= %d)", M, H, I8_MAX_ROWS, I8_MAX_K);
    QCHECK(ldx >= H && ldq >= H && ldq % 16 == 0 && (!delta || (ldd >= H && lds >= H)),
           "rmsnorm_int8: row strides ldx=%d ldd=%d lds=%d ldq=%d (need >= H, ldq %% 16 == 0)", ldx, ldd, lds, ldq);
    QCHECK((sum != x || lds == ldx) && (!sum || sum != delta || lds == ldd), "rmsnorm_int8: sum in the place of x or delta needs its row stride");
    QCHECK((((uintptr_t)x | (uintptr_t)delta | (uintptr_t)w | (uintptr_t)sum) & 1) == 0 && ((uintptr_t)q & 15) == 0 &&
           ((uintptr_t)scales & 3) == 0, "rmsnorm_int8: misaligned pointer");
    RowsI8Args a{};
    a.x = (const bf16_t *)x; a.ldx = ldx; a.delta = (const bf16_t *)delta; a.ldd = ldd; a.w = (const bf16_t *)w; a.eps = eps;
    a.sum = (bf16_t *)sum; a.lds = lds; a.q = (int8_t *)q; a.ldq = ldq; a.scales = scales; a.M = M; a.K = H;
    launch_rows_int8<true>(a, (hipStream_t)stream);
    QLAUNCH();
    return QTTS_OK;
}

// ------------------------------------------------------------------ weight packing
// Once per weight, at load time: a byte at a time is fast enough (bound by those loads).
// packed[tile][k-step][lane][16 B]: lane (g, r) of k-step ks holds row 16 * tile + r, columns 64 * ks + 16 * g .. +16 - the
// 16 bytes a lane feeds to v_mfma_i32_16x16x64_i8.  Rows and columns behind the last are zeros; k-steps come in pairs.
// gate/up: the tile's packed row 4 * p + j holds output i = 8 * tile + 2 * p + (j & 1), gate for j < 2 and up for j >= 2: a
// lane's four sums are two gates and the two ups of the same outputs, and the epilogue needs no other lane.
static inline int i8_ksteps(int K) { return 2 * ceil_div(K, 128); }

__global__ __launch_bounds__(256) void pack_int8_kernel(const int8_t *__restrict__ w, const int8_t *__restrict__ up, int ldw,
                                                        uint4 *__restrict__ packed, int N, int K, int ksteps, size_t total) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (size_t)gridDim.x * 256) {
        const int lane = i & 63;
        const size_t rest = i >> 6;
        const int ks = (int)(rest % ksteps), tile = (int)(rest / ksteps), r = lane & 15, k0 = 64 * ks + 16 * (lane >> 4);
        const int n = up ? 8 * tile + 2 * (r >> 2) + (r & 1) : 16 * tile + r;
        const int8_t *src = (up && (r & 2) ? up : w) + (size_t)n * ldw;
        union { uint4 u; int8_t b[16]; } v;
        v.u = make_uint4(0, 0, 0, 0);
        if (n < N)
            for (int j = 0; j < 16; ++j) if (k0 + j < K) v.b[j] = src[k0 + j];
        packed[i] = v.u;
    }
}

extern "C" size_t qtts_packed_weight_int8_bytes(int N, int K) {
    if (N <= 0 || K <= 0 || N > I8_MAX_N || K > I8_MAX_K) return 0;
    return (size_t)ceil_div(N, 16) * i8_ksteps(K) * 1024;
}
extern "C" size_t qtts_packed_gate_up_int8_bytes(int I, int K) {
    if (I <= 0 || K <= 0 || I > I8_MAX_N || K > I8_MAX_K) return 0;
    return (size_t)ceil_div(I, 8) * i8_ksteps(K) * 1024;
}

static int pack_int8(const char *who, const void *w, const void *up, int ldw, void *packed, int N, int K, hipStream_t s) {
    QCHECK(N > 0 && N <= I8_MAX_N && K > 0 && K <= I8_MAX_K && ldw >= K, "%s: bad shape N=%d K=%d ldw=%d (N <= %d, K <= %d)", who, N, K, ldw, I8_MAX_N, I8_MAX_K);
    QCHECK(((uintptr_t)packed & 15) == 0, "%s: misaligned pointer", who);
    const size_t total = (size_t)ceil_div(N, up ? 8 : 16) * i8_ksteps(K) * 64;
    hipLaunchKernelGGL(pack_int8_kernel, dim3((unsigned)std::min<size_t>((total + 255) / 256, 1 << 20)), dim3(256), 0, s,
                       (const int8_t *)w, (const int8_t *)up, ldw, (uint4 *)packed, N, K, i8_ksteps(K), total);
    QLAUNCH();
    return QTTS_OK;
}
extern "C" int qtts_pack_weight_int8(const void *w, int ldw, void *packed, int N, int K, qtts_stream_t stream) {
    QCHECK(w && packed, "pack_weight_int8: null pointer");
    return pack_int8("pack_weight_int8", w, nullptr, ldw, packed, N, K, (hipStream_t)stream);
}
extern "C" int qtts_pack_gate_up_int8(const void *gate, const void *up, int ldw, void *packed, int I, int K, qtts_stream_t stream) {
    QCHECK(gate && up && packed, "pack_gate_up_int8: null pointer");
    return pack_int8("pack_gate_up_int8", gate, up, ldw, packed, I, K, (hipStream_t)stream);
}

// ------------------------------------------------------------------ the product
struct LinI8Args {
    const int8_t *x; int ldx;
    const float *xs;
    const uint4 *wp;
    const float *ws, *us;          // scales per output channel; SwiGLU: of the gate and the up rows
    const bf16_t *bias, *res; int ldr;
    bf16_t *out; int ldo;
    int M, N, K, ksteps;           // N: output columns; ksteps: of a packed tile
};

// What follows a sum, in the same operations in every kernel: a row's result does not depend on the form it came from.  A sum
// is below 2^31, so times a row scale of 2^96 or more it might pass fp32's range although the result does not: the channel's
// scale comes first then, and passes the range only with the result.  (Not for NaN, which stays in either order.)
struct I8Scale { float row; bool later; };
__device__ __forceinline__ I8Scale i8_row_scale(float xs) { return {xs, __builtin_fabsf(xs) >= 0x1p96f}; }
__device__ __forceinline__ float i8_scaled(int acc, I8Scale x, float ws, float bias) {
    return __builtin_fmaf((float)acc * (x.later ? ws : x.row), x.later ? x.row : ws, bias);
}
__device__ __forceinline__ float i8_swiglu(int g, int u, I8Scale x, float gs, float us) {
    const float gate = (float)g * (x.later ? gs : x.row) * (x.later ? x.row : gs);
    return silu_f(gate) * ((float)u * (x.later ? us : x.row) * (x.later ? x.row : us));
}

// One 16 x 16 tile of sums, this lane's four of them: weight rows 4 * (lane / 16) .. +3 of `tile`, activation row m.
template <bool SWIGLU>
__device__ __forceinline__ void i8_store(const LinI8Args &a, int4_t acc, int tile, int m, int lane) {
    if (m >= a.M) return;
    const I8Scale xs = i8_row_scale(a.xs[m]);
    bf16_t *o = a.out + (size_t)m * a.ldo;
    if (SWIGLU) {
        const int n = 8 * tile + 2 * (lane >> 4);
        float y[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int nn = min(n + j, a.N - 1);
            y[j] = i8_swiglu(acc[j], acc[2 + j], xs, a.ws[nn], a.us[nn]);
        }
        for (int j = 0; j < 2; ++j) if (n + j < a.N) o[n + j] = f2bf(y[j]);
        return;
    }
    const int n = 16 * tile + 4 * (lane >> 4);
    float y[4];
    const bool full = n + 4 <= a.N;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int nn = min(n + j, a.N - 1);
        y[j] = i8_scaled(acc[j], xs, a.ws[nn], a.bias ? bf2f(a.bias[nn]) : 0.f);
    }
    if (a.res) {
        const bf16_t *rr = a.res + (size_t)m * a.ldr;
        if (full) {
            const u32x2_t r = *reinterpret_cast<const u32x2_any *>(rr + n);
            float p, q;
            unpack2(r[0], p, q); y[0] += p; y[1] += q;
            unpack2(r[1], p, q); y[2] += p; y[3] += q;
        } else
            for (int j = 0; j < 4; ++j) y[j] += bf2f(rr[min(n + j, a.N - 1)]);
    }
    if (full) *reinterpret_cast<u32x2_any *>(o + n) = u32x2_t{pack2v(float2_t{y[0], y[1]}), pack2v(float2_t{y[2], y[3]})};
    else
        for (int j = 0; j < 4; ++j) if (n + j < a.N) o[n + j] = f2bf(y[j]);
}

union I8Frag { uint4 u; int4_t v; };

// Few rows: a workgroup owns TM row tiles x TN weight tiles and its NW waves share K, each wave a contiguous run of
// k-steps straight from memory to registers; the waves' sums meet in LDS.  U k-steps are requested at a time, the next U
// before the current are multiplied.  Every weight byte is used 16 TM times at most, so what bounds it is weights coming in:
// the launch and one latency (1 row x 4096 x 2048: 3.8 us), then the 40-60 GB/s a CU takes of row-major activations and
// weights together (16 x 2048 x 6144 with residual 7.6 us; SwiGLU 8 x 6144 x 2048 6.9 us, 3.6 TB/s).  Sixteen waves a
// workgroup, or the epilogue's scales requested in front of the loop, are no faster.
template <int TM, int TN, int NW, int U, bool SWIGLU>
__global__ __launch_bounds__(NW * 64) void linear_int8_split_kernel(LinI8Args a) {
    __shared__ int4_t red[NW][TM * TN][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int tiles = SWIGLU ? ceil_div(a.N, 8) : ceil_div(a.N, 16);
    const int t0 = blockIdx.x * TN, m0 = blockIdx.y * TM * 16;
    const int steps = ceil_div(a.K, 64), per = ceil_div(steps, NW), ks0 = min(steps, wave * per), n = min(steps, ks0 + per) - ks0;
    const int8_t *xp[TM];
    const uint4 *wp[TN];
#pragma unroll
    for (int i = 0; i < TM; ++i) xp[i] = a.x + (size_t)min(m0 + 16 * i + r, a.M - 1) * a.ldx;
#pragma unroll
    for (int i = 0; i < TN; ++i) wp[i] = a.wp + (size_t)min(t0 + i, tiles - 1) * a.ksteps * 64 + lane;
    int4_t acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = int4_t{0, 0, 0, 0};
    struct Batch { I8Frag x[U][TM], w[U][TN]; } b0, b1;
    auto request = [&](Batch &b, int at) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int ks = ks0 + min(at + u, n - 1);                                // behind the run: its last step again, not multiplied
            const int k = 64 * ks + 16 * g, kk = k < a.K ? k : 0;                    // behind the last column the packed weights are zeros
#pragma unroll
            for (int i = 0; i < TM; ++i) b.x[u][i].u = *reinterpret_cast<const uint4 *>(xp[i] + kk);
#pragma unroll
            for (int i = 0; i < TN; ++i) b.w[u][i].u = wp[i][(size_t)ks * 64];
        }
    };
    auto multiply = [&](const Batch &b, int at) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (at + u >= n) break;
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(b.w[u][j].v, b.x[u][i].v, acc[i][j], 0, 0, 0);
        }
    };
    if (n > 0) {
        request(b0, 0);
        for (int at = 0; at < n; at += 2 * U) {
            if (at + U < n) request(b1, at + U);
            multiply(b0, at);
            if (at + U >= n) break;
            if (at + 2 * U < n) request(b0, at + 2 * U);
            multiply(b1, at + U);
        }
    }
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) red[wave][i * TN + j][lane] = acc[i][j];
    __syncthreads();
    for (int t = wave; t < TM * TN; t += NW) {
        int4_t part[NW], sum = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < NW; ++w) part[w] = red[w][t][lane];
#pragma unroll
        for (int w = 0; w < NW; ++w) sum += part[w];
        if (t0 + t % TN < tiles) i8_store<SWIGLU>(a, sum, t0 + t % TN, m0 + 16 * (t / TN) + r, lane);
    }
}

// Few rows and few columns: 8 rows and half a packed tile a workgroup, so that twice as many CUs take part.  An instruction takes
// two k-steps: its weight rows 0-7 and activation rows 0-7 are a step's, 8-15 the same rows of the next; of the four quarters
// of its sums two are wanted, and added up.  Bound by latency, then by what a CU takes in: 8 x 2048 x 6144 5.6 us (6.2 in
// whole tiles, whose activations are requested for 16 rows), 8 x 512 x 8192 5.0 us (5.8), 16 x 512 x 8192 5.1 us (7.0); 16 rows
// of whole steps to half a tile, other U (1, 3, 4) and four or sixteen waves are slower on most shapes.
template <int NW, int U, bool SWIGLU>
__global__ __launch_bounds__(NW * 64) void linear_int8_half_kernel(LinI8Args a) {
    __shared__ int4_t red[NW][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int tile = blockIdx.x >> 1, half = blockIdx.x & 1, m = blockIdx.y * 8 + (r & 7), odd = r >> 3;
    const int pairs = ceil_div(a.K, 128), per = ceil_div(pairs, NW), p0 = min(pairs, wave * per), n = min(pairs, p0 + per) - p0;
    const int8_t *xp = a.x + (size_t)min(m, a.M - 1) * a.ldx;
    const uint4 *wp = a.wp + (size_t)tile * a.ksteps * 64 + 16 * g + 8 * half + (r & 7);
    int4_t acc = {0, 0, 0, 0};
    struct Batch { I8Frag x[U], w[U]; } b0, b1;
    auto request = [&](Batch &b, int at) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int ks = 2 * (p0 + min(at + u, n - 1)) + odd;                     // behind the run: its last pair again, not multiplied
            const int k = 64 * ks + 16 * g, kk = k < a.K ? k : 0;                    // behind the last column the packed weights are zeros
            b.x[u].u = *reinterpret_cast<const uint4 *>(xp + kk);
            b.w[u].u = wp[(size_t)ks * 64];
        }
    };
    auto multiply = [&](const Batch &b, int at) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (at + u >= n) break;
            acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(b.w[u].v, b.x[u].v, acc, 0, 0, 0);
        }
    };
    if (n > 0) {
        request(b0, 0);
        for (int at = 0; at < n; at += 2 * U) {
            if (at + U < n) request(b1, at + U);
            multiply(b0, at);
            if (at + U >= n) break;
            if (at + 2 * U < n) request(b0, at + 2 * U);
            multiply(b1, at + U);
        }
    }
    red[wave][lane] = acc;
    __syncthreads();
    if (wave > 0 || g > 1 || r > 7) return;
    int4_t sum = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < NW; ++w) sum += red[w][lane] + red[w][lane + 40];            // weight row + 8, activation row + 8
    i8_store<SWIGLU>(a, sum, tile, m, lane + 32 * half);
}

#pragma clang diagnostic ignored "-Winline-asm"     // "reserved register" m0 in a clobber list: it is what the block writes
// 16 bytes per lane from memory to LDS, lane i's to place i behind the LDS address `at` (the same in every lane).  In
// assembly because the compiler, which sees a write to LDS in the builtin, waits for it in front of the next read of any
// LDS; here the waits are the caller's: s_waitcnt vmcnt before the barrier in front of the reads.  M0 written by the scalar
// unit is seen by the request one wait state later.
__device__ __forceinline__ void lds_request16(const void *from, uint32_t at) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(at), "v"(from) : "memory", "m0");
}
__device__ __forceinline__ uint32_t lds_address(const void *p) {
    return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void *)p);
}

// Many rows: a workgroup owns BM activation rows x BN weight rows (packed order) and its WM x WN waves an equal part each.
// KS k-steps (64 columns each) of both go to LDS at a time, straight from memory, 16 bytes a lane; ST stages of LDS, so ST - 1
// of them are on their way while one is multiplied.  The weights keep their fragment order; the rows of a 1 KiB request (16
// rows x 64 columns or 8 x 128) stay row-major, the 16-byte chunk c of row r at place c ^ swizzle(r), so that the 16 rows a
// fragment read touches lie in 16 different places modulo 256 bytes.
// Small tiles are bound by what comes in: 64 x 64 takes 0.29 us per 128 columns, 0.23 of them for the requests alone (16 KB,
// 70 GB/s a CU; rows that all lie in L2 would come at 117) and 0.18 for LDS reads and products alone (200 x 4096 x 2048 7.8 us,
// 200 x 2048 x 6144 in 32 x 64 tiles above 13 us).  More stages, eight waves, fragments read a step ahead, padded rows and a
// start along K that differs between workgroups change nothing or cost 2-9 %.  The largest tile is bound by the matrix units' power: 16384 x 2048 x
// 6144 in 171-187 us, 2.2-2.4 POPS (the library's product 175-179), at 1.93 GHz - with zeros for data 136 us.  The 32 x 32 x 32
// instruction, more stages, and fragments read a step ahead into registers are not faster there (186, 168 and 168 us where
// this form took 168); without the turns of the two waves of a SIMD (ALT) it takes 183.
template <int KS>
__device__ __forceinline__ int i8_swizzle(int r) {
    // A 16-byte read is served 16 lanes at a time: 0-3, 12-15, 20-23, 24-27, then 4-7, 8-11, 16-19, 28-31, and so on.  With
    // 64-byte rows four rows share 256 bytes and the swizzle 0, 2, 3, 1 of the row quads keeps such a set apart (0, 1, 2, 3: two
    // lanes to a place, and half the rate).
    return KS == 1 ? ((r >> 1) & 2) ^ (((r >> 3) & 1) * 3) : (r >> 1) & 7;
}

template <int N>
__device__ __forceinline__ void wait_and_meet() {
    // this wave's requests but the last N are in and its reads of LDS are done; behind the barrier, everybody's
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// What a lane needs of the outputs it stores: scale (SwiGLU: of the gate) and bias (SwiGLU: the up rows' scale) of its
// columns, and the row scales of its wave's rows, one row per lane and word.
template <int XW, int OUT>
struct I8Tail {
    float s0[OUT], s1[OUT], xs[XW];
    __device__ __forceinline__ void arrived() const {          // the loads' wait goes here, in front of what follows in assembly
#pragma unroll
        for (int j = 0; j < OUT; ++j) asm volatile("" ::"v"(s0[j]), "v"(s1[j]));
#pragma unroll
        for (int j = 0; j < XW; ++j) asm volatile("" ::"v"(xs[j]));
    }
};

template <int BM, int BN, int WM, int WN, int KS, int ST, bool ALT, bool SWIGLU>
__global__ __launch_bounds__(WM * WN * 64) void linear_int8_tile_kernel(LinI8Args a, int mtiles, int ntiles) {
    constexpr int NW = WM * WN, RPR = 16 / KS, CPR = 4 * KS;       // rows of a request, 16-byte chunks of a row
    constexpr int NA = BM / RPR / NW, NB = BN / 16 * KS / NW, TM = BM / WM / 16, TN = BN / WN / 16;
    constexpr int STAGE = (BM + BN) * CPR;                         // 16-byte places of a stage
    constexpr int WAIT = (ST - 2) * (NA + NB);
    static_assert(BM % (RPR * NW) == 0 && (BN / 16 * KS) % NW == 0 && (RPR * NW) % 16 == 0, "whole requests per wave");
    static_assert(WAIT <= 63, "the wait counter's range");
    // the epilogue: a lane's OUT outputs come from CP sums; LPR lanes to a row, RPP rows a pass; HT row tiles turned at a time,
    // in the last stage's place where that holds a row tile of every wave, otherwise behind the stages
    constexpr int OUT = SWIGLU && TN < 4 ? 4 : 8, CP = SWIGLU ? 2 * OUT : OUT;
    constexpr int LPR = TN * 16 / CP, RPP = 64 / LPR, CMASK = (TN * 4 < 16 ? TN * 4 : 16) - 1;
    constexpr int ROWTILE = NW * 64 * TN;                          // places of one row tile of every wave
    constexpr bool OVER = STAGE >= ROWTILE;
    constexpr int HT0 = OVER ? STAGE / ROWTILE : 1, HT = HT0 >= TM ? TM : HT0 >= 4 && TM % 4 == 0 ? 4 : HT0 >= 2 && TM % 2 == 0 ? 2 : 1;
    constexpr int NP = 16 * HT / RPP, XW = (TM * 16 + 63) / 64;
    static_assert(TM % HT == 0 && (16 * HT) % RPP == 0, "whole passes");
    constexpr int PLACES = ST * STAGE + (OVER ? 0 : ROWTILE);
    static_assert(PLACES <= 10240, "160 KB of LDS");
    __shared__ uint4 lds[PLACES];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN, r = lane & 15, g = lane >> 4;
    const int tiles = SWIGLU ? ceil_div(a.N, 8) : ceil_div(a.N, 16);
    const int nk = a.ksteps / KS, total = mtiles * ntiles;
    const uint32_t lds_at = lds_address(lds) + wave * 1024;
    const int rr = lane / CPR, chunk = (lane % CPR) ^ i8_swizzle<KS>(RPR * wave + rr);
    const int xat = (wm * TM * 16 + r) * CPR + (g ^ i8_swizzle<KS>(r)), wat = BM * CPR + wn * TN * 64 * KS + lane;

    // the tile whose requests go out
    int m0, t0;
    const int8_t *xp[NA];
    const uint4 *wp[NB];
    auto place = [&](int b) {
        // Workgroups are dealt to the 8 XCDs in turn: an XCD takes a run of tiles that lie together, four row blocks wide, so that
        // its workgroups share rows and weights in its L2.
        const int xcd = b & 7, each = total >> 3, id = xcd * each + min(xcd, total & 7) + (b >> 3);
        const int band = id / (4 * ntiles), in = id - band * 4 * ntiles, rows = min(4, mtiles - 4 * band);
        m0 = (4 * band + in % rows) * BM;
        t0 = in / rows * (BN / 16);
#pragma unroll
        for (int i = 0; i < NA; ++i) xp[i] = a.x + (size_t)min(m0 + RPR * (wave + i * NW) + rr, a.M - 1) * a.ldx;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int v = wave + i * NW;
            wp[i] = a.wp + ((size_t)min(t0 + v / KS, tiles - 1) * a.ksteps + v % KS) * 64 + lane;
        }
    };
    auto request = [&](int it, int stage) {
        const int k = 64 * KS * it + 16 * chunk, kk = k < a.K ? k : 0;
        const uint32_t to = lds_at + stage * (STAGE * 16);
#pragma unroll
        for (int i = 0; i < NA; ++i) lds_request16(xp[i] + kk, to + i * NW * 1024);
#pragma unroll
        for (int i = 0; i < NB; ++i) lds_request16(wp[i] + (size_t)it * (64 * KS), to + BM * CPR * 16 + i * NW * 1024);
    };
    auto begin = [&] {
#pragma unroll
        for (int i = 0; i < ST - 1; ++i) if (i < nk) request(i, i);
    };

    // Requests return in the order they were made, stores among them.  Behind an epilogue whose stores are known to be STORES
    // instructions of this wave, they may be under way still while the stages requested before them are waited for.
    constexpr int STORES = TM / HT * NP;                           // one a pass
    static_assert(WAIT + STORES <= 63, "the wait counter's range");
    int loose = 0;                                                 // stages requested before those stores
    auto meet = [&](int it) {                                      // stage `it` is complete, in every wave
        if (it < min(loose, nk - ST + 2)) wait_and_meet<WAIT + STORES>();
        else if (it < nk - ST + 2) wait_and_meet<WAIT>();
        else wait_and_meet<0>();
    };
    int4_t acc[TM][TN];
    place(blockIdx.x);
    begin();
    for (int b = blockIdx.x; b < total; b += gridDim.x) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j] = int4_t{0, 0, 0, 0};
        int stage = 0, next = ST - 1;
        if (!ALT) {
#pragma unroll 1
            for (int it = 0; it < nk; ++it) {
                meet(it);
                if (it + ST - 1 < nk) request(it + ST - 1, next);
                const uint4 *st = lds + stage * STAGE;
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    I8Frag xf[TM], wf[TN];
#pragma unroll
                    for (int j = 0; j < TN; ++j) wf[j].u = st[wat + j * 64 * KS + s * 64];
#pragma unroll
                    for (int i = 0; i < TM; ++i) xf[i].u = st[(xat ^ (4 * s)) + i * 16 * CPR];
#pragma unroll
                    for (int i = 0; i < TM; ++i)
#pragma unroll
                        for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[j].v, xf[i].v, acc[i][j], 0, 0, 0);
                }
                stage = stage + 1 == ST ? 0 : stage + 1;
                next = next + 1 == ST ? 0 : next + 1;
            }
            wait_and_meet<0>();
        } else {
            // The two waves of a SIMD take turns: while one multiplies, the other reads its fragments of the next k-step, and a
            // barrier after each turn keeps them so.  Turns: waves 0-3 read step k in turn 2k and multiply it in turn 2k + 1,
            // waves 4-7 one turn later.  Stage k is complete before turn 2k: every wave waits for its own requests of it at the
            // end of turn 2k - 1.  Requests into the place of stage k - 1, last read in turn 2k - 1, go out from turn 2k on.
            const bool late = wave >= NW / 2;
            meet(0);
            if (late) asm volatile("s_barrier" ::: "memory");
#pragma unroll 1
            for (int it = 0; it < nk; ++it) {
                I8Frag xf[KS][TM], wf[KS][TN];
                const uint4 *st = lds + stage * STAGE;
#pragma unroll
                for (int s = 0; s < KS; ++s) {
#pragma unroll
                    for (int j = 0; j < TN; ++j) wf[s][j].u = st[wat + j * 64 * KS + s * 64];
#pragma unroll
                    for (int i = 0; i < TM; ++i) xf[s][i].u = st[(xat ^ (4 * s)) + i * 16 * CPR];
                }
                if (it + ST - 1 < nk) request(it + ST - 1, next);
                __builtin_amdgcn_sched_barrier(0);
                if (late) meet(it + 1);
                else asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
                __builtin_amdgcn_sched_barrier(0);
                __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int s = 0; s < KS; ++s)
#pragma unroll
                    for (int i = 0; i < TM; ++i)
#pragma unroll
                        for (int j = 0; j < TN; ++j)
                            acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[s][j].v, xf[s][i].v, acc[i][j], 0, 0, 0);
                __builtin_amdgcn_s_setprio(0);
                __builtin_amdgcn_sched_barrier(0);
                if (!late) meet(it + 1);
                else asm volatile("s_barrier" ::: "memory");
                __builtin_amdgcn_sched_barrier(0);
                stage = stage + 1 == ST ? 0 : stage + 1;
                next = next + 1 == ST ? 0 : next + 1;
            }
            if (!late) asm volatile("s_barrier" ::: "memory");
        }
        // Every read of the stages is done (the barriers above).  The next tile's first ST - 1 stages are requested now and come
        // in under the epilogue, which turns the sums round in the last stage's place.
        // What the epilogue needs of the scales is waited for before that: requests return in order.
        const int row0 = m0 + wm * TM * 16, nw = (t0 + wn * TN) * (SWIGLU ? 8 : 16), n0 = nw + OUT * (lane % LPR);
        I8Tail<XW, OUT> now;
#pragma unroll
        for (int j = 0; j < OUT; ++j) {
            const int n = min(n0 + j, a.N - 1);
            now.s0[j] = a.ws[n];
            now.s1[j] = SWIGLU ? a.us[n] : a.bias ? bf2f(a.bias[n]) : 0.f;
        }
#pragma unroll
        for (int j = 0; j < XW; ++j) now.xs[j] = a.xs[min(row0 + 64 * j + lane, a.M - 1)];
        const int whole = a.N / OUT * OUT;                         // the columns behind these are stored one by one
        const bool rest = whole < a.N && whole >= nw && whole < nw + TN * (SWIGLU ? 8 : 16);      // they are this wave's
        // Residual rows are requested RB passes ahead.  Behind the last row the last is read: the loads stay unconditional.
        constexpr int PASSES = TM / HT * NP, RB = SWIGLU ? 1 : PASSES < 8 ? PASSES : 8;
        u32x4_t rf[RB];
        const bool add = !SWIGLU && a.res && whole > 0;
        auto residual = [&](int pass) {
            return (u32x4_t)*reinterpret_cast<const u32x4_any *>(a.res + (size_t)min(row0 + lane / LPR + pass * RPP, a.M - 1) * a.ldr + min(n0, whole - OUT));
        };
        if (add) {
#pragma unroll
            for (int p = 0; p < RB; ++p) rf[p] = residual(p);
#pragma unroll
            for (int p = 0; p < RB; ++p) asm volatile("" ::"v"(rf[p]));
        }
        now.arrived();
        if (b + (int)gridDim.x < total) {
            place(b + gridDim.x);
            begin();
        }
        // Epilogue.  A wave turns its sums round in LDS of its own, HT row tiles at a time, so that a lane has neighbouring
        // outputs of a row: 16-byte loads and stores, and the same columns - hence the same scales and bias, in registers - in
        // every pass.  The 16-byte chunk c of row q lies at place c ^ q (modulo the chunks of a row, 16 at most).
        int4_t *mine = reinterpret_cast<int4_t *>(lds + (OVER ? ST - 1 : ST) * STAGE) + wave * HT * 64 * TN;
        const int lrow = lane / LPR, c = lane % LPR;
        auto outputs = [&](int pass, I8Scale xs, float (&y)[OUT]) {
            const int4_t *v = mine + (pass * RPP + lrow) * (TN * 4);
            const int turn = (lrow & CMASK) ^ ((pass * RPP) & CMASK);
            if (SWIGLU) {
#pragma unroll
                for (int q = 0; q < OUT / 2; ++q) {
                    const int4_t t = v[(OUT / 2 * c + q) ^ turn];
#pragma unroll
                    for (int j = 0; j < 2; ++j) y[2 * q + j] = i8_swiglu(t[j], t[2 + j], xs, now.s0[2 * q + j], now.s1[2 * q + j]);
                }
            } else {
#pragma unroll
                for (int q = 0; q < OUT / 4; ++q) {
                    const int4_t t = v[(OUT / 4 * c + q) ^ turn];
#pragma unroll
                    for (int j = 0; j < 4; ++j) y[4 * q + j] = i8_scaled(t[j], xs, now.s0[4 * q + j], now.s1[4 * q + j]);
                }
            }
        };
        auto row_scale = [&](int row) { return __shfl(now.xs[row >> 6], (row & 63) + lrow); };    // row: a constant, a multiple of RPP
        const int have = n0 < whole ? a.M - row0 - lrow : 0;      // rows from this lane's first on
        bf16_t *op = a.out + (size_t)(row0 + lrow) * a.ldo + n0;
        const size_t ostep = (size_t)RPP * a.ldo;
        // every pass stores something: the rows are there, and the wave's first columns
        loose = row0 + TM * 16 <= a.M && nw < whole ? ST - 1 : 0;
        // Rows whose scale comes last (i8_row_scale) are rare: the two selects an output that they need, 3-4 % of the time (SwiGLU
        // 8192 x 6144 x 2048 193 -> 200 us), are in a copy of the epilogue for waves that have such a row.
        auto epilogue = [&](auto huge_rows) {
            auto scale = [](float xs) { return decltype(huge_rows)::value ? i8_row_scale(xs) : I8Scale{xs, false}; };
#pragma unroll
            for (int h = 0; h < TM; h += HT) {
#pragma unroll
                for (int i = 0; i < HT; ++i)
#pragma unroll
                    for (int j = 0; j < TN; ++j) mine[(16 * i + r) * (TN * 4) + ((4 * j + g) ^ (r & CMASK))] = acc[h + i][j];
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int p = 0; p < NP; ++p) {
                    float y[OUT];
                    outputs(p, scale(row_scale(h * 16 + p * RPP)), y);
                    if (add) {
                        const int pass = h / HT * NP + p;
#pragma unroll
                        for (int j = 0; j < OUT; j += 2) {
                            float lo, hi;
                            unpack2(rf[pass % RB][j / 2], lo, hi);
                            y[j] += lo;
                            y[j + 1] += hi;
                        }
                        if (pass + RB < PASSES) rf[pass % RB] = residual(pass + RB);
                    }
                    uint32_t packed[OUT / 2];
#pragma unroll
                    for (int j = 0; j < OUT; j += 2) packed[j / 2] = pack2v(float2_t{y[j], y[j + 1]});
                    if (h * 16 + p * RPP < have) {
                        // nothing of this launch reads the output again: kept out of the way of the rows and weights in L2 (2-4 %)
                        if constexpr (OUT == 8)
                            __builtin_nontemporal_store(u32x4_t{packed[0], packed[1], packed[2], packed[3]}, reinterpret_cast<u32x4_any *>(op));
                        else __builtin_nontemporal_store(u32x2_t{packed[0], packed[1]}, reinterpret_cast<u32x2_any *>(op));
                    }
                    op += ostep;
                }
                if (rest) {                                            // neighbouring lanes neighbouring columns, 64 / OUT rows at a time
                    const int tc = lane % OUT, n = min(whole + tc, a.N - 1), col = n - nw;
                    const int pc = SWIGLU ? (col >> 1) * 4 + (col & 1) : col;                  // packed column of the sum (of the gate's)
                    const int *flat = reinterpret_cast<const int *>(mine);
                    const float s0 = a.ws[n], s1 = SWIGLU ? a.us[n] : a.bias ? bf2f(a.bias[n]) : 0.f;
#pragma unroll
                    for (int e = 0; e < 16 * HT * OUT / 64; ++e) {
                        const int row = e * (64 / OUT) + lane / OUT, m = min(row0 + h * 16 + row, a.M - 1);
                        const int at = (row * (TN * 4) + ((pc >> 2) ^ (row & CMASK))) * 4 + (pc & 3);
                        const I8Scale xs = scale(__shfl(now.xs[h >> 2], (h & 3) * 16 + row));
                        float y;
                        if (SWIGLU) y = i8_swiglu(flat[at], flat[at + 2], xs, s0, s1);
                        else {
                            y = i8_scaled(flat[at], xs, s0, s1);
                            if (a.res) y += bf2f(a.res[(size_t)m * a.ldr + n]);
                        }
                        if (row0 + h * 16 + row < a.M && whole + tc < a.N) a.out[(size_t)m * a.ldo + n] = f2bf(y);
                    }
                }
                __builtin_amdgcn_wave_barrier();
            }
        };
        bool huge = false;
#pragma unroll
        for (int j = 0; j < XW; ++j) huge |= i8_row_scale(now.xs[j]).later;
        if (__builtin_expect(__any(huge), 0)) epilogue(std::true_type{});
        else epilogue(std::false_type{});
    }
}

// ---- which form a product takes
// A workgroup's time is a fixed part and a part per k-step, the bytes its CU pulls in at 50-70 GB/s (few bytes: latency); a
// launch's is that times the workgroups a CU gets, on top of what the launch itself takes:
//   us = launch + (fixed + step * ceil(K / 64)) * load,   load = max(1, r + 3/4 (ceil(r) - r)),  r = workgroups / 256
// but no less than the weights take from memory at 6 TB/s, times ceil(r) / r for the CUs that idle at the end or throughout
// (2.4 at most: that is what a CU takes alone; SwiGLU 8 x 6144 x 2048 7.5 us in the form chosen without this, 6.9 with it).  The
// table is fitted to the times of every form over 1-8192 rows and nine N x K from 1024 x 1024 to 8192 x 512 (cold weights, in
// a graph).  The form with the smallest estimate is taken.  Over 100 shapes drawn at random it is 3.6 % slower on average than the
// fastest form, by more than 5 % in 22 and by 30-36 % in five: many rows or columns and K below 260, where the fixed parts decide.
// Some shapes (us of the forms in the table's order, '-' far off):
//   1 x 4096 x 2048 (plain)       4.0  3.9  4.1  4.7  5.4  4.0  7.7   -    -    -    -
//   8 x 2048 x 6144 (plain)       7.6  6.2  8.0  8.1   12  5.6   17   -    -    -    -
//   64 x 2048 x 6144 (plain)       11   11  8.8   12   16   20   17   -    -    -    -
//   200 x 4096 x 2048 (plain)      17   17   12   12   11   -   7.9   13   13   17   26
//   800 x 4096 x 2048 (plain)       -    -    -    -    -   -    20   15   14   18   29
//   4096 x 4096 x 2048 (plain)      -    -    -    -    -   -    65   44   50   41   38
struct I8Form { int bm, bn; float launch, fixed, step; };
static constexpr I8Form I8_FORMS[] = {
    {16, 16, 2.52f, 0.117f, 0.037f},     // K over 4 waves
    {16, 16, 2.37f, 0.448f, 0.031f},     // over 8
    {16, 32, 2.42f, 0.147f, 0.048f},     // over 4
    {32, 32, 2.04f, 0.565f, 0.073f},     // over 8
    {32, 64, 1.84f, 1.029f, 0.109f},     // over 8
    {8, 8, 2.48f, 0.201f, 0.019f},       // half a packed tile, over 8
    {64, 64, 3.50f, 0.409f, 0.112f},     // through LDS, as the rest
    {128, 128, 3.97f, 1.346f, 0.279f},
    {128, 128, 1.57f, 3.497f, 0.280f},   // two k-steps a stage, waves in turns
    {128, 256, 0.94f, 6.138f, 0.387f},   // the same
    {256, 256, 0.04f, 11.115f, 0.670f},  // one k-step a stage, waves in turns
};
static constexpr int I8_SPLIT_FORMS = 6;
#ifdef QTTS_TUNING
static int g_i8_form = -1;
extern "C" void qtts_tune_int8(int form) { g_i8_form = form; }      // measurement builds: this form whatever the shape
#else
static constexpr int g_i8_form = -1;
#endif

static int choose_int8_form(int M, int columns, int K) {
    if (g_i8_form >= 0) return g_i8_form;
    int best = -1;
    double least = 0;
    for (int f = 0; f < (int)(sizeof(I8_FORMS) / sizeof(I8_FORMS[0])); ++f) {
        const I8Form &F = I8_FORMS[f];
        // these take a workgroup per tile: row blocks are blockIdx.y, and a row of blocks takes fewer than 2^32 threads
        if (f < I8_SPLIT_FORMS && (ceil_div(M, F.bm) > 65535 || ceil_div(columns, F.bn) > 1 << 22)) continue;
        const double r = (double)ceil_div(M, F.bm) * ceil_div(columns, F.bn) / 256;
        const double cu = (F.fixed + F.step * ceil_div(K, 64)) * std::max(1.0, 0.25 * r + 0.75 * ceil(r));
        const double us = F.launch + std::max(cu, 64.0 * columns * ceil_div(K, 64) / 6e6 * std::min(2.4, ceil(r) / r));
        if (best < 0 || us < least) { best = f; least = us; }
    }
    return best;
}

extern "C" int qtts_linear_int8_form(int M, int N, int K, int swiglu) {
    QCHECK(M > 0 && M <= I8_MAX_ROWS && N > 0 && N <= I8_MAX_N && K > 0 && K <= I8_MAX_K, "linear_int8_form: bad shape M=%d N=%d K=%d (M <= %d, N <= %d, K <= %d)",
           M, N, K, I8_MAX_ROWS, I8_MAX_N, I8_MAX_K);
    return choose_int8_form(M, 16 * ceil_div(N, swiglu ? 8 : 16), K);
}

template <bool SWIGLU>
static void launch_int8_form(const LinI8Args &a, int tiles, int form, hipStream_t s) {
#define QTTS_TILE_I8(BM, BN, WM, WN, KS, ST, ALT, PER_CU) do { const int mt = ceil_div(a.M, BM), nt = ceil_div(tiles, BN / 16); \
        hipLaunchKernelGGL((linear_int8_tile_kernel<BM, BN, WM, WN, KS, ST, ALT, SWIGLU>), dim3((unsigned)std::min<long>((long)mt * nt, 256 * PER_CU)), \
                           dim3(WM * WN * 64), 0, s, a, mt, nt); } while (0)
#define QTTS_SPLIT_I8(TM, TN, NW, U) hipLaunchKernelGGL((linear_int8_split_kernel<TM, TN, NW, U, SWIGLU>), \
        dim3(ceil_div(tiles, TN), ceil_div(a.M, 16 * TM)), dim3(NW * 64), 0, s, a)
    switch (form) {
    case 0: QTTS_SPLIT_I8(1, 1, 4, 4); break;
    case 1: QTTS_SPLIT_I8(1, 1, 8, 4); break;
    case 2: QTTS_SPLIT_I8(1, 2, 4, 4); break;
    case 3: QTTS_SPLIT_I8(2, 2, 8, 2); break;
    case 4: QTTS_SPLIT_I8(2, 4, 8, 2); break;
    case 5: hipLaunchKernelGGL((linear_int8_half_kernel<8, 2, SWIGLU>), dim3(ceil_div(a.N, SWIGLU ? 4 : 8), ceil_div(a.M, 8)), dim3(512), 0, s, a); break;
    case 6: QTTS_TILE_I8(64, 64, 2, 2, 2, 4, false, 2); break;
    case 7: QTTS_TILE_I8(128, 128, 2, 4, 1, 4, false, 2); break;
    case 8: QTTS_TILE_I8(128, 128, 2, 4, 2, 4, true, 1); break;
    case 9: QTTS_TILE_I8(128, 256, 2, 4, 2, 3, true, 1); break;
    case 10: QTTS_TILE_I8(256, 256, 2, 4, 1, 4, true, 1); break;
    }
#undef QTTS_TILE_I8
#undef QTTS_SPLIT_I8
}

static int linear_int8_checked(const char *who, const void *x, int ldx, const float *xs, const void *wp, const float *ws,
                               const float *us, const void *bias, const void *res, int ldr, void *out, int ldo, int M, int N,
                               int K, bool swiglu, qtts_stream_t stream) {
    QCHECK(x && xs && wp && ws && out && (!swiglu || us), "%s: null pointer", who);
    QCHECK(M > 0 && M <= I8_MAX_ROWS && N > 0 && N <= I8_MAX_N && K > 0 && K <= I8_MAX_K, "%s: bad shape M=%d N=%d K=%d (M <= %d, N <= %d, K <= %d)", who, M, N, K,
           I8_MAX_ROWS, I8_MAX_N, I8_MAX_K);
    QCHECK(ldx % 16 == 0 && ldx >= K, "%s: x row stride %d too small or not a multiple of 16", who, ldx);
    QCHECK(ldo >= N && (!res || ldr >= N), "%s: row strides ldo=%d ldr=%d < N=%d", who, ldo, ldr, N);
    QCHECK(out != res || ldo == ldr, "%s: out in the place of the residual needs its row stride", who);
    QCHECK((((uintptr_t)x | (uintptr_t)wp) & 15) == 0 && (((uintptr_t)xs | (uintptr_t)ws | (uintptr_t)us) & 3) == 0 &&
           (((uintptr_t)out | (uintptr_t)bias | (uintptr_t)res) & 1) == 0, "%s: misaligned pointer", who);
    LinI8Args a{};
    a.x = (const int8_t *)x; a.ldx = ldx; a.xs = xs; a.wp = (const uint4 *)wp; a.ws = ws; a.us = us;
    a.bias = (const bf16_t *)bias; a.res = (const bf16_t *)res; a.ldr = ldr; a.out = (bf16_t *)out; a.ldo = ldo;
    a.M = M; a.N = N; a.K = K; a.ksteps = i8_ksteps(K);
    const int tiles = ceil_div(N, swiglu ? 8 : 16), form = choose_int8_form(M, 16 * tiles, K);
    if (swiglu) launch_int8_form<true>(a, tiles, form, (hipStream_t)stream);
    else launch_int8_form<false>(a, tiles, form, (hipStream_t)stream);
    QLAUNCH();
    return QTTS_OK;
}

extern "C" int qtts_linear_int8(const void *x, int ldx, const float *x_scales, const void *w_packed, const float *w_scales,
                                const void *bias, const void *residual, int ldr, void *out, int ldo, int M, int N, int K,
                                qtts_stream_t stream) {
    return linear_int8_checked("linear_int8", x, ldx, x_scales, w_packed, w_scales, nullptr, bias, residual, ldr, out, ldo, M, N, K,
                               false, stream);
}

extern "C" int qtts_linear_swiglu_int8(const void *x, int ldx, const float *x_scales, const void *w_gate_up_packed,
                                       const float *gate_scales, const float *up_scales, void *out, int ldo, int M, int I, int K,
                                       qtts_stream_t stream) {
    return linear_int8_checked("linear_swiglu_int8", x, ldx, x_scales, w_gate_up_packed, gate_scales, up_scales, nullptr, nullptr, 0,
                               out, ldo, M, I, K, true, stream);
}
