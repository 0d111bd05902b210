// lonnx_quantize_fp8: block quantisation to 8-bit float (e4m3), one fp32
// scale per block of 128 columns and 1 or 128 rows.
//
//   amax  = max(2^-96, max |x| over the block)
//   scale = amax / 448                      (448: the largest e4m3 value)
//   q     = e4m3(448 x / amax)              (the quotient's nearest, ties to even)
//
// so q * scale stands for x.  2^-96 keeps 448 / amax finite, and a block of
// zeros quantises to zeros.  The maximum skips NaN, which stays NaN in q; an
// infinity makes its block's scale infinite and 448 / amax zero, so every
// element of the block dequantises to NaN.
//
// q is the correctly rounded quotient although it comes from an fp32 product
// p = x * inv, inv = 448 / amax: a point halfway between two e4m3 values has
// its low 16 bits zero, and p is within two steps of the quotient (half a step
// from each of its two roundings, at most twice that across a power of two),
// so p can be on the wrong side only where its low bits are within 2 of zero
// (one element in 13000).  There the quotient is taken as p + e, with the
// remainders of both roundings in e.
//
// Bound by HBM: x is read once (into registers, where it waits for its
// block's maximum), q and the scales are written once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>

#include "lonnx_internal.cuh"

namespace {

constexpr int QB = 128;  // columns (and, for weights, rows) of a block
constexpr float kE4M3Max = 448.0f, kTiny = 0x1p-96f;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

// one 16-byte vector of T as floats (4 or 8 of them)
template <typename T>
__device__ __forceinline__ void unpack(const uint4 &u, float (&f)[16 / sizeof(T)]) {
    const T *p = reinterpret_cast<const T *>(&u);
#pragma unroll
    for (int i = 0; i < (int)(16 / sizeof(T)); ++i) f[i] = to_f32(p[i]);
}

// One block's factors: inv = 448 / amax, and what that rounding left, relative.
struct Factor {
    float inv, rest;
};
__device__ __forceinline__ Factor factor(float amax) {
    const float inv = __fdiv_rn(kE4M3Max, amax);
    return {inv, __fmaf_rn(-amax, inv, kE4M3Max) * (1.0f / kE4M3Max)};
}

__device__ __forceinline__ bool may_be_halfway(float p) { return ((__float_as_uint(p) + 2u) & 0xffffu) <= 4u; }

// A float that rounds to the same e4m3 value as 448 x / amax = p + e: the sum,
// with its last bit set where it is not exact, which no halfway point has.  e
// is right to 2^-46 of p; a quotient is a halfway point or, as 448 X = D A has
// integers under 2^33 times powers of two on both sides, 2^-34 away from it.
__device__ __forceinline__ float quotient(float x, float p, Factor f) {
    const float e = __fmaf_rn(x, f.inv, -p) + p * f.rest;
    const float s = p + e, left = (p - s) + e;
    const uint32_t b = __float_as_uint(s);
    const bool inexact = fabsf(left) > 0x1p-40f * fabsf(s) && !(b & 1);
    return !inexact ? s : __uint_as_float((left > 0.0f) == (s > 0.0f) ? b + 1 : b - 1);
}

__device__ __forceinline__ uint32_t quant4(float a, float b, float c, float d, Factor f) {
    float p[4] = {a * f.inv, b * f.inv, c * f.inv, d * f.inv};
    if (may_be_halfway(p[0]) | may_be_halfway(p[1]) | may_be_halfway(p[2]) | may_be_halfway(p[3])) {
        // (most often zeros, which stay)
        if (p[0] != 0.0f && may_be_halfway(p[0])) p[0] = quotient(a, p[0], f);
        if (p[1] != 0.0f && may_be_halfway(p[1])) p[1] = quotient(b, p[1], f);
        if (p[2] != 0.0f && may_be_halfway(p[2])) p[2] = quotient(c, p[2], f);
        if (p[3] != 0.0f && may_be_halfway(p[3])) p[3] = quotient(d, p[3], f);
    }
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(p[0], p[1]), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(p[2], p[3]), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
}

// 1 x 128 blocks, 8 lanes to a block and 16 elements to a lane, so that the
// block's two divisions and the shuffles for its maximum are shared by 16
// elements (a warp to a block of floats, 4 elements a lane, took 72 us instead
// of 48 at 32768 x 1536: it was bound by instructions).  VEC: rows of x start
// on 16 bytes and rows of q on 16 / sizeof(T) bytes, and a lane's elements are
// 16-byte vectors, 8 vectors apart; otherwise single elements, 8 apart.
template <typename T, bool VEC, typename I>
__global__ void __launch_bounds__(256) k_quantize_rows(const T *__restrict__ x, int64_t ldx, I rows, I cols,
                                                       uint8_t *__restrict__ q, int64_t ldq,
                                                       float *__restrict__ scale, int64_t lds) {
    constexpr int VN = VEC ? 16 / (int)sizeof(T) : 1;  // elements of one access
    constexpr int LANES = 8, NV = QB / LANES / VN;
    const int lane = threadIdx.x % LANES;
    const I nkb = (cols + QB - 1) / QB, total = rows * nkb;
    const I first = (I)blockIdx.x * (256 / LANES), step = (I)gridDim.x * (256 / LANES);
    for (I base = first; base < total; base += step) {
        const I b = base + (I)(threadIdx.x / LANES);
        const bool in = b < total;
        const I row = in ? b / nkb : 0, kb = in ? b - row * nkb : 0;
        const I c = kb * QB;
        const int nc = !in ? 0 : cols - c < QB ? (int)(cols - c) : QB;
        const T *xb = x + (int64_t)row * ldx + c;
        float v[NV][VN];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int at = (lane + LANES * i) * VN;
            if constexpr (VEC) {
                if (at + VN <= nc) {
                    unpack<T>(__ldcs(reinterpret_cast<const uint4 *>(xb + at)), v[i]);
                } else {
#pragma unroll
                    for (int j = 0; j < VN; ++j) v[i][j] = at + j < nc ? to_f32(xb[at + j]) : 0.0f;
                }
            } else {
                v[i][0] = at < nc ? to_f32(xb[at]) : 0.0f;
            }
        }
        float m = kTiny;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < VN; ++j) m = fmaxf(m, fabsf(v[i][j]));
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (!in) continue;
        const Factor f = factor(m);
        if (lane == 0) scale[(int64_t)row * lds + kb] = __fdiv_rn(m, kE4M3Max);
        uint8_t *qb = q + (int64_t)row * ldq + c;
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int at = (lane + LANES * i) * VN;
                uint32_t w[VN / 4];
#pragma unroll
                for (int j = 0; j < VN / 4; ++j)
                    w[j] = quant4(v[i][4 * j], v[i][4 * j + 1], v[i][4 * j + 2], v[i][4 * j + 3], f);
                if (at + VN <= nc) {
                    if constexpr (VN == 4) *reinterpret_cast<uint32_t *>(qb + at) = w[0];
                    else *reinterpret_cast<uint2 *>(qb + at) = make_uint2(w[0], w[VN / 4 - 1]);
                } else {
#pragma unroll
                    for (int j = 0; j < VN; ++j)
                        if (at + j < nc) qb[at + j] = (uint8_t)(w[j / 4] >> 8 * (j % 4));
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < NV; i += 4) {
                const uint32_t w = quant4(v[i][0], v[i + 1][0], v[i + 2][0], v[i + 3][0], f);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int at = lane + LANES * (i + j);
                    if (at < nc) qb[at] = (uint8_t)(w >> 8 * j);
                }
            }
        }
    }
}

// 128 x 128 blocks: a CTA of 8 warps per block, which stays in registers (64
// values a thread) while the maximum crosses the CTA.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) k_quantize_blocks(const T *__restrict__ x, int64_t ldx, int64_t rows,
                                                         int64_t cols, uint8_t *__restrict__ q, int64_t ldq,
                                                         float *__restrict__ scale, int64_t lds) {
    constexpr int VN = VEC ? 16 / (int)sizeof(T) : 4;
    constexpr int LANES = QB / VN, TALL = 256 / LANES;  // rows per step
    constexpr int STEPS = QB / TALL;
    __shared__ float red[8];
    const int lane = threadIdx.x % LANES, r0 = threadIdx.x / LANES;
    const int64_t nkb = (cols + QB - 1) / QB, total = (rows + QB - 1) / QB * nkb;
    for (int64_t b = blockIdx.x; b < total; b += gridDim.x) {
        const int64_t rb = b / nkb, kb = b - rb * nkb;
        const T *xb = x + rb * QB * ldx + kb * QB;
        uint8_t *qb = q + rb * QB * ldq + kb * QB;
        const int nr = (int)min((int64_t)QB, rows - rb * QB), nc = (int)min((int64_t)QB, cols - kb * QB);
        float v[STEPS][VN];
        float m = kTiny;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const int r = r0 + s * TALL;
            const T *xr = xb + (int64_t)r * ldx;
            if constexpr (VEC) {
                const int at = lane * VN;
                if (r < nr && at + VN <= nc) {
                    unpack<T>(__ldcs(reinterpret_cast<const uint4 *>(xr + at)), v[s]);
                } else {
#pragma unroll
                    for (int j = 0; j < VN; ++j) v[s][j] = r < nr && at + j < nc ? to_f32(xr[at + j]) : 0.0f;
                }
            } else {
#pragma unroll
                for (int j = 0; j < VN; ++j)
                    v[s][j] = r < nr && lane + 32 * j < nc ? to_f32(xr[lane + 32 * j]) : 0.0f;
            }
        }
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
#pragma unroll
            for (int j = 0; j < VN; ++j) m = fmaxf(m, fabsf(v[s][j]));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 8; ++w) m = fmaxf(m, red[w]);
        __syncthreads();
        const Factor f = factor(m);
        if (threadIdx.x == 0) scale[rb * lds + kb] = __fdiv_rn(m, kE4M3Max);
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const int r = r0 + s * TALL;
            if (r >= nr) continue;
            uint8_t *qr = qb + (int64_t)r * ldq;
            uint32_t w[VN / 4];
#pragma unroll
            for (int j = 0; j < VN / 4; ++j)
                w[j] = quant4(v[s][4 * j], v[s][4 * j + 1], v[s][4 * j + 2], v[s][4 * j + 3], f);
            if constexpr (VEC) {
                const int at = lane * VN;
                if (at + VN <= nc) {
                    if constexpr (VN == 4) *reinterpret_cast<uint32_t *>(qr + at) = w[0];
                    else *reinterpret_cast<uint2 *>(qr + at) = make_uint2(w[0], w[VN / 4 - 1]);
                } else {
#pragma unroll
                    for (int j = 0; j < VN; ++j)
                        if (at + j < nc) qr[at + j] = (uint8_t)(w[j / 4] >> 8 * (j % 4));
                }
            } else {
#pragma unroll
                for (int j = 0; j < VN; ++j)
                    if (lane + 32 * j < nc) qr[lane + 32 * j] = (uint8_t)(w[0] >> 8 * j);
            }
        }
    }
}

template <typename T>
int quantize(lonnx_ctx *ctx, const void *xv, int64_t rows, int64_t cols, int64_t ldx, int block_rows, uint8_t *q,
             int64_t ldq, float *scale, int64_t lds) {
    const T *x = static_cast<const T *>(xv);
    constexpr int VN = 16 / (int)sizeof(T);
    const bool vec = ((uintptr_t)x & 15) == 0 && ldx % VN == 0 && ((uintptr_t)q & (VN - 1)) == 0 && ldq % VN == 0;
    const int64_t nkb = (cols + QB - 1) / QB;
    cudaStream_t st = ctx->stream;
    if (block_rows == 1) {
        const int64_t total = rows * nkb, per_cta = 256 / 8;
        const unsigned grid = (unsigned)std::min<int64_t>((total + per_cta - 1) / per_cta, (int64_t)ctx->num_sms * 32);
        // 32-bit indices (one 32-bit division per block) where blocks and columns allow it
        const bool small = total + (int64_t)grid * per_cta < (1ll << 31) && cols < (1ll << 30);
        if (vec && small)
            k_quantize_rows<T, true, int><<<grid, 256, 0, st>>>(x, ldx, (int)rows, (int)cols, q, ldq, scale, lds);
        else if (vec)
            k_quantize_rows<T, true, int64_t><<<grid, 256, 0, st>>>(x, ldx, rows, cols, q, ldq, scale, lds);
        else if (small)
            k_quantize_rows<T, false, int><<<grid, 256, 0, st>>>(x, ldx, (int)rows, (int)cols, q, ldq, scale, lds);
        else
            k_quantize_rows<T, false, int64_t><<<grid, 256, 0, st>>>(x, ldx, rows, cols, q, ldq, scale, lds);
    } else {
        const int64_t total = (rows + QB - 1) / QB * nkb;
        const unsigned grid = (unsigned)std::min<int64_t>(total, 1ll << 30);
        if (vec)
            k_quantize_blocks<T, true><<<grid, 256, 0, st>>>(x, ldx, rows, cols, q, ldq, scale, lds);
        else
            k_quantize_blocks<T, false><<<grid, 256, 0, st>>>(x, ldx, rows, cols, q, ldq, scale, lds);
    }
    LONNX_CHECK_LAUNCH(ctx);
    return LONNX_OK;
}

}  // namespace

using namespace lonnx;

extern "C" LONNX_API int lonnx_quantize_fp8(lonnx_ctx *ctx, const void *x, int dtype, int64_t rows, int64_t cols,
                                            int64_t ldx, int block_rows, void *q, int64_t ldq, float *scale,
                                            int64_t lds) {
    const int es = dtype == LONNX_DT_F32 ? 4 : dtype == LONNX_DT_F16 || dtype == LONNX_DT_BF16 ? 2 : 0;
    if (!es) return set_error(LONNX_E_UNSUPPORTED, "quantize_fp8: input type %d (float, float16 and bfloat16 are supported)", dtype);
    if (block_rows != 1 && block_rows != QB)
        return set_error(LONNX_E_BADARG, "quantize_fp8: blocks of %d rows (1 or 128 are supported)", block_rows);
    if (rows < 0 || cols < 0) return set_error(LONNX_E_BADARG, "quantize_fp8: negative size");
    if (ldx < cols || ldq < cols || lds < (cols + QB - 1) / QB)
        return set_error(LONNX_E_SHAPE, "quantize_fp8: a leading dimension is smaller than its row");
    if (((uintptr_t)x & (es - 1)) || ((uintptr_t)scale & 3))
        return set_error(LONNX_E_BADARG, "quantize_fp8: a pointer is not aligned to its element type");
    int rc = device_guard(ctx);
    if (rc) return rc;
    if (rows == 0 || cols == 0) return LONNX_OK;
    if (!x || !q || !scale) return set_error(LONNX_E_BADARG, "quantize_fp8: null pointer");
    uint8_t *qb = static_cast<uint8_t *>(q);
    if (dtype == LONNX_DT_F32) return quantize<float>(ctx, x, rows, cols, ldx, block_rows, qb, ldq, scale, lds);
    if (dtype == LONNX_DT_F16) return quantize<__half>(ctx, x, rows, cols, ldx, block_rows, qb, ldq, scale, lds);
    return quantize<__nv_bfloat16>(ctx, x, rows, cols, ldx, block_rows, qb, ldq, scale, lds);
}
