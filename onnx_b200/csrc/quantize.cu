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
// p = x * inv.  A point halfway between two e4m3 values has the low 20 bits
// 0x80000 (the low 16 zero under 2^-6, where the steps no longer shrink).  A
// quotient is one of them or, as 448 X = D A has integers on both sides, at
// least 2^-(5 + bits of A) away from it.
//   16-bit types: inv is 448 / amax and up to two steps more, so p is the
//     quotient or up to 4 steps above it in magnitude; with the low 3 bits
//     cleared a halfway quotient is exact, and any other is 2^-16 away.
//   float: p is within two steps of the quotient, so it can be on the wrong
//     side only within two steps of a halfway point (one element in 200000);
//     there the quotient is taken as p + e, with the remainders of both
//     roundings in e.
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

// One block's factors: inv (above), and what rounding 448 / amax left, relative.
struct Factor {
    float inv, rest;
};
template <typename T>
__device__ __forceinline__ Factor factor(float amax) {
    const float inv = __fdiv_rn(kE4M3Max, amax);
    if (sizeof(T) == 2) return {inv > 0.0f ? __uint_as_float(__float_as_uint(inv) + 2u) : inv, 0.0f};
    return {inv, __fmaf_rn(-amax, inv, kE4M3Max) * (1.0f / kE4M3Max)};
}

__device__ __forceinline__ bool may_be_halfway(float p) {
    return ((__float_as_uint(p) - 0x7fffeu) & 0xfffffu) <= 4u || fabsf(p) < 0x1p-6f;
}

// A float that rounds to the same e4m3 value as 448 x / amax = p + e: the sum,
// with its last bit set where it is not exact, which no halfway point has.  e
// is right to 2^-46 of p, and a quotient that is no halfway point is 2^-34 away.
__device__ __forceinline__ float quotient(float x, float p, Factor f) {
    const float e = __fmaf_rn(x, f.inv, -p) + p * f.rest;
    const float s = p + e, left = (p - s) + e;
    const uint32_t b = __float_as_uint(s);
    const bool inexact = fabsf(left) > 0x1p-40f * fabsf(s) && !(b & 1);
    return !inexact ? s : __uint_as_float((left > 0.0f) == (s > 0.0f) ? b + 1 : b - 1);
}

// four elements' bytes
template <typename T>
__device__ __forceinline__ uint32_t quant4(float a, float b, float c, float d, Factor f) {
    const float x[4] = {a, b, c, d};
    float p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        p[i] = x[i] * f.inv;
        if (sizeof(T) == 2) p[i] = __uint_as_float(__float_as_uint(p[i]) & ~7u);
    }
    if (sizeof(T) == 4 && (may_be_halfway(p[0]) | may_be_halfway(p[1]) | may_be_halfway(p[2]) | may_be_halfway(p[3]))) {
        // (most often zeros, which stay; under 2^-6 any p takes the longer way)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (p[i] != 0.0f) p[i] = quotient(x[i], p[i], f);
    }
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(p[0], p[1]), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(p[2], p[3]), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
}

// 1 x 128 blocks where rows of x start on 16 bytes and rows of q on 16 /
// sizeof(T): 8 lanes to a block and 16 elements to a lane, so that the block's
// two divisions and the shuffles for its maximum are shared by 16 elements (a
// warp to a block, 4 elements a lane, was bound by instructions: 72 us instead
// of 43 at 32768 x 1536 floats).  The next 64 bytes a thread are in flight
// meanwhile.
template <typename T>
struct RowWalk {
    static constexpr int VN = 16 / (int)sizeof(T);
    static constexpr int LANES = 8, NV = QB / LANES / VN;
    static constexpr int U = 4 / NV;            // blocks of a group of lanes at a time: 64 bytes a thread
    static constexpr int GROUPS = 256 / LANES;  // of a CTA
};
template <typename T, typename I>
__global__ void __launch_bounds__(256) k_quantize_rows(const T *__restrict__ x, int64_t ldx, I rows, I cols,
                                                       uint8_t *__restrict__ q, int64_t ldq,
                                                       float *__restrict__ scale, int64_t lds) {
    using W = RowWalk<T>;
    constexpr int VN = W::VN, LANES = W::LANES, NV = W::NV, U = W::U;
    const int lane = threadIdx.x % LANES;
    const I nkb = (cols + QB - 1) / QB;
    const I groups = (I)gridDim.x * W::GROUPS, srow = groups / nkb, skb = groups - srow * nkb;
    I b0 = (I)blockIdx.x * W::GROUPS + (I)(threadIdx.x / LANES), row = b0 / nkb, kb = b0 - row * nkb;
    const auto advance = [&] {  // to the block `groups` further on
        row += srow;
        kb += skb;
        if (kb >= nkb) kb -= nkb, ++row;
    };
    const auto fetch = [&](uint4 (&raw)[NV], I row_, I kb_) {  // elements past the row's end are 0
        const T *xb = x + (int64_t)row_ * ldx + kb_ * QB;
        const int nc = row_ >= rows ? 0 : cols - kb_ * QB < QB ? (int)(cols - kb_ * QB) : QB;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int at = (lane + LANES * i) * VN;
            raw[i] = make_uint4(0, 0, 0, 0);
            if (at + VN <= nc) {
                raw[i] = __ldcs(reinterpret_cast<const uint4 *>(xb + at));
            } else if (at < nc) {
                T part[VN];
#pragma unroll
                for (int j = 0; j < VN; ++j) part[j] = at + j < nc ? xb[at + j] : T(0.0f);
                raw[i] = *reinterpret_cast<const uint4 *>(part);
            }
        }
    };
    uint4 next[U][NV];
    I nrow[U], nkbs[U];
    const auto fetch_all = [&] {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            nrow[u] = row, nkbs[u] = kb;
            fetch(next[u], row, kb);
            advance();
        }
    };
    fetch_all();
    // (a warp's four groups of lanes have neighbouring blocks: it ends with the last)
    while (__any_sync(0xffffffffu, nrow[0] < rows)) {
        uint4 raw[U][NV];
        I r[U], k[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            r[u] = nrow[u], k[u] = nkbs[u];
#pragma unroll
            for (int i = 0; i < NV; ++i) raw[u][i] = next[u][i];
        }
        fetch_all();
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float m = kTiny;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                float v[VN];
                unpack<T>(raw[u][i], v);
#pragma unroll
                for (int j = 0; j < VN; ++j) m = fmaxf(m, fabsf(v[j]));
            }
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            if (r[u] >= rows) continue;
            const int nc = cols - k[u] * QB < QB ? (int)(cols - k[u] * QB) : QB;
            const Factor f = factor<T>(m);
            if (lane == 0) scale[(int64_t)r[u] * lds + k[u]] = __fdiv_rn(m, kE4M3Max);
            uint8_t *qb = q + (int64_t)r[u] * ldq + k[u] * QB;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int at = (lane + LANES * i) * VN;
                float v[VN];
                unpack<T>(raw[u][i], v);
                uint32_t w[VN / 4];
#pragma unroll
                for (int j = 0; j < VN / 4; ++j) w[j] = quant4<T>(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3], f);
                if (at + VN <= nc) {
                    if constexpr (VN == 4) *reinterpret_cast<uint32_t *>(qb + at) = w[0];
                    else *reinterpret_cast<uint2 *>(qb + at) = make_uint2(w[0], w[VN / 4 - 1]);
                } else {
#pragma unroll
                    for (int j = 0; j < VN; ++j)
                        if (at + j < nc) qb[at + j] = (uint8_t)(w[j / 4] >> 8 * (j % 4));
                }
            }
        }
    }
}

// The same at any alignment: a run of up to four blocks of a row to a warp,
// elements 4 lane .. 4 lane + 3 of each block to a lane (X4: as one load).  The
// bytes leave as aligned words, put together from neighbouring lanes' and
// blocks': L2 pays for each partly written 32-byte sector (single bytes, 8 to 32
// in a row: 66 to 83 us at 11212 x 4229 halves; 53 us this way, and 47 at 11212 x
// 4228 with one load for four elements).  Lane b takes the divisions of
// block b.
template <typename T, bool X4>
__global__ void __launch_bounds__(256, 4) k_quantize_rows_any(const T *__restrict__ x, int64_t ldx, int64_t rows,
                                                              int64_t cols, uint8_t *__restrict__ q, int64_t ldq,
                                                              float *__restrict__ scale, int64_t lds) {
    constexpr int NB = 4, RUN = NB * QB;
    const int lane = threadIdx.x & 31;
    const int64_t runs = (cols + RUN - 1) / RUN, warps = (int64_t)gridDim.x * 8;
    const int64_t srow = warps / runs, srun = warps - srow * runs;
    const int64_t first = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    int64_t row = first / runs, run = first - row * runs;
    while (row < rows) {
        const T *xb = x + row * ldx + run * RUN + 4 * lane;
        uint8_t *qb = q + row * ldq + run * RUN;
        float *sb = scale + row * lds + run * NB;
        const int nc = (int)min((int64_t)RUN, cols - run * RUN);  // columns of the run
        float v[NB][4], m[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int at = b * QB + 4 * lane;
            if (X4 && at + 4 <= nc) {
                if constexpr (sizeof(T) == 4) {
                    const float4 f = __ldcs(reinterpret_cast<const float4 *>(xb + b * QB));
                    v[b][0] = f.x, v[b][1] = f.y, v[b][2] = f.z, v[b][3] = f.w;
                } else {
                    const uint2 f = __ldcs(reinterpret_cast<const uint2 *>(xb + b * QB));
                    const T *p = reinterpret_cast<const T *>(&f);
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[b][j] = to_f32(p[j]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[b][j] = at + j < nc ? to_f32(xb[b * QB + j]) : 0.0f;
            }
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const float a = fmaxf(fmaxf(kTiny, fmaxf(fabsf(v[b][0]), fabsf(v[b][1]))), fmaxf(fabsf(v[b][2]), fabsf(v[b][3])));
            m[b] = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(a)));  // (positive: ordered as its bits)
        }
        const float mm = (lane & 2) ? (lane & 1 ? m[3] : m[2]) : (lane & 1 ? m[1] : m[0]);
        const Factor fm = factor<T>(mm);
        if (lane < NB && lane * QB < nc) sb[lane] = __fdiv_rn(mm, kE4M3Max);
        uint32_t w[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const Factor f{__shfl_sync(0xffffffffu, fm.inv, b), sizeof(T) == 4 ? __shfl_sync(0xffffffffu, fm.rest, b) : 0.0f};
            w[b] = quant4<T>(v[b][0], v[b][1], v[b][2], v[b][3], f);
        }
        const int sh = (int)((uintptr_t)qb & 3);
        const int full = nc & ~(QB - 1);  // what words cover; the rest of the row leaves as bytes
        uint8_t *at = qb + 4 * lane - sh;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            // the word that ends where this lane's begins: the last lane's or the last block's
            uint32_t before = __shfl_up_sync(0xffffffffu, w[b], 1);
            const uint32_t last = __shfl_sync(0xffffffffu, w[b > 0 ? b - 1 : 0], 31);
            if (lane == 0) before = last;
            if (b * QB < full) {
                if (b > 0 || lane > 0 || sh == 0)
                    *reinterpret_cast<uint32_t *>(at + b * QB) = __funnelshift_l(before, w[b], 8 * sh);
                else
                    for (int j = 0; j < 4 - sh; ++j) qb[j] = (uint8_t)(w[0] >> 8 * j);
                if (lane == 31 && b * QB + QB == full)
                    for (int j = 4 - sh; j < 4; ++j) qb[b * QB + 124 + j] = (uint8_t)(w[b] >> 8 * j);
            } else if (b * QB < nc) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (b * QB + 4 * lane + j < nc) qb[b * QB + 4 * lane + j] = (uint8_t)(w[b] >> 8 * j);
            }
        }
        row += srow;
        run += srun;
        if (run >= runs) run -= runs, ++row;
    }
}

// 128 x 128 blocks: a CTA of 16 warps per block, which stays in registers (32
// values a thread) while the maximum crosses the CTA.  250037 x 384 floats: 90 us,
// 5.3 TB/s; bfloat16 84 us, 3.4 TB/s: a CTA has no load in flight from its
// block's last one to its end, and only other CTAs' fill that time.
constexpr int kBlockThreads = 512;
template <typename T, bool VEC>
__global__ void __launch_bounds__(kBlockThreads, VEC && sizeof(T) == 2 ? 3 : 2)
    k_quantize_blocks(const T *__restrict__ x, int64_t ldx, int64_t rows, int64_t cols, uint8_t *__restrict__ q,
                      int64_t ldq, float *__restrict__ scale, int64_t lds) {
    // VEC: a lane's elements are 16-byte vectors, kept as they come; otherwise 4 elements, 32 apart
    constexpr int VN = VEC ? 16 / (int)sizeof(T) : 4;
    constexpr int LANES = QB / VN, TALL = kBlockThreads / LANES;  // rows per step
    constexpr int STEPS = QB / TALL;
    __shared__ float red[kBlockThreads / 32];
    const int lane = threadIdx.x % LANES, r0 = threadIdx.x / LANES;
    const int64_t nkb = (cols + QB - 1) / QB, total = (rows + QB - 1) / QB * nkb;
    for (int64_t b = blockIdx.x; b < total; b += gridDim.x) {
        const int64_t rb = b / nkb, kb = b - rb * nkb;
        const T *xb = x + rb * QB * ldx + kb * QB;
        uint8_t *qb = q + rb * QB * ldq + kb * QB;
        const int nr = (int)min((int64_t)QB, rows - rb * QB), nc = (int)min((int64_t)QB, cols - kb * QB);
        T part[STEPS][VN];
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const int r = r0 + s * TALL;
            const T *xr = xb + (int64_t)r * ldx;
            if (VEC && r < nr && lane * VN + VN <= nc) {
                *reinterpret_cast<uint4 *>(part[s]) = __ldcs(reinterpret_cast<const uint4 *>(xr + lane * VN));
            } else {
#pragma unroll
                for (int j = 0; j < VN; ++j) {
                    const int at = VEC ? lane * VN + j : lane + 32 * j;
                    part[s][j] = r < nr && at < nc ? xr[at] : T(0.0f);
                }
            }
        }
        float m = kTiny;
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
#pragma unroll
            for (int j = 0; j < VN; ++j) m = fmaxf(m, fabsf(to_f32(part[s][j])));
        m = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m)));  // (positive: ordered as its bits)
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
        __syncthreads();
        m = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(red[threadIdx.x % (kBlockThreads / 32)])));
        __syncthreads();
        const Factor f = factor<T>(m);
        if (threadIdx.x == 0) scale[rb * lds + kb] = __fdiv_rn(m, kE4M3Max);
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const int r = r0 + s * TALL;
            if (r >= nr) continue;
            uint8_t *qr = qb + (int64_t)r * ldq;
            uint32_t w[VN / 4];
#pragma unroll
            for (int j = 0; j < VN / 4; ++j)
                w[j] = quant4<T>(to_f32(part[s][4 * j]), to_f32(part[s][4 * j + 1]), to_f32(part[s][4 * j + 2]),
                                 to_f32(part[s][4 * j + 3]), f);
            if (VEC && lane * VN + VN <= nc) {
                if constexpr (VN == 4) *reinterpret_cast<uint32_t *>(qr + lane * VN) = w[0];
                else *reinterpret_cast<uint2 *>(qr + lane * VN) = make_uint2(w[0], w[VN / 4 - 1]);
            } else {
#pragma unroll
                for (int j = 0; j < VN; ++j) {
                    const int at = VEC ? lane * VN + j : lane + 32 * j;
                    if (at < nc) qr[at] = (uint8_t)(w[j / 4] >> 8 * (j % 4));
                }
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
        if (vec) {
            // the CTAs that an SM holds at once (by registers), each walking over blocks
            const int64_t total = rows * nkb;
            const unsigned grid = (unsigned)std::min<int64_t>((total + 31) / 32, ctx->num_sms * (sizeof(T) == 4 ? 4 : 3));
            // 32-bit indices where blocks and columns allow it.  A group of lanes whose
            // neighbour in the warp has the last block (3 blocks before its own) has U
            // blocks at hand and U in flight, each a grid's groups further on, and has
            // stepped past them: the furthest block whose row it computes.
            using W = RowWalk<T>;
            const int64_t furthest = total + 3 + (int64_t)2 * W::U * W::GROUPS * grid;
            if (furthest < (1ll << 31) && cols < (1ll << 30))
                k_quantize_rows<T, int><<<grid, 256, 0, st>>>(x, ldx, (int)rows, (int)cols, q, ldq, scale, lds);
            else
                k_quantize_rows<T, int64_t><<<grid, 256, 0, st>>>(x, ldx, rows, cols, q, ldq, scale, lds);
        } else {
            const int64_t total = rows * ((nkb + 3) / 4);
            const unsigned grid = (unsigned)std::min<int64_t>((total + 7) / 8, ctx->num_sms * 4);
            if (((uintptr_t)x & (4 * sizeof(T) - 1)) == 0 && ldx % 4 == 0)
                k_quantize_rows_any<T, true><<<grid, 256, 0, st>>>(x, ldx, rows, cols, q, ldq, scale, lds);
            else
                k_quantize_rows_any<T, false><<<grid, 256, 0, st>>>(x, ldx, rows, cols, q, ldq, scale, lds);
        }
    } else {
        const int64_t total = (rows + QB - 1) / QB * nkb;
        const unsigned grid = (unsigned)std::min<int64_t>(total, 1ll << 30);
        if (vec)
            k_quantize_blocks<T, true><<<grid, kBlockThreads, 0, st>>>(x, ldx, rows, cols, q, ldq, scale, lds);
        else
            k_quantize_blocks<T, false><<<grid, kBlockThreads, 0, st>>>(x, ldx, rows, cols, q, ldq, scale, lds);
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
