// lonnx_gemm_fp8: C = act(A . B^T + bias) with A [M, K] and B [N, K] in e4m3
// and one fp32 scale per 1 x 128 block of A and per 128 x 128 block of B:
//
//   C[m, n] = act(sum_b sA[m, b] * sB[n / 128, b] * sum_{k in block b} A[m, k] B[n, k] + bias[n])
//
// The tensor cores (tcgen05.mma kind::f8f6f4) sum one block of 128 columns of
// K into TMEM; warps read that sum back, scale it and add it to fp32 registers
// while the next block runs into the other of two TMEM buffers.  So a block's
// products are exact fp32-accumulated sums of 128 terms, and scales of any
// value (not only powers of two) cost one FMA an element and block.
//
// What bounds it.  8192^3: 0.52 ms in a burst (2130 TFLOP/s), 0.61 under the
// power cap (1.47 GHz at 1 kW); a block of a 128 x 256 tile takes 860 cycles, of
// which shared memory (operands written once and read once, 96 KB at 128 bytes a
// cycle) needs 768 and the tensor cores 512.  32768 x 1536 x 384 to floats: 46 us,
// 4.4 TB/s of output, with GELU 59, bound by the epilogue's instructions.
//
// Two kernels.  k_fp8_wide: tiles of 128 rows of A x BN rows of B, for
// problems that fill the GPU with them.  k_fp8_split: B's rows as the tensor
// core's 128 and 16 to 64 rows of A as its columns, K split over the CTAs of
// a cluster that add their sums over distributed shared memory: for few rows,
// where the weights' bytes and the latency count.  Neither needs a workspace.
#include <cooperative_groups.h>
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "lonnx_internal.cuh"
#include "tc_common.cuh"

namespace cg = cooperative_groups;

namespace {

using namespace lonnx::tc;

constexpr int KB = 128;  // columns of a block: one 128-byte row of the swizzled tiles
constexpr int BM = 128;  // rows of a tile on the tensor core
constexpr int kTile = BM * KB;  // bytes of 128 rows of one block

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ float activate(float v, int epi) {
    if (epi == LONNX_EPI_RELU) return v > 0.0f ? v : 0.0f;  // NaN gives 0, as lonnx_gemm_f32's
    return epi == LONNX_EPI_GELU_ERF ? lonnx_gelu_fast(v) : v;
}

// lonnx_gelu_fast of two values, with one reciprocal for both (1 / d0 = d1 / (d0
// d1)) and the multiplications and FMAs in pairs.  The clamp keeps the product
// finite; beyond it erf is +-1, and the last line has infinities and NaN.
__device__ __forceinline__ uint64_t pack2(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ void gelu2(float &x, float &y) {
    const uint64_t a = pack2(fminf(fabsf(x) * 0.707106769084930419921875f, 1e10f),
                             fminf(fabsf(y) * 0.707106769084930419921875f, 1e10f));
    const float2 d = unpack2(fma2(pack2(0.3275911f, 0.3275911f), a, pack2(1.0f, 1.0f)));
    float r, e0, e1;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d.x * d.y));
    const uint64_t t = pack2(r * d.y, r * d.x);
    const float2 q = unpack2(mul2(mul2(a, a), pack2(-1.44269504102162933349609375f, -1.44269504102162933349609375f)));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(q.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(q.y));
    uint64_t p = fma2(pack2(-1.061405429f, -1.061405429f), t, pack2(1.453152027f, 1.453152027f));
    p = fma2(p, t, pack2(-1.421413741f, -1.421413741f));
    p = fma2(p, t, pack2(0.284496736f, 0.284496736f));
    p = fma2(p, t, pack2(-0.254829592f, -0.254829592f));
    const float2 erf = unpack2(fma2(mul2(p, t), pack2(e0, e1), pack2(1.0f, 1.0f)));
    const uint64_t h = mul2(pack2(x, y), pack2(0.5f, 0.5f));
    const float2 g = unpack2(fma2(h, pack2(copysignf(erf.x, x), copysignf(erf.y, y)), h));
    x = g.x;
    y = g.y;
}

// D[tmem] (+)= A[smem desc] x B[smem desc], kind::f8f6f4 (32 columns of K), one CTA
__device__ __forceinline__ void mma_fp8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                        uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Instruction descriptor for kind::f8f6f4: D fp32 [4,6)=1, A and B e4m3
// ([7,10) and [10,13) = 0), both K-major, N >> 3 at [17,23), M >> 4 at [24,29).
__host__ __device__ constexpr uint32_t idesc_e4m3(int M, int N) {
    return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

// Four blocks' scales of one row, from block b (0 past the row's end)
__device__ __forceinline__ void load_scales(float (&s)[4], const float *row, int b, int nkb, bool valid) {
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = valid && b + i < nkb ? __ldg(row + b + i) : 0.0f;
}

// ---- wide tiles -----------------------------------------------------------------
//
// CTA = 20 warps, one per SM, walking tiles of 128 x BN:
//   warps 0-15   drain: each thread one row x 64 columns in registers (four
//                warps a scheduler: the TMEM loads of one hide behind the FMAs
//                of the others); then the epilogue, 128 bytes of a row at a
//                time through 4 KB of shared memory per warp and out by TMA (or,
//                where rows of C do not start and end on 16 bytes, by element
//                stores that coalesce along rows)
//   warp 16      TMA producer
//   warps 17, 18 MMA issuers of every other block (warp 17 has TMEM): one's waits
//                run while the other issues (a single issuer: 2048^3 in 14.5 us
//                instead of 13.0)
//   warp 19      the block's scales: sA[m, b] * sB[n / 128, b] of the tile's 128
//                rows and BN / 128 column blocks into shared memory, one slot
//                per TMEM buffer, under the same barriers
// BN = 256 has one set of 16 drain warps and two TMEM buffers.  BN = 128 has two
// sets of 8, with two buffers each, that take turns at tiles: the epilogue of
// one set runs beside the other's blocks.
// The drain warps take registers from the other four (setmaxnreg): 512 x 112 +
// 128 x 32 = 640 x 96, the launch's.
template <int BN>
struct Wide {
    static constexpr int STAGE = kTile + BN * KB;
    static constexpr int SETS = 256 / BN, BUFS = 2 * SETS;
    static constexpr int S = BN == 256 ? 3 : 4;
    static constexpr bool TURNS = S % 2 != 0;  // of the two issuers (see there)
    static constexpr int STAGING = 16 * 4096;  // 128 bytes x 32 rows per warp in the epilogue
    static constexpr int SCALES = BUFS * BN * 4;  // a slot per buffer: BN / 128 column blocks x 128 rows
    static constexpr int BARS = 2 * S + 2 * BUFS + 3;
    static constexpr int SMEM = S * STAGE + STAGING + SCALES + BARS * 8 + 8;
    static_assert(SMEM <= 227 * 1024, "shared memory of a CTA");
};
constexpr int kWideThreads = 640;
constexpr int W_TMA = 16, W_MMA = 17, W_SCALE = 19;

// Tiles in groups of `group` rows of tiles, column by column within a group, so
// that the CTAs at work share both operands' tiles in L2.  Where C leaves by
// element stores, its rows do not start on sectors, and neighbours' halves of a
// sector have to meet in L2: groups of 1 row where K is one or two blocks and C's
// bytes are all that counts (18651 x 17257 x 78 to floats: 341 us, 445 in groups
// of 4; to bfloat16: 227, 247, 299 in groups of 16), of 4 rows for longer K, where
// the operands' bytes count too (1000 x 30001 x 2000 to halves: 95 us, 99 row by
// row; 300 x 50001 x 1024 to floats: 38.5, 42).
__device__ __forceinline__ int tile_group(bool by_tma, int nkb) { return by_tma ? 16 : nkb <= 2 ? 1 : 4; }
__device__ __forceinline__ void tile_at(int t, int group, int tiles_m, int tiles_n, int &tm, int &tn) {
    const int per = group * tiles_n, g = t / per, first = g * group;
    const int h = min(group, tiles_m - first), r = t - g * per;
    tn = r / h;
    tm = first + r - tn * h;
}

template <int BN, typename T, bool BY_TMA>
__global__ void __launch_bounds__(kWideThreads, 1)
    k_fp8_wide(const __grid_constant__ CUtensorMap mapA, const __grid_constant__ CUtensorMap mapB,
               const __grid_constant__ CUtensorMap mapC, const float *__restrict__ sA, int64_t ldsA,
               const float *__restrict__ sB, int64_t ldsB, const float *__restrict__ bias, T *__restrict__ C,
               int64_t ldc, int M, int N, int nkb, int epi, int *flags) {
    using W = Wide<BN>;
    const int group = tile_group(BY_TMA, nkb);
    constexpr int S = W::S, SETS = W::SETS, COLS = 64;
    extern __shared__ __align__(1024) uint8_t base[];
    uint8_t *staging = base + S * W::STAGE;
    float *slots = reinterpret_cast<float *>(staging + W::STAGING);
    uint64_t *bar0 = reinterpret_cast<uint64_t *>(slots + W::BUFS * BN);
    const uint32_t bars = smem_u32(bar0);
    auto full = [&](int s) { return bars + 8 * s; };
    auto empty = [&](int s) { return bars + 8 * (S + s); };
    auto tfull = [&](int b) { return bars + 8 * (2 * S + b); };
    auto tempty = [&](int b) { return bars + 8 * (2 * S + W::BUFS + b); };
    auto turn = [&](int e) { return bars + 8 * (2 * S + 2 * W::BUFS + e); };
    const uint32_t drained = bars + 8 * (2 * S + 2 * W::BUFS + 2);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(bar0 + W::BARS);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bar0 + W::BARS) + 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        *abort_flag = 0;
        for (int s = 0; s < S; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
        }
        for (int b = 0; b < W::BUFS; ++b) {
            mbar_init(tfull(b), 1 + 32);  // the MMAs' commit and the scale warp's lanes
            mbar_init(tempty(b), 16 / SETS);
        }
        mbar_init(turn(0), 1);
        mbar_init(turn(1), 1);
        mbar_init(drained, 2);  // a commit of each MMA warp
        fence_mbar_init();
    }
    if (warp == W_MMA) {
        tmem_alloc(smem_u32(tmem_slot), 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // all 512 columns, which start at 0: a constant for the MMA's uniform registers
    constexpr uint32_t tmem = 0;

    const int tiles_m = (M + BM - 1) / BM, tiles_n = (N + BN - 1) / BN, tiles = tiles_m * tiles_n;
    bool ok = true;
    int issued = 0;  // TMA: stages filled
    if (warp >= 16) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 32;");
        if (warp == W_TMA) {
            if (lane == 0) {
                for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
                    int tm, tn;
                    tile_at(t, group, tiles_m, tiles_n, tm, tn);
                    for (int b = 0; b < nkb; ++b, ++issued) {
                        const int s = issued % S;
                        if (!mbar_wait(empty(s), ((issued / S) & 1) ^ 1, abort_flag)) { ok = false; break; }
                        const uint32_t at = smem_u32(base + s * W::STAGE);
                        mbar_arrive_expect_tx(full(s), W::STAGE);
                        tma_load_2d(at, &mapA, full(s), b * KB, tm * BM);
                        tma_load_2d(at + kTile, &mapB, full(s), b * KB, tn * BN);
                    }
                }
            }
        } else if (warp < W_SCALE) {
            // the whole warp walks the loop and one elected lane issues, so that
            // descriptors stay in uniform registers
            constexpr uint32_t idesc = idesc_e4m3(BM, BN);
            const uint64_t desc0 = smem_desc_sw128(smem_u32(base));
            // Issuer e takes blocks e, e + 2, .. of the ring's order.  A parity wait
            // must not be two phases ahead of its barrier, or it returns at once.
            // full(): loads land in any order, so a block may be there before the one
            // S earlier, in the same slot.  With S even that one was this issuer's,
            // which has waited for it; with S odd the issuers take turns at this wait
            // (turn), and it is always for the block after the last one seen.
            // tempty(): the block two before in its TMEM buffer is this issuer's own
            // or, where sets have an odd number of blocks, 5 or more before in the
            // ring, and this block's load waited for the MMAs up to S before it.
            const int e = warp - W_MMA;
            int js[2] = {0, 0}, i = 0;  // blocks of each set, blocks of all
            for (int t = blockIdx.x, n = 0; t < tiles && ok; t += gridDim.x, ++n) {
                const int set = SETS == 2 ? n & 1 : 0;
                int j = js[set];
                js[set] += nkb;
                for (int b = 0; b < nkb; ++b, ++j, ++i) {
                    if ((i & 1) != e) continue;
                    const int s = i % S, buf = 2 * set + (j & 1);
                    bool ready = (!W::TURNS || mbar_wait(turn(e), ((i >> 1) & 1) ^ (e ^ 1), abort_flag)) &&
                                 mbar_wait(full(s), (i / S) & 1, abort_flag);
                    if (W::TURNS) {
                        if (!__all_sync(0xffffffffu, ready)) { ok = false; break; }
                        if (lane == 0) mbar_arrive(turn(e ^ 1));
                    }
                    ready = ready && mbar_wait(tempty(buf), ((j >> 1) & 1) ^ 1, abort_flag);
                    if (!__all_sync(0xffffffffu, ready)) { ok = false; break; }
                    tc_fence_after();
                    const uint64_t da = desc0 + (uint32_t)(s * (W::STAGE / 16)), db = da + kTile / 16;
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < KB / 32; ++k) mma_fp8(tmem + buf * BN, da + 2 * k, db + 2 * k, idesc, k > 0);
                        mma_commit(empty(s));
                        mma_commit(tfull(buf));
                    }
                    __syncwarp();
                }
            }
        } else {
            // rows lane + 32 i of the tile; the next block's scales are loaded
            // before this one's slot is waited for
            constexpr int NB = BN / 128;
            int js[2] = {0, 0};  // blocks of each set
            for (int t = blockIdx.x, n = 0; t < tiles && ok; t += gridDim.x, ++n) {
                const int set = SETS == 2 ? n & 1 : 0;
                int tm, tn;
                tile_at(t, group, tiles_m, tiles_n, tm, tn);
                const float *ra[4], *rb[NB];
                float x[4], y[NB];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    ra[i] = sA + (int64_t)min(tm * BM + lane + 32 * i, M - 1) * ldsA;
                    x[i] = __ldg(ra[i]);
                }
#pragma unroll
                for (int i = 0; i < NB; ++i) {
                    // (a column block past N has no scales: its columns are not written)
                    rb[i] = sB + (int64_t)min(tn * NB + i, (N - 1) / KB) * ldsB;
                    y[i] = __ldg(rb[i]);
                }
                int j = js[set];
                js[set] += nkb;
                for (int b = 0; b < nkb; ++b, ++j) {
                    const int buf = 2 * set + (j & 1), nx = min(b + 1, nkb - 1);
                    if (!mbar_wait(tempty(buf), ((j >> 1) & 1) ^ 1, abort_flag)) { ok = false; break; }
                    float *slot = slots + buf * BN;
#pragma unroll
                    for (int n = 0; n < NB; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) slot[n * 128 + lane + 32 * i] = x[i] * y[n];
                    mbar_arrive(tfull(buf));
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] = __ldg(ra[i] + nx);
#pragma unroll
                    for (int i = 0; i < NB; ++i) y[i] = __ldg(rb[i] + nx);
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 112;");
        const int q = warp & 3, grp = warp >> 2;
        const int set = SETS == 2 ? grp >> 1 : 0, part = SETS == 2 ? grp & 1 : grp;  // 64 columns of the set's tile
        const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16) + 2 * set * BN + part * COLS;
        const bool bias4 = ((uintptr_t)bias & 15) == 0;
        const float *my_scale = slots + 2 * set * BN + part / 2 * 128 + q * 32 + lane;
        int j = 0;  // blocks of the set
        for (int t = blockIdx.x + set * gridDim.x; t < tiles && ok; t += SETS * gridDim.x) {
            float acc[COLS];
#pragma unroll
            for (int i = 0; i < COLS; ++i) acc[i] = 0.0f;
            for (int b = 0; b < nkb; ++b, ++j) {
                const int buf = j & 1;
                // (one answer for the warp: its next steps are collective)
                if (!__all_sync(0xffffffffu, mbar_wait(tfull(2 * set + buf), (j >> 1) & 1, abort_flag))) { ok = false; break; }
                tc_fence_after();
                const float s = my_scale[buf * BN];
#pragma unroll
                for (int c = 0; c < COLS / 32; ++c) {
                    uint32_t r[32];
                    tmem_ld_32x32b_x32(lanes + buf * BN + c * 32, r);
                    tmem_ld_wait();
                    if (c == COLS / 32 - 1) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(tempty(2 * set + buf));
                    }
#pragma unroll
                    for (int u = 0; u < 32; ++u) acc[c * 32 + u] = fmaf(__uint_as_float(r[u]), s, acc[c * 32 + u]);
                }
            }
            if (!ok) break;
            int tm, tn;
            tile_at(t, group, tiles_m, tiles_n, tm, tn);
            const int row0 = tm * BM + q * 32, col0 = tn * BN + part * COLS;
            // bias and activation of columns [i, i + 32), in place
            auto finish = [&](int i) {
                if (bias) {
                    if (bias4 && col0 + COLS <= N) {
#pragma unroll
                        for (int u = i; u < i + 32; u += 4) {
                            const float4 v = __ldg(reinterpret_cast<const float4 *>(bias + col0 + u));
                            acc[u] += v.x;
                            acc[u + 1] += v.y;
                            acc[u + 2] += v.z;
                            acc[u + 3] += v.w;
                        }
                    } else {
#pragma unroll
                        for (int u = i; u < i + 32; ++u) acc[u] += __ldg(bias + min(col0 + u, N - 1));
                    }
                }
                if (epi == LONNX_EPI_RELU) {
#pragma unroll
                    for (int u = i; u < i + 32; ++u) acc[u] = activate(acc[u], LONNX_EPI_RELU);
                } else if (epi == LONNX_EPI_GELU_ERF) {
#pragma unroll
                    for (int u = i; u < i + 32; u += 2) gelu2(acc[u], acc[u + 1]);
                }
            };
            constexpr int CN = 16 / (int)sizeof(T);
            auto pack = [&](int i) {  // 16 bytes of C from column i
                T out[CN];
#pragma unroll
                for (int u = 0; u < CN; ++u) out[u] = from_f32<T>(acc[i + u]);
                return *reinterpret_cast<const uint4 *>(out);
            };
            uint8_t *stage = staging + warp * 4096;
            if constexpr (BY_TMA) {
                // 128 bytes of each of the warp's 32 rows at a time: one piece is
                // computed in registers while the last one leaves shared memory
                constexpr int PIECE = 128 / (int)sizeof(T);
#pragma unroll
                for (int p = 0; p < COLS / PIECE; ++p) {
#pragma unroll
                    for (int i = p * PIECE; i < (p + 1) * PIECE; i += 32) finish(i);
                    if (lane == 0) bulk_wait_group_read0();
                    __syncwarp();
#pragma unroll
                    for (int c = 0; c < 8; ++c)  // 16-byte chunks of this lane's row, 128B-swizzled
                        *reinterpret_cast<uint4 *>(stage + lane * 128 + ((c ^ (lane & 7)) << 4)) = pack(p * PIECE + c * CN);
                    fence_proxy_async_smem();
                    __syncwarp();
                    const int col = col0 + p * PIECE;
                    if (lane == 0 && col < N && row0 < M) {
                        tma_store_2d(&mapC, smem_u32(stage), col, row0);
                        bulk_commit_group();
                    }
                }
            } else {
                // whole 64-column runs of a row by element stores, the warp along
                // the row, 4 KB of rows at a time and 8 rows in flight
                constexpr int ROW = COLS * (int)sizeof(T), TALL = 4096 / ROW;
                const int rows = M - row0;
#pragma unroll
                for (int h = 0; h < 32 / TALL; ++h) {
                    __syncwarp();
                    if (h == 0) {
#pragma unroll
                        for (int i = 0; i < COLS; i += 32) finish(i);
                    }
                    if (lane / TALL == h) {
#pragma unroll
                        for (int c = 0; c < COLS / CN; ++c)
                            *reinterpret_cast<uint4 *>(stage + lane % TALL * ROW + ((c ^ (lane & 7)) << 4)) = pack(c * CN);
                    }
                    __syncwarp();
                    T *dst = C + (int64_t)(row0 + h * TALL) * ldc + col0 + lane;
#pragma unroll
                    for (int r0 = 0; r0 < TALL; r0 += 8) {
                        T x[8][COLS / 32];
#pragma unroll
                        for (int r = 0; r < 8; ++r)
#pragma unroll
                            for (int e = 0; e < COLS / 32; ++e) {
                                const int i = lane + 32 * e;
                                x[r][e] = *reinterpret_cast<const T *>(stage + (r0 + r) * ROW + (((i / CN) ^ r) << 4) + i % CN * sizeof(T));
                            }
#pragma unroll
                        for (int r = 0; r < 8; ++r)
#pragma unroll
                            for (int e = 0; e < COLS / 32; ++e)
                                if (col0 + lane + 32 * e < N && h * TALL + r0 + r < rows) dst[(int64_t)(r0 + r) * ldc + 32 * e] = x[r][e];
                    }
                }
            }
        }
        if (lane == 0) bulk_wait_group0();
    }
    if (!ok) {
        *abort_flag = 1;
        atomicExch(flags + lonnx::FLAG_TIMEOUT, 8);
    }
    __syncthreads();
    if (*abort_flag) {
        // copies and MMAs in flight end before shared memory and TMEM go (bounded waits)
        if (warp == W_MMA || warp == W_MMA + 1) {
            if (elect_one()) mma_commit(drained);  // the lane that issued
            mbar_wait(drained, 0, nullptr, 400000000ll);
        }
        if (warp == W_TMA && lane == 0)
            for (int i = max(issued - S, 0); i < issued; ++i) mbar_wait(full(i % S), (i / S) & 1, nullptr, 400000000ll);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == W_MMA) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// ---- few rows: K split over a cluster ---------------------------------------------
//
// Tiles of 128 rows of B (the tensor core's rows) x TOK rows of A (its columns),
// each by a cluster of CTAs that take a run of K's blocks each; where one CTA
// takes all of K (parts = 1), it walks several tiles, the next one's loads
// running under the epilogue.
//   warps 0-3  drain: each thread one row of B x TOK sums in registers
//   warp 4     TMA producer, warp 5 MMA issuer (and TMEM)
// A thread writes consecutive elements of C's rows with its neighbours, so C
// needs no alignment.  The CTAs' sums meet in shared memory, TOK / parts rows of
// A to each CTA, added in the CTAs' order.
constexpr int kSplitThreads = 192;
// 1 x 4096 x 4096: 6.1 us (the weights' bytes need 2.6), latency of a launch, a
// load, the blocks' chain and the cluster's barriers; 32 x 250037 x 384 to floats:
// 27 us, 4.7 TB/s of weights and logits, whose rows start between sectors.
template <int TOK>
struct Split {
    static constexpr int STAGE = kTile + TOK * KB;
    static constexpr int TMEM = 2 * TOK < 32 ? 32 : 2 * TOK;
    static constexpr int SCALES = 4 * 4 * TOK * 4;  // 4 warps x 4 blocks
    static constexpr int MAX_STAGES = 12;
    static constexpr int BARS = 2 * MAX_STAGES + 5;
    static constexpr int PER_SM = TOK == 64 ? 2 : 3;  // CTAs, by registers
    static int smem(int stages, int parts) {
        return std::max(stages * STAGE, parts > 1 ? TOK * BM * 4 : 0) + SCALES + BARS * 8 + 8;
    }
    // as many stages as fit with `per_sm` CTAs on an SM: few CTAs have to keep more bytes in flight each
    static int stages(int blocks, int per_sm) {
        const int room = 227 * 1024 / per_sm - 1024 - SCALES - BARS * 8 - 8;
        return std::max(1, std::min({blocks, room / STAGE, MAX_STAGES}));
    }
};

template <typename T>
__device__ __forceinline__ void finish_store(T *C, int64_t at, float v, float bias, int epi) {
    C[at] = from_f32<T>(activate(v + bias, epi));
}

template <int TOK, typename T>
__global__ void __launch_bounds__(kSplitThreads, Split<TOK>::PER_SM)
    k_fp8_split(const __grid_constant__ CUtensorMap mapA, const __grid_constant__ CUtensorMap mapB,
                const float *__restrict__ sA, int64_t ldsA, const float *__restrict__ sB, int64_t ldsB,
                const float *__restrict__ bias, T *__restrict__ C, int64_t ldc, int M, int N, int nkb, int stages,
                int epi, int *flags) {
    using P = Split<TOK>;
    extern __shared__ __align__(1024) uint8_t base[];
    auto cluster = cg::this_cluster();
    const int parts = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
    float *sums = reinterpret_cast<float *>(base);  // parts > 1: [TOK][128], over the stages once they are read
    float *scales = reinterpret_cast<float *>(base + max(stages * P::STAGE, parts > 1 ? TOK * BM * 4 : 0));
    uint64_t *bar0 = reinterpret_cast<uint64_t *>(scales + 16 * TOK);
    const uint32_t bars = smem_u32(bar0);
    auto full = [&](int s) { return bars + 8 * s; };
    auto empty = [&](int s) { return bars + 8 * (P::MAX_STAGES + s); };
    auto tfull = [&](int b) { return bars + 8 * (2 * P::MAX_STAGES + b); };
    auto tempty = [&](int b) { return bars + 8 * (2 * P::MAX_STAGES + 2 + b); };
    const uint32_t drained = bars + 8 * (2 * P::MAX_STAGES + 4);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(bar0 + P::BARS);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bar0 + P::BARS) + 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tiles_n = (N + BM - 1) / BM, tiles_m = (M + TOK - 1) / TOK, tiles = tiles_n * tiles_m;
    // (parts > 1: the grid has a cluster for each tile)
    const int first_tile = blockIdx.x / parts, tile_step = gridDim.x / parts;
    const int b_first = (int)((int64_t)nkb * part / parts), b_last = (int)((int64_t)nkb * (part + 1) / parts);
    const int blocks = b_last - b_first;

    if (threadIdx.x == 0) {
        *abort_flag = 0;
        for (int s = 0; s < stages; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(tfull(b), 1);
            mbar_init(tempty(b), 4);
        }
        mbar_init(drained, 1);
        fence_mbar_init();
    }
    if (warp == 5) {
        tmem_alloc(smem_u32(tmem_slot), P::TMEM);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    bool ok = true;
    int issued = 0;
    if (warp == 4) {
        if (lane == 0) {
            for (int tile = first_tile, s = 0, phase = 1; tile < tiles && ok; tile += tile_step) {
                const int tm = tile / tiles_n, n0 = (tile - tm * tiles_n) * BM;
                for (int b = b_first; b < b_last; ++b, ++issued) {
                    if (!mbar_wait(empty(s), phase, abort_flag)) { ok = false; break; }
                    const uint32_t at = smem_u32(base + s * P::STAGE);
                    mbar_arrive_expect_tx(full(s), P::STAGE);
                    tma_load_2d(at, &mapB, full(s), b * KB, n0);
                    tma_load_2d(at + kTile, &mapA, full(s), b * KB, tm * TOK);
                    if (++s == stages) s = 0, phase ^= 1;
                }
            }
        }
    } else if (warp == 5) {
        constexpr uint32_t idesc = idesc_e4m3(BM, TOK);
        const uint64_t desc0 = smem_desc_sw128(smem_u32(base));
        const uint32_t d0 = __shfl_sync(0xffffffffu, tmem, 0);
        int j = 0;
        for (int tile = first_tile, s = 0, phase = 0; tile < tiles && ok; tile += tile_step) {
            for (int b = 0; b < blocks; ++b, ++j) {
                const int buf = j & 1;
                const bool ready = mbar_wait(tempty(buf), ((j >> 1) & 1) ^ 1, abort_flag) &&
                                   mbar_wait(full(s), phase, abort_flag);
                if (!__all_sync(0xffffffffu, ready)) { ok = false; break; }
                tc_fence_after();
                const uint64_t da = desc0 + (uint32_t)(s * (P::STAGE / 16)), db = da + kTile / 16;
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < KB / 32; ++k) mma_fp8(d0 + buf * TOK, da + 2 * k, db + 2 * k, idesc, k > 0);
                    mma_commit(empty(s));
                    mma_commit(tfull(buf));
                }
                __syncwarp();
                if (++s == stages) s = 0, phase ^= 1;
            }
        }
    } else {
        const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
        constexpr int PER = (TOK + 31) / 32;  // rows of A whose scales a lane fetches
        float *my = scales + warp * 4 * TOK;  // [4 blocks][TOK], this warp's copy
        int j = 0;
        for (int tile = first_tile; tile < tiles && ok; tile += tile_step) {
            const int tm = tile / tiles_n, n0 = (tile - tm * tiles_n) * BM, m0 = tm * TOK;
            const float *rb = sB + (int64_t)(n0 / KB) * ldsB;
            float acc[TOK];
#pragma unroll
            for (int i = 0; i < TOK; ++i) acc[i] = 0.0f;
            float na[PER][4], nb[4];
            auto fetch = [&](int b) {
#pragma unroll
                for (int p = 0; p < PER; ++p) {
                    const int m = m0 + lane + 32 * p;
                    const bool valid = m < M && lane + 32 * p < TOK;
                    load_scales(na[p], sA + (int64_t)(valid ? m : 0) * ldsA, b, b_last, valid);
                }
                load_scales(nb, rb, b, b_last, true);
            };
            fetch(b_first);
            for (int b0 = 0; b0 < blocks && ok; b0 += 4) {
                __syncwarp();
#pragma unroll
                for (int p = 0; p < PER; ++p)
                    if (lane + 32 * p < TOK)
#pragma unroll
                        for (int i = 0; i < 4; ++i) my[i * TOK + lane + 32 * p] = na[p][i] * nb[i];
                __syncwarp();
                fetch(b_first + b0 + 4);
                for (int i = 0; i < 4 && b0 + i < blocks; ++i, ++j) {
                    const int buf = j & 1;
                    // (one answer for the warp: its next steps are collective)
                    if (!__all_sync(0xffffffffu, mbar_wait(tfull(buf), (j >> 1) & 1, abort_flag))) { ok = false; break; }
                    tc_fence_after();
                    constexpr int CH = TOK < 32 ? TOK : 32;
#pragma unroll
                    for (int c = 0; c < TOK / CH; ++c) {
                        uint32_t r[CH];
                        if constexpr (CH == 16) tmem_ld_32x32b_x16(lanes + buf * TOK + c * CH, r);
                        else tmem_ld_32x32b_x32(lanes + buf * TOK + c * CH, r);
                        tmem_ld_wait();
                        if (c == TOK / CH - 1) {
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(tempty(buf));
                        }
                        const float4 *s4 = reinterpret_cast<const float4 *>(my + i * TOK + c * CH);
#pragma unroll
                        for (int u = 0; u < CH / 4; ++u) {
                            const float4 s = s4[u];
                            float *a = acc + c * CH + 4 * u;
                            a[0] = fmaf(__uint_as_float(r[4 * u]), s.x, a[0]);
                            a[1] = fmaf(__uint_as_float(r[4 * u + 1]), s.y, a[1]);
                            a[2] = fmaf(__uint_as_float(r[4 * u + 2]), s.z, a[2]);
                            a[3] = fmaf(__uint_as_float(r[4 * u + 3]), s.w, a[3]);
                        }
                    }
                }
            }
            if (!ok) break;
            if (parts > 1) {
                // the last block's MMAs have read the stages: the sums may go over them
#pragma unroll
                for (int i = 0; i < TOK; ++i) sums[i * BM + threadIdx.x] = acc[i];
            } else {
                const int n = n0 + threadIdx.x;
                if (n < N) {
                    const float bv = bias ? __ldg(bias + n) : 0.0f;
                    const int rows = M - m0;
#pragma unroll
                    for (int i = 0; i < TOK; ++i)
                        if (i < rows) finish_store(C, (int64_t)(m0 + i) * ldc + n, acc[i], bv, epi);
                }
            }
        }
    }
    if (!ok) {
        *abort_flag = 1;
        atomicExch(flags + lonnx::FLAG_TIMEOUT, 9);
    }
    __syncthreads();
    if (*abort_flag) {
        if (warp == 5) {
            if (elect_one()) mma_commit(drained);  // the lane that issued
            mbar_wait(drained, 0, nullptr, 400000000ll);
        }
        if (warp == 4 && lane == 0)
            for (int i = max(issued - stages, 0); i < issued; ++i)
                mbar_wait(full(i % stages), (i / stages) & 1, nullptr, 400000000ll);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 5) {
        // before the cluster's barrier: a CTA never holds TMEM while it waits for another CTA
        tc_fence_after();
        tmem_dealloc(tmem, P::TMEM);
    }
    if (parts > 1) {
        cluster.sync();
        const int tm = first_tile / tiles_n, n = (first_tile - tm * tiles_n) * BM + (int)threadIdx.x, m0 = tm * TOK;
        if (threadIdx.x < BM) {
            const int first = TOK * part / parts, last = min(TOK * (part + 1) / parts, M - m0);
            const float bv = bias && n < N ? __ldg(bias + n) : 0.0f;
            for (int m = first; m < last; m += 4) {
                float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
                for (int p = 0; p < parts; ++p) {
                    const float *of = cluster.map_shared_rank(sums, p) + m * BM + threadIdx.x;
#pragma unroll
                    for (int u = 0; u < 4; ++u) v[u] += m + u < last ? of[u * BM] : 0.0f;
                }
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (n < N && m + u < last) finish_store(C, (int64_t)(m0 + m + u) * ldc + n, v[u], bv, epi);
            }
        }
        cluster.sync();  // the others' shared memory is read until here
    }
}

// K = 0: the bias through the activation
template <typename T>
__global__ void k_fp8_no_columns(const float *__restrict__ bias, T *__restrict__ C, int64_t ldc, int M, int N, int epi) {
    const int64_t total = (int64_t)M * N, step = (int64_t)gridDim.x * blockDim.x;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += step) {
        const int64_t m = i / N, n = i - m * N;
        C[m * ldc + n] = from_f32<T>(activate(bias ? bias[n] : 0.0f, epi));
    }
}

// ---- host side ------------------------------------------------------------------

// row-major [rows, cols] of es-byte elements, leading dimension ld elements, box of 128 bytes x box_rows
int tile_map(CUtensorMap *map, const void *base, CUtensorMapDataType type, int es, int64_t rows, int64_t cols,
             int64_t ld, int box_rows) {
    lonnx::tc::EncodeTiledFn enc = lonnx::tc::encode_tiled();
    if (!enc) return lonnx::set_error(LONNX_E_CUDA, "cuTensorMapEncodeTiled unavailable");
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)ld * es};
    const cuuint32_t box[2] = {(cuuint32_t)(128 / es), (cuuint32_t)box_rows};
    const cuuint32_t estr[2] = {1, 1};
    const CUresult r = enc(map, type, 2, const_cast<void *>(base), dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return lonnx::set_error(LONNX_E_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return LONNX_OK;
}

struct Problem {
    const uint8_t *A, *B;
    const float *sA, *sB, *bias;
    void *C;
    int64_t lda, ldb, ldsA, ldsB, ldc;
    int dtype, M, N, K, epi;
};

template <int BN, typename T, bool BY_TMA>
int launch_wide(lonnx_ctx *ctx, const Problem &p) {
    using W = Wide<BN>;
    CUtensorMap ma, mb, mc;
    int rc = tile_map(&ma, p.A, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.M, p.K, p.lda, BM);
    if (!rc) rc = tile_map(&mb, p.B, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.N, p.K, p.ldb, BN);
    if (rc) return rc;
    mc = ma;  // unused unless BY_TMA
    if (BY_TMA) {
        const CUtensorMapDataType type = sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                         : p.dtype == LONNX_DT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                   : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
        rc = tile_map(&mc, p.C, type, (int)sizeof(T), p.M, p.N, p.ldc, 32);
        if (rc) return rc;
    }
    const int64_t tiles = (int64_t)((p.M + BM - 1) / BM) * ((p.N + BN - 1) / BN);
    if (tiles >= (1ll << 31) - 1024) return lonnx::set_error(LONNX_E_UNSUPPORTED, "gemm_fp8: too many tiles");
    auto kernel = k_fp8_wide<BN, T, BY_TMA>;
    static bool attr_set[64] = {false};
    if (!attr_set[ctx->device & 63]) {
        LONNX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, W::SMEM));
        attr_set[ctx->device & 63] = true;
    }
    kernel<<<(unsigned)std::min<int64_t>(tiles, ctx->num_sms), kWideThreads, W::SMEM, ctx->stream>>>(
        ma, mb, mc, p.sA, p.ldsA, p.sB, p.ldsB, p.bias, static_cast<T *>(p.C), p.ldc, p.M, p.N, (p.K + KB - 1) / KB,
        p.epi, ctx->dev_flags);
    LONNX_CHECK_LAUNCH(ctx);
    return LONNX_OK;
}

template <int BN, typename T>
int launch_wide(lonnx_ctx *ctx, const Problem &p) {
    // (a TMA store ends on 16 bytes: where N does not, it would write past the row's end)
    const bool by_tma = ((uintptr_t)p.C & 15) == 0 && p.ldc * (int64_t)sizeof(T) % 16 == 0 &&
                        p.N * (int64_t)sizeof(T) % 16 == 0;
    return by_tma ? launch_wide<BN, T, true>(ctx, p) : launch_wide<BN, T, false>(ctx, p);
}

template <int TOK, typename T>
int launch_split(lonnx_ctx *ctx, const Problem &p, int parts) {
    using P = Split<TOK>;
    CUtensorMap ma, mb;
    int rc = tile_map(&ma, p.A, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.M, p.K, p.lda, TOK);
    if (!rc) rc = tile_map(&mb, p.B, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.N, p.K, p.ldb, BM);
    if (rc) return rc;
    const int nkb = (p.K + KB - 1) / KB;
    const int64_t tiles = (int64_t)((p.N + BM - 1) / BM) * ((p.M + TOK - 1) / TOK);
    if (tiles > (1 << 27)) return lonnx::set_error(LONNX_E_UNSUPPORTED, "gemm_fp8: too many tiles");
    const int64_t grid = parts > 1 ? tiles * parts : std::min<int64_t>(tiles, (int64_t)ctx->num_sms * P::PER_SM);
    const int per_sm = (int)std::min<int64_t>(P::PER_SM, (grid + ctx->num_sms - 1) / ctx->num_sms);
    const int stages = P::stages((nkb + parts - 1) / parts, per_sm), smem = P::smem(stages, parts);
    auto kernel = k_fp8_split<TOK, T>;
    static bool attr_set[64] = {false};
    if (!attr_set[ctx->device & 63]) {
        LONNX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
        attr_set[ctx->device & 63] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(kSplitThreads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)parts;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    ctx->launches++;
    LONNX_CUDA(cudaLaunchKernelEx(&cfg, kernel, ma, mb, p.sA, p.ldsA, p.sB, p.ldsB, p.bias, static_cast<T *>(p.C), p.ldc,
                                  p.M, p.N, nkb, stages, p.epi, ctx->dev_flags));
    return LONNX_OK;
}

// Which kernel and tile: the least time by a model of both, in microseconds.
// Wide tiles take a time per block and one per epilogue, in rounds over the
// SMs; split ones a time per block, an addition of sums per cluster, and more
// where SMs get several CTAs.  Either takes at least its tiles' bytes through
// L2.  The constants are fitted to 24 shapes from 1 x 1000 x 8000 to 1000 x 20000
// x 300 in all 14 variants; the choice is within 3.5% of the best of them on
// average (e.g. 1 x 4096 x 4096: split 16 by 4 at 6.2 us, unsplit 10.7, wide
// 13.5; 777 x 1000 x 1111: wide 128 7.6, wide 256 9.9, split 64 9.1; 256 x 4096 x
// 4096: wide 128 15.3, split 64 18.3).
struct Choice {
    int width, parts;  // 256, 128: wide tiles; 64, 32, 16: rows of A of a split tile
};
Choice choose(int64_t M, int64_t N, int64_t K, int es, int sms) {
    const auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
    const double l2 = 7.5e6;  // bytes a microsecond
    const int64_t nkb = up(K, KB);
    Choice best{128, 1};
    double least = 1e30;
    const auto offer = [&](int width, int parts, double t) {
        if (t < least) {
            least = t;
            best = {width, parts};
        }
    };
    for (int bn : {256, 128}) {
        const int64_t tiles = up(M, BM) * up(N, bn), rounds = up(tiles, sms);
        const double block = bn == 256 ? 0.58 : tiles > sms ? 0.36 : 0.31;
        const double epilogue = bn == 256 ? (es == 4 ? 2.6 : 1.5) : (es == 4 ? 1.1 : 0.8);
        offer(bn, 1, std::max(rounds * (nkb * block + epilogue), tiles * nkb * double(kTile + bn * KB) / l2));
    }
    // CTAs that run at once in clusters of 1, 2, 4, 8 (a GPC has 16 to 18 SMs)
    const double at_once[4] = {1.0, 0.98, 0.89, 0.70};
    for (int tok : {16, 32, 64}) {
        const int64_t tiles = up(N, BM) * up(M, tok);
        const double block = tok == 16 ? 0.235 : tok == 32 ? 0.265 : 0.33, epilogue = tok == 64 ? 0.6 : 0.3;
        for (int i = 0; i < 4; ++i) {
            const int parts = 1 << i;
            if (parts > std::max<int64_t>(1, nkb / 2)) break;
            const int64_t rounds = up(tiles * parts, (int64_t)(sms * at_once[i]));
            const double t = up(nkb, parts) * block * (1 + 0.75 * (rounds - 1)) + epilogue * rounds;
            const double join = parts > 1 ? 1.4 + 2.0 * (rounds - 1) : 0.0;
            offer(tok, parts, std::max(t, tiles * nkb * double(kTile + tok * KB) / l2) + join);
        }
    }
    return best;
}

template <typename T>
int launch(lonnx_ctx *ctx, const Problem &p) {
    if (p.K == 0) {
        const int64_t total = (int64_t)p.M * p.N;
        k_fp8_no_columns<T><<<(unsigned)std::min<int64_t>((total + 255) / 256, ctx->num_sms * 16), 256, 0, ctx->stream>>>(
            p.bias, static_cast<T *>(p.C), p.ldc, p.M, p.N, p.epi);
        LONNX_CHECK_LAUNCH(ctx);
        return LONNX_OK;
    }
    const Choice c = choose(p.M, p.N, p.K, (int)sizeof(T), ctx->num_sms);
    switch (c.width) {
        case 256: return launch_wide<256, T>(ctx, p);
        case 128: return launch_wide<128, T>(ctx, p);
        case 64: return launch_split<64, T>(ctx, p, c.parts);
        case 32: return launch_split<32, T>(ctx, p, c.parts);
        default: return launch_split<16, T>(ctx, p, c.parts);
    }
}

}  // namespace

using namespace lonnx;

extern "C" LONNX_API int lonnx_gemm_fp8(lonnx_ctx *ctx, const void *A, int64_t lda, const float *scaleA, int64_t ldsA,
                                        const void *B, int64_t ldb, const float *scaleB, int64_t ldsB,
                                        const float *bias, void *C, int dtypeC, int64_t ldc, int M, int N, int K,
                                        int epilogue) {
    const int es = dtypeC == LONNX_DT_F32 ? 4 : dtypeC == LONNX_DT_F16 || dtypeC == LONNX_DT_BF16 ? 2 : 0;
    if (!es) return set_error(LONNX_E_UNSUPPORTED, "gemm_fp8: output type %d (float, float16 and bfloat16 are supported)", dtypeC);
    if (M < 0 || N < 0 || K < 0) return set_error(LONNX_E_BADARG, "gemm_fp8: negative size");
    if (M > 1 << 30 || N > 1 << 30 || K > 1 << 30)
        return set_error(LONNX_E_UNSUPPORTED, "gemm_fp8: %d x %d x %d (at most 2^30 each)", M, N, K);
    if (epilogue < LONNX_EPI_NONE || epilogue > LONNX_EPI_GELU_ERF)
        return set_error(LONNX_E_BADARG, "gemm_fp8: epilogue %d", epilogue);
    if (lda < K || ldb < K || ldc < N || ldsA < ((int64_t)K + KB - 1) / KB || ldsB < ((int64_t)K + KB - 1) / KB)
        return set_error(LONNX_E_SHAPE, "gemm_fp8: a leading dimension is smaller than its row");
    if (((uintptr_t)A & 15) || ((uintptr_t)B & 15) || lda % 16 || ldb % 16)
        return set_error(LONNX_E_BADARG, "gemm_fp8: rows of A and B must start on 16 bytes (pointers and leading dimensions)");
    if (((uintptr_t)C & (es - 1)) || ((uintptr_t)scaleA & 3) || ((uintptr_t)scaleB & 3) || ((uintptr_t)bias & 3))
        return set_error(LONNX_E_BADARG, "gemm_fp8: a pointer is not aligned to its element type");
    int rc = device_guard(ctx);
    if (rc) return rc;
    if (M == 0 || N == 0) return LONNX_OK;
    if (!C || (K > 0 && (!A || !B || !scaleA || !scaleB))) return set_error(LONNX_E_BADARG, "gemm_fp8: null pointer");
    const Problem p{static_cast<const uint8_t *>(A), static_cast<const uint8_t *>(B), scaleA, scaleB, bias, C,
                    lda, ldb, ldsA, ldsB, ldc, dtypeC, M, N, K, epilogue};
    if (dtypeC == LONNX_DT_F32) return launch<float>(ctx, p);
    if (dtypeC == LONNX_DT_F16) return launch<__half>(ctx, p);
    return launch<__nv_bfloat16>(ctx, p);
}
