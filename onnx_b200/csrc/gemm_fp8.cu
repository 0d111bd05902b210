// lonnx_gemm_fp8: C = act(A . B^T + bias) with A [M, K] and B [N, K] in e4m3
// and one fp32 scale per 1 x 128 block of A and per 128 x 128 block of B:
//
//   C[m, n] = act(sum_b sA[m, b] * sB[n / 128, b] * sum_{k in block b} A[m, k] B[n, k] + bias[n])
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>

#include "lonnx_internal.cuh"

namespace {

constexpr int KB = 128;

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ float from_e4m3(uint8_t b) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(b, __NV_E4M3)));
}

// A 16 x 16 tile of C per CTA, one element per thread, one 128-block at a time
template <typename T>
__global__ void __launch_bounds__(256) k_gemm_fp8_plain(const uint8_t *__restrict__ A, int64_t lda,
                                                        const float *__restrict__ sA, int64_t ldsA,
                                                        const uint8_t *__restrict__ B, int64_t ldb,
                                                        const float *__restrict__ sB, int64_t ldsB,
                                                        const float *__restrict__ bias, T *__restrict__ C, int64_t ldc,
                                                        int M, int N, int K, int epi) {
    __shared__ float ta[16][KB + 1], tb[16][KB + 1];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int m = blockIdx.y * 16 + ty, n = blockIdx.x * 16 + tx;
    float acc = 0.0f;
    for (int b = 0; b * KB < K; ++b) {
        for (int i = threadIdx.x; i < 16 * KB; i += 256) {
            const int r = i / KB, c = b * KB + i % KB;
            const int64_t ra = blockIdx.y * 16 + r, rb = blockIdx.x * 16 + r;
            ta[r][i % KB] = ra < M && c < K ? from_e4m3(A[ra * lda + c]) : 0.0f;
            tb[r][i % KB] = rb < N && c < K ? from_e4m3(B[rb * ldb + c]) : 0.0f;
        }
        __syncthreads();
        float part = 0.0f;
        for (int k = 0; k < KB; ++k) part = fmaf(ta[ty][k], tb[tx][k], part);
        if (m < M && n < N) acc = fmaf(part, sA[m * ldsA + b] * sB[(int64_t)(n / KB) * ldsB + b], acc);
        __syncthreads();
    }
    if (m < M && n < N) {
        if (bias) acc += bias[n];
        if (epi == LONNX_EPI_RELU) acc = acc > 0.0f ? acc : 0.0f;
        else if (epi == LONNX_EPI_GELU_ERF) acc = lonnx_gelu_fast(acc);
        C[m * ldc + n] = from_f32<T>(acc);
    }
}

template <typename T>
int gemm_fp8(lonnx_ctx *ctx, const uint8_t *A, int64_t lda, const float *sA, int64_t ldsA, const uint8_t *B,
             int64_t ldb, const float *sB, int64_t ldsB, const float *bias, void *C, int64_t ldc, int M, int N, int K,
             int epi) {
    const dim3 grid((N + 15) / 16, (M + 15) / 16);
    k_gemm_fp8_plain<T><<<grid, 256, 0, ctx->stream>>>(A, lda, sA, ldsA, B, ldb, sB, ldsB, bias, static_cast<T *>(C),
                                                      ldc, M, N, K, epi);
    LONNX_CHECK_LAUNCH(ctx);
    return LONNX_OK;
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
    if (epilogue < LONNX_EPI_NONE || epilogue > LONNX_EPI_GELU_ERF)
        return set_error(LONNX_E_BADARG, "gemm_fp8: epilogue %d", epilogue);
    if (lda < K || ldb < K || ldc < N || ldsA < (K + KB - 1) / KB || ldsB < (K + KB - 1) / KB)
        return set_error(LONNX_E_SHAPE, "gemm_fp8: a leading dimension is smaller than its row");
    if (((uintptr_t)A & 15) || ((uintptr_t)B & 15) || lda % 16 || ldb % 16)
        return set_error(LONNX_E_BADARG, "gemm_fp8: rows of A and B must start on 16 bytes (pointers and leading dimensions)");
    if (((uintptr_t)C & (es - 1)) || ((uintptr_t)scaleA & 3) || ((uintptr_t)scaleB & 3) || ((uintptr_t)bias & 3))
        return set_error(LONNX_E_BADARG, "gemm_fp8: a pointer is not aligned to its element type");
    int rc = device_guard(ctx);
    if (rc) return rc;
    if (M == 0 || N == 0) return LONNX_OK;
    if (!C || (K > 0 && (!A || !B || !scaleA || !scaleB))) return set_error(LONNX_E_BADARG, "gemm_fp8: null pointer");
    const uint8_t *a = static_cast<const uint8_t *>(A), *b = static_cast<const uint8_t *>(B);
    if (dtypeC == LONNX_DT_F32)
        return gemm_fp8<float>(ctx, a, lda, scaleA, ldsA, b, ldb, scaleB, ldsB, bias, C, ldc, M, N, K, epilogue);
    if (dtypeC == LONNX_DT_F16)
        return gemm_fp8<__half>(ctx, a, lda, scaleA, ldsA, b, ldb, scaleB, ldsB, bias, C, ldc, M, N, K, epilogue);
    return gemm_fp8<__nv_bfloat16>(ctx, a, lda, scaleA, ldsA, b, ldb, scaleB, ldsB, bias, C, ldc, M, N, K, epilogue);
}
