// lonnx_token_logprobs: for each row x of logits over the vocabulary and
// z = x / T,
//
//   logprob = z[target] - lse(z)
//   entropy = lse(z) - E_p[z] = ln S - W / (S T)
//             S = sum exp((x - m) / T),  W = sum (x - m) exp((x - m) / T)
//   the k likeliest tokens, their log-probabilities, lowest index first where
//   values are equal
//
// in one pass over the row: a running maximum m with S and W rescaled when it
// grows, and a sorted list of the k best per warp.  All sums are fp32; a
// thread adds at most vocab / 256 terms, the rest is a tree.  x - m is taken
// before any scaling, so logits of the type's lowest value stay ordinary
// numbers; -inf adds exactly zero.
//
// Bound by HBM (each logit is read once, 16 bytes a thread and load).  Per
// element it issues about a load's share, a subtraction, a multiplication, a
// base-2 exponential, a clamp, a sum and an FMA; the list costs one comparison
// of 16 or 32 elements' maximum with the k-th best, and an insertion about
// k (1 + ln(vocab / k)) times a row.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cfloat>

#include "lonnx_internal.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int kMaxTop = 32;  // one list entry per lane
constexpr int U = 4;         // 16-byte loads in flight per thread
constexpr unsigned kAll = 0xffffffffu;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A float's bits in the order of its values (NaN below -inf, -0 as +0), never 0.
__device__ __forceinline__ uint32_t ordered(float v) {
    if (v != v) return 1u;
    const uint32_t b = __float_as_uint(v + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t o) {
    if (o == 1u) return __uint_as_float(0x7fc00000u);
    return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
// (value, lowest index first) as one number; 0 is "no entry"
__device__ __forceinline__ uint64_t make_key(float v, uint32_t idx) { return (uint64_t)ordered(v) << 32 | (uint32_t)~idx; }

struct Softmax {
    float m, s, w;  // w: sum of (x - m) e^((x - m) / T)
};

// b's sums added to a's, both to the larger maximum; c = log2(e) / T
__device__ __forceinline__ void rescale(Softmax &a, float m, float c) {
    const float d = a.m - m, f = ex2(d * c);
    // f == 0: the old terms vanish (d may be -inf there); * 0 keeps a NaN
    a.w = f == 0.0f ? a.w * 0.0f : f * fmaf(a.s, d, a.w);
    a.s *= f;
    a.m = m;
}
__device__ __forceinline__ void join(Softmax &a, Softmax b, float c) {
    const float m = fmaxf(a.m, b.m);
    if (a.m != m) rescale(a, m, c);
    if (b.m != m) rescale(b, m, c);
    a.s += b.s;
    a.w += b.w;
}

// Bitonic: 32 keys, one a lane, into descending order
__device__ __forceinline__ uint64_t sort_desc(uint64_t key, int lane) {
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int stride = size >> 1; stride > 0; stride >>= 1) {
            const uint64_t other = __shfl_xor_sync(kAll, key, stride);
            const bool keep_max = ((lane & size) == 0) == ((lane & stride) == 0);
            key = keep_max == (key > other) ? key : other;
        }
    return key;
}
// the best 32 of two descending lists, descending
__device__ __forceinline__ uint64_t merge_desc(uint64_t a, uint64_t b, int lane) {
    const uint64_t r = __shfl_sync(kAll, b, 31 - lane);
    uint64_t key = a > r ? a : r;
#pragma unroll
    for (int stride = 16; stride > 0; stride >>= 1) {
        const uint64_t other = __shfl_xor_sync(kAll, key, stride);
        key = ((lane & stride) == 0) == (key > other) ? key : other;
    }
    return key;
}

// What a warp has seen of its row.
template <bool TOP>
struct Warp {
    Softmax a;       // m is the same in every lane, s and w are the lane's
    uint64_t list;   // lane's entry of the descending list
    uint64_t kth;    // the k-th entry; 0 while there are fewer
    float thr;       // its value, NaN while there are fewer
    float c;
    int k;

    __device__ __forceinline__ void reset(float c_, int k_) {
        a = {-FLT_MAX, 0.0f, 0.0f};
        list = 0;
        kth = 0;
        thr = __uint_as_float(0x7fc00000u);
        c = c_;
        k = k_;
    }
    __device__ __forceinline__ void set_thr() {
        kth = __shfl_sync(kAll, list, k - 1);
        const uint32_t o = (uint32_t)(kth >> 32);
        thr = o ? unordered(o) : __uint_as_float(0x7fc00000u);
    }
    __device__ __forceinline__ void insert(uint64_t key, int lane) {
        const int p = __popc(__ballot_sync(kAll, list > key));
        if (p >= k) return;
        const uint64_t up = __shfl_up_sync(kAll, list, 1);
        list = lane < p ? list : lane == p ? key : up;
        set_thr();
    }
    __device__ __forceinline__ void add(float x) {
        const float d = x - a.m, e = ex2(d * c);
        a.s += e;
        a.w = fmaf(e, fmaxf(d, -FLT_MAX), a.w);  // d = -inf: e = 0, and 0 * -inf would be NaN
    }
    // N values a lane; value j has index idx(j), or is not there (valid(j) false)
    template <int N, typename Idx, typename Valid>
    __device__ __forceinline__ void take(const float (&x)[N], float best, bool first, int lane, const int *shared_thr,
                                         Idx idx, Valid valid) {
        bool slow = best > a.m;
        if (TOP && !(best <= thr))
            slow |= !shared_thr || !(best < unordered((uint32_t)*(volatile const int *)shared_thr));
        if (__any_sync(kAll, slow)) {
            float top = best;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kAll, top, o));
            if (top > a.m) rescale(a, top, c);
            if constexpr (TOP) {
                uint64_t mine = 0;
                if (first) {
                    // the lanes' best values, sorted, are the first list
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        const uint64_t key = valid(j) ? make_key(x[j], idx(j)) : 0;
                        mine = key > mine ? key : mine;
                    }
                    list = sort_desc(mine, lane);
                    set_thr();
                }
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const uint64_t key = make_key(x[j], idx(j));
                    unsigned todo = __ballot_sync(kAll, valid(j) && key > kth && key != mine);
                    while (todo) {
                        const int src = __ffs(todo) - 1;
                        todo &= todo - 1;
                        insert(__shfl_sync(kAll, key, src), lane);
                    }
                }
            }
        }
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (valid(j)) add(x[j]);
    }
};

struct Args {
    int64_t rows, ld;
    uint32_t vocab;
    const int64_t *targets;
    float inv_t;
    float *logprob, *entropy;
    int k;
    float *top_logprob;
    int64_t *top_id;
    int *flags;
};

// The row's answer from its sums and list: one warp, every lane with the same `a`.
template <typename T, bool TOP>
__device__ __forceinline__ void finish(const Args &g, const T *xr, int64_t row, const Softmax &a, uint64_t list,
                                       int lane) {
    const bool none = a.s == 0.0f;  // every logit -inf: no token has any probability
    const float log_s = logf(a.s);
    if (lane == 0) {
        if (g.targets && g.logprob) {
            const int64_t t = g.targets[row];
            float lp = __uint_as_float(0x7fc00000u);
            if (t < (int64_t)g.vocab)
                lp = none ? -INFINITY : fmaf(to_f32(xr[t]) - a.m, g.inv_t, -log_s);
            else
                atomicExch(g.flags + lonnx::FLAG_TARGET, 1);
            g.logprob[row] = lp;
        }
        if (g.entropy) g.entropy[row] = none ? 0.0f : log_s - a.w / a.s * g.inv_t;
    }
    if constexpr (TOP) {
        if (lane < g.k) {
            g.top_id[row * g.k + lane] = (int64_t)(uint32_t)~(uint32_t)list;
            g.top_logprob[row * g.k + lane] =
                none ? -INFINITY : fmaf(unordered((uint32_t)(list >> 32)) - a.m, g.inv_t, -log_s);
        }
    }
}

__device__ __forceinline__ bool padding(const Args &g, int64_t row) { return g.targets && g.targets[row] < 0; }

template <bool TOP>
__device__ __forceinline__ void finish_padding(const Args &g, int64_t row, int lane) {
    if (lane == 0) {
        if (g.logprob) g.logprob[row] = 0.0f;
        if (g.entropy) g.entropy[row] = 0.0f;
    }
    if constexpr (TOP)
        if (lane < g.k) {
            g.top_id[row * g.k + lane] = -1;
            g.top_logprob[row * g.k + lane] = -INFINITY;
        }
}

// Warp `w` of `nw` over one row: 16-byte vectors from the row's first aligned
// one in chunks of 32 * U, chunk i to warp i % nw; the elements before and
// after them (under 16 bytes each) to the last warp, one a lane.
template <typename T, bool TOP>
__device__ __forceinline__ void scan(Warp<TOP> &st, const T *xr, uint32_t vocab, int w, int nw, int lane,
                                     int *shared_thr) {
    constexpr int VN = 16 / (int)sizeof(T);
    const uint32_t head = min(vocab, (uint32_t)((16 - ((uintptr_t)xr & 15)) & 15) / (uint32_t)sizeof(T));
    const uint32_t nvec = (vocab - head) / VN, tail = vocab - head - nvec * VN;
    const uint4 *xv = reinterpret_cast<const uint4 *>(xr + head);
    bool first = true;
    for (uint32_t v0 = w * 32 * U; v0 < nvec; v0 += nw * 32 * U) {
        uint4 raw[U];
        const uint32_t at = v0 + lane;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (at + 32 * u < nvec) raw[u] = __ldcs(xv + at + 32 * u);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (v0 + 32 * u >= nvec) break;
            const bool in = at + 32 * u < nvec;
            float x[VN];
            const T *p = reinterpret_cast<const T *>(&raw[u]);
            float best = -INFINITY;
#pragma unroll
            for (int j = 0; j < VN; ++j) {
                x[j] = in ? to_f32(p[j]) : -INFINITY;
                best = fmaxf(best, x[j]);
            }
            const uint32_t i0 = head + (at + 32 * u) * VN;
            st.take(x, best, first, lane, shared_thr, [&](int j) { return i0 + j; }, [&](int) { return in; });
            first = false;
        }
        if (TOP && shared_thr && lane == 0 && st.thr == st.thr) atomicMax((unsigned *)shared_thr, ordered(st.thr));
    }
    if (w == nw - 1 && head + tail) {
        const bool in = lane < head || (lane >= 16 && lane - 16 < tail);
        const uint32_t idx = lane < 16 ? lane : head + nvec * VN + lane - 16;
        float x[1] = {in ? to_f32(xr[idx]) : -INFINITY};
        // the head's indices are below the list's: no shortcut for equal values
        const float thr = st.thr;
        if (TOP && in && x[0] == thr) st.thr = __uint_as_float(0x7fc00000u);
        st.take(x, x[0], first, lane, nullptr, [&](int) { return idx; }, [&](int) { return in; });
    }
}

// A warp per row
template <typename T, bool TOP>
__global__ void __launch_bounds__(256) k_logprobs_warp(const T *__restrict__ x, Args g) {
    const int lane = threadIdx.x & 31;
    for (int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); row < g.rows; row += (int64_t)gridDim.x * 8) {
        if (padding(g, row)) {
            finish_padding<TOP>(g, row, lane);
            continue;
        }
        const T *xr = x + row * g.ld;
        const float c = g.inv_t * 1.44269504088896340736f;
        Warp<TOP> st;
        st.reset(c, g.k);
        scan<T, TOP>(st, xr, g.vocab, 0, 1, lane, nullptr);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            st.a.s += __shfl_xor_sync(kAll, st.a.s, o);
            st.a.w += __shfl_xor_sync(kAll, st.a.w, o);
        }
        finish<T, TOP>(g, xr, row, st.a, st.list, lane);
    }
}

// A cluster of CTAs per row (one CTA without cluster launch): the warps' sums
// and lists meet in the CTA's shared memory, the CTAs' in the first CTA's warp
// 0, which reads the others' over distributed shared memory.  No workspace.
template <typename T, bool TOP>
__global__ void __launch_bounds__(256) k_logprobs_cta(const T *__restrict__ x, Args g) {
    constexpr int NW = 8;
    __shared__ Softmax sums[NW];
    __shared__ uint64_t lists[NW][32];
    __shared__ Softmax cta_sums;
    __shared__ uint64_t cta_list[32];
    __shared__ int thr;
    auto cluster = cg::this_cluster();
    const int parts = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const float c = g.inv_t * 1.44269504088896340736f;
    for (int64_t row = blockIdx.x / parts; row < g.rows; row += gridDim.x / parts) {
        if (padding(g, row)) {
            if (part == 0 && w == 0) finish_padding<TOP>(g, row, lane);
            continue;
        }
        const T *xr = x + row * g.ld;
        if (threadIdx.x == 0) thr = 0;
        __syncthreads();
        Warp<TOP> st;
        st.reset(c, g.k);
        scan<T, TOP>(st, xr, g.vocab, part * NW + w, parts * NW, lane, &thr);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            st.a.s += __shfl_xor_sync(kAll, st.a.s, o);
            st.a.w += __shfl_xor_sync(kAll, st.a.w, o);
        }
        if (lane == 0) sums[w] = st.a;
        if constexpr (TOP) lists[w][lane] = st.list;
        __syncthreads();
        if (w == 0) {
#pragma unroll
            for (int i = 1; i < NW; ++i) {
                join(st.a, sums[i], c);
                if constexpr (TOP) st.list = merge_desc(st.list, lists[i][lane], lane);
            }
            if (parts > 1) {
                if (lane == 0) cta_sums = st.a;
                if constexpr (TOP) cta_list[lane] = st.list;
            }
        }
        if (parts > 1) {
            cluster.sync();
            if (part == 0 && w == 0) {
                for (int i = 1; i < parts; ++i) {
                    join(st.a, *cluster.map_shared_rank(&cta_sums, i), c);
                    if constexpr (TOP) st.list = merge_desc(st.list, cluster.map_shared_rank(cta_list, i)[lane], lane);
                }
            }
            cluster.sync();  // the others' shared memory is read until here
        } else {
            __syncthreads();
        }
        if (part == 0 && w == 0) finish<T, TOP>(g, xr, row, st.a, st.list, lane);
    }
}

template <typename T, bool TOP>
int launch(lonnx_ctx *ctx, const void *xv, const Args &g) {
    const T *x = static_cast<const T *>(xv);
    const int64_t row_bytes = (int64_t)g.vocab * (int)sizeof(T);
    // Up to one chunk's worth a warp of a CTA, a warp has a row of its own.
    if (row_bytes <= 8192) {
        const unsigned grid = (unsigned)std::min<int64_t>((g.rows + 7) / 8, 1 << 30);
        k_logprobs_warp<T, TOP><<<grid, 256, 0, ctx->stream>>>(x, g);
        LONNX_CHECK_LAUNCH(ctx);
        return LONNX_OK;
    }
    // Few rows: as many CTAs to a row as fill the SMs twice, while each still has 16 KB to read.
    int parts = 1;
    while (parts < 16 && g.rows * parts < 2 * ctx->num_sms && row_bytes / (parts * 2) >= 16384) parts *= 2;
    auto kernel = k_logprobs_cta<T, TOP>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(std::min<int64_t>(g.rows, (1 << 30) / parts) * parts));
    cfg.blockDim = dim3(256);
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)parts;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (parts > 8)
        LONNX_CUDA(cudaFuncSetAttribute((const void *)kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    ctx->launches++;
    LONNX_CUDA(cudaLaunchKernelEx(&cfg, kernel, x, g));
    return LONNX_OK;
}

template <typename T>
int launch_top(lonnx_ctx *ctx, const void *x, const Args &g) {
    return g.k ? launch<T, true>(ctx, x, g) : launch<T, false>(ctx, x, g);
}

}  // namespace

using namespace lonnx;

extern "C" LONNX_API int lonnx_token_logprobs(lonnx_ctx *ctx, const void *logits, int dtype, int64_t rows,
                                              int64_t vocab, int64_t ld, const int64_t *targets, float temperature,
                                              float *logprob, float *entropy, int k, float *top_logprob,
                                              int64_t *top_id) {
    const int es = dtype == LONNX_DT_F32 ? 4 : dtype == LONNX_DT_F16 || dtype == LONNX_DT_BF16 ? 2 : 0;
    if (!es) return set_error(LONNX_E_UNSUPPORTED, "token_logprobs: logits of type %d (float, float16 and bfloat16 are supported)", dtype);
    if (rows < 0 || vocab < 1 || vocab > (1ll << 30))
        return set_error(LONNX_E_BADARG, "token_logprobs: %lld rows of %lld tokens (1 to 2^30 tokens are supported)", (long long)rows, (long long)vocab);
    if (ld < vocab) return set_error(LONNX_E_SHAPE, "token_logprobs: rows of %lld tokens %lld apart", (long long)vocab, (long long)ld);
    if (!(temperature >= 1e-3f && temperature <= 1e3f))
        return set_error(LONNX_E_BADARG, "token_logprobs: temperature %g outside [0.001, 1000]", (double)temperature);
    if (k < 0 || k > kMaxTop || k > vocab)
        return set_error(LONNX_E_BADARG, "token_logprobs: %d alternatives (0 to %d, at most the vocabulary)", k, kMaxTop);
    if ((uintptr_t)logits & (es - 1)) return set_error(LONNX_E_BADARG, "token_logprobs: logits not aligned to their element type");
    if (((uintptr_t)targets & 7) || ((uintptr_t)top_id & 7) || ((uintptr_t)logprob & 3) || ((uintptr_t)entropy & 3) || ((uintptr_t)top_logprob & 3))
        return set_error(LONNX_E_BADARG, "token_logprobs: a pointer is not aligned to its element type");
    if (rows > 0 && (!logits || (k && (!top_logprob || !top_id)) || (logprob && !targets)))
        return set_error(LONNX_E_BADARG, "token_logprobs: null pointer");
    int rc = device_guard(ctx);
    if (rc) return rc;
    if (rows == 0) return LONNX_OK;
    const Args g{rows, ld, (uint32_t)vocab, targets, 1.0f / temperature, logprob, entropy, k, top_logprob, top_id, ctx->dev_flags};
    if (dtype == LONNX_DT_F32) return launch_top<float>(ctx, logits, g);
    if (dtype == LONNX_DT_F16) return launch_top<__half>(ctx, logits, g);
    return launch_top<__nv_bfloat16>(ctx, logits, g);
}
