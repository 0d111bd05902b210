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
// grows, and a sorted list of the k best groups of elements per warp.  All sums
// are fp32: 64 terms of a thread in turn, which then go into the thread's total
// with what that addition rounded off kept beside it, and a tree over threads.  So
// the error does not grow with the vocabulary, nor with the elements that a
// thread gets (a warp's row of 250037 equal logits under one peak: S is off by up
// to 4e-6; by 2e-4 where all 3900 terms are added to one fp32 number).  x - m is
// taken before any scaling, so logits of the type's lowest value stay ordinary
// numbers; -inf adds exactly zero.
//
// The alternatives.  A group is what one lane loads at once, 64 bytes of a row;
// its key is its best element under (value, lowest index first).  The k best
// elements lie in the k groups of the best keys, so the scan lists groups, with
// one comparison per 64 bytes and lane, and the elements of the k listed groups
// are read again at the end.  A key holds the group's first index instead of its
// best element's unless two groups of a chunk enter with the same value: chunks
// are runs of the row, so between chunks either index gives the same order.  (A
// list of elements took a comparison each and four times the insertions: one row
// of 250037 floats with 20 alternatives took 33 us instead of 18, and 11 since
// the warps share what they have reached and join in halves.)
//
// Bound by HBM (each logit is read once, 16 bytes a thread and load, the next
// 64 bytes in flight while the last are summed).  Pairs of elements share their
// additions, multiplications and FMAs (f32x2); per element that leaves about
// 5 instructions and one base-2 exponential.  2048 x 250037 floats: 305 us
// (6.7 TB/s), with 20 alternatives 330; bfloat16 172 us (6.0 TB/s), with 20
// alternatives 222, where instructions for the lists bound it (4000 x 60000 floats
// with 20: 178 us, 5.4 TB/s); short rows are bound by a row's chain of loads and
// reductions (16384 x 1001 halves: 12.6 us, with 20 alternatives 34).  Folding the
// sums costs long rows 1 to 4% of that.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cfloat>
#include <type_traits>

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

// two fp32 operations in one instruction
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
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
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

// With t = (x - m) c, c = log2(e) / T: s = sum of 2^t, w = sum of t 2^t
struct Softmax {
    float m, s, w;
};

// a's sums to a larger maximum
__device__ __forceinline__ void rescale(Softmax &a, float m, float c) {
    const float t = (a.m - m) * c, f = ex2(t);
    // f == 0: the old terms vanish (t may be -inf there); * 0 keeps a NaN
    a.w = f == 0.0f ? a.w * 0.0f : f * fmaf(a.s, t, a.w);
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

// A row's vectors: 16-byte ones from the first aligned element, the elements
// before and after them (under 16 bytes each).  Groups are U vectors, 32 apart,
// of a chunk of 32 * U.
template <typename T>
struct Row {
    static constexpr int VN = 16 / (int)sizeof(T), N = U * VN;
    const T *x;
    const uint4 *v;
    uint32_t vocab, head, nvec, tail;
    __device__ __forceinline__ Row(const T *x_, uint32_t vocab_) : x(x_), vocab(vocab_) {
        head = min(vocab, (uint32_t)((16 - ((uintptr_t)x & 15)) & 15) / (uint32_t)sizeof(T));
        nvec = (vocab - head) / VN;
        tail = vocab - head - nvec * VN;
        v = reinterpret_cast<const uint4 *>(x + head);
    }
    // vectors at + 32 u, -inf past the end
    __device__ __forceinline__ void load(uint4 (&r)[U], uint32_t at) const {
        const uint32_t inf = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
#pragma unroll
        for (int u = 0; u < U; ++u) r[u] = at + 32 * u < nvec ? __ldcs(v + at + 32 * u) : make_uint4(inf, inf, inf, inf);
    }
    // two elements of a vector as floats
    static __device__ __forceinline__ float2 pair(const uint4 &r, int i) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
        if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
        else if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        else return make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    }
    // the largest element, NaN aside
    static __device__ __forceinline__ float best(const uint4 (&r)[U]) {
        if constexpr (sizeof(T) == 4) {
            float m = -INFINITY;
#pragma unroll
            for (int u = 0; u < U; ++u)
                m = fmaxf(fmaxf(m, fmaxf(__uint_as_float(r[u].x), __uint_as_float(r[u].y))),
                          fmaxf(__uint_as_float(r[u].z), __uint_as_float(r[u].w)));
            return m;
        } else {
            using T2 = std::conditional_t<std::is_same<T, __half>::value, __half2, __nv_bfloat162>;
            const T2 *p = reinterpret_cast<const T2 *>(r);
            T2 m = p[0];
#pragma unroll
            for (int i = 1; i < U * 4; ++i) m = __hmax2(m, p[i]);
            const float a = to_f32(m.x), b = to_f32(m.y);
            return fmaxf(fmaxf(a, b), -INFINITY);
        }
    }
    __device__ __forceinline__ uint32_t index(uint32_t at, int j) const { return head + (at + 32 * (j / VN)) * VN + j % VN; }
    // the best element's key (a NaN's where there is nothing else)
    __device__ __forceinline__ uint64_t best_key(const uint4 (&r)[U], float best, uint32_t at) const {
        uint32_t idx = index(at, 0);
        bool any = false;
#pragma unroll
        for (int j = N - 1; j >= 0; --j) {
            const float2 p = pair(r[j / VN], j % VN / 2);
            if ((j & 1 ? p.y : p.x) == best && at + 32 * (j / VN) < nvec) {
                idx = index(at, j);
                any = true;
            }
        }
        return make_key(any ? best : __uint_as_float(0x7fc00000u), idx);
    }
};

// The k best of a descending list and the keys of the lanes in `todo`, descending
// (and perhaps more after them).  (Not inlined: it is called where few warps go,
// and its code would be many times the scan's.)
__device__ __noinline__ uint64_t with_keys(uint64_t list, uint64_t key, unsigned todo, int k, int lane) {
    const int n = __popc(todo);
    if (n > k && k <= 12) {
        // k times the best of all: a k-th of the work of an insertion for each key
        if (!(todo >> lane & 1)) key = 0;
        uint64_t mine = 0;
        for (int i = 0; i < k; ++i) {
            const bool from_list = list > key;
            const uint64_t cand = from_list ? list : key;
            const uint32_t hi = __reduce_max_sync(kAll, (uint32_t)(cand >> 32));
            const uint32_t lo = __reduce_max_sync(kAll, (uint32_t)(cand >> 32) == hi ? (uint32_t)cand : 0u);
            const uint64_t won = (uint64_t)hi << 32 | lo;
            if (cand == won) {  // (keys differ; 0, no entry, may stay)
                if (from_list) list = 0;
                else key = 0;
            }
            if (lane == i) mine = won;
        }
        return mine;
    }
    // sorting and merging cost about as much as 6 single insertions
    if (n > 6) {
        key = sort_desc(todo >> lane & 1 ? key : 0, lane);
        return __any_sync(kAll, list != 0) ? merge_desc(list, key, lane) : key;
    }
    while (todo) {
        const int src = __ffs(todo) - 1;
        todo &= todo - 1;
        const uint64_t one = __shfl_sync(kAll, key, src);
        const int p = __popc(__ballot_sync(kAll, list > one));
        const uint64_t up = __shfl_up_sync(kAll, list, 1);
        list = lane < p ? list : lane == p ? one : up;
    }
    return list;
}

// What a warp has seen of its row.  LONG: a lane may get more than 64 terms in
// each half, so its sums are folded (short rows do without: 16384 x 1001 halves,
// 2000 of them padding, 11.7 us instead of 12.5).
template <bool TOP, bool LONG>
struct Warp {
    float m;            // running maximum, the same in every lane
    uint64_t s2, w2;    // the lane's sums since the last fold, in two halves
    uint64_t list;      // lane's entry of the descending list of groups
    uint64_t kth;       // the k-th entry; 0 while there are fewer
    float thr;          // its value, NaN while there are fewer
    float c;
    int k;

    __device__ __forceinline__ void reset(float c_, int k_) {
        m = -FLT_MAX;
        s2 = w2 = list = kth = 0;
        if constexpr (LONG) before() = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        thr = __uint_as_float(0x7fc00000u);
        c = c_;
        k = k_;
    }
    // keys of lanes in `todo` into the list
    __device__ __forceinline__ void insert(uint64_t key, unsigned todo, int lane) {
        list = with_keys(list, key, todo, k, lane);
        kth = __shfl_sync(kAll, list, k - 1);
        const uint32_t o = (uint32_t)(kth >> 32);
        thr = o ? unordered(o) : __uint_as_float(0x7fc00000u);
    }
    // the lane's sums before the last fold: s, w, and what their additions rounded
    // off (in shared memory: they are touched every 64 terms, and registers are short)
    static __device__ __forceinline__ float4 &before() {
        __shared__ float4 all[256];
        return all[threadIdx.x];
    }
    // a + x with its rounding added to l
    static __device__ __forceinline__ void add_exact(float &a, float &l, float x) {
        const float t = a + x, b = t - a;
        l += (a - (t - b)) + (x - b);
        a = t;
    }
    // all sums so far, the last ones added
    __device__ __forceinline__ float4 folded() {
        const float2 a = unpack2(s2), b = unpack2(w2);
        float4 f = before();
        add_exact(f.x, f.z, a.x + a.y);
        add_exact(f.y, f.w, b.x + b.y);
        s2 = w2 = 0;
        return f;
    }
    __device__ __forceinline__ void fold() { before() = folded(); }
    __device__ __forceinline__ void raise(float best) {
        const float top = unordered(__reduce_max_sync(kAll, ordered(best)));
        if constexpr (LONG) {
            const float4 f = folded();
            Softmax a{m, f.x, f.y}, l{m, f.z, f.w};
            rescale(a, top, c);
            rescale(l, top, c);
            before() = make_float4(a.s, a.w, l.s, l.w);
        } else {
            const float2 s = unpack2(s2), w = unpack2(w2);
            Softmax a{m, s.x, w.x}, b{m, s.y, w.y};
            rescale(a, top, c);
            rescale(b, top, c);
            s2 = pack2(a.s, b.s);
            w2 = pack2(a.w, b.w);
        }
        m = top;
    }
    __device__ __forceinline__ void add(float x, float y) {
        const uint64_t t = mul2(add2(pack2(x, y), pack2(-m, -m)), pack2(c, c));
        const float2 u = unpack2(t);
        // -inf: 2^t = 0, and 0 * -inf would be NaN; a NaN stays in s
        const uint64_t e = pack2(ex2(u.x), ex2(u.y));
        s2 = add2(s2, e);
        w2 = fma2(e, pack2(fmaxf(u.x, -FLT_MAX), fmaxf(u.y, -FLT_MAX)), w2);
    }
    template <typename T>
    __device__ __forceinline__ void sum(const Row<T> &, const uint4 (&raw)[U], uint32_t left) {  // of the row, for the warp
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (32 * u >= left) break;
#pragma unroll
            for (int i = 0; i < Row<T>::VN / 2; ++i) {
                const float2 p = Row<T>::pair(raw[u], i);
                add(p.x, p.y);
            }
        }
    }
    // A group: `best` its largest element, first its first index, exact() its best
    // element's key, `here` whether the lane has one.  It can enter the list if it
    // is above the k-th entry, and not below `floor`, which k groups of the row are
    // known to reach.  True if the list changed.
    template <typename Key>
    __device__ __forceinline__ bool offer(float best, bool here, float floor, int lane, uint32_t first, Key exact) {
        const bool enters = TOP && here && !(best <= thr) && !(best < floor), higher = best > m;
        if (!__any_sync(kAll, enters || higher)) return false;
        if (__any_sync(kAll, higher)) raise(best);
        if constexpr (TOP) {
            const unsigned todo = __ballot_sync(kAll, enters);
            if (todo) {
                // (-inf: the group may have nothing but NaN)
                bool alike = false;
                if (enters) {  // (every lane of `todo` takes part in the match)
                    const unsigned same = __match_any_sync(todo, best + 0.0f);
                    alike = same != 1u << lane || best == -INFINITY;
                }
                const uint64_t key = __any_sync(kAll, alike) ? exact() : make_key(best, first);
                insert(key, todo, lane);
            }
            return todo != 0;
        }
        return false;
    }
    // the warp's sums, the same in every lane
    __device__ __forceinline__ Softmax total() {
        Softmax a{m, 0.0f, 0.0f};
        if constexpr (LONG) {
            const float4 f = folded();
            a.s = f.x + f.z;
            a.w = f.y + f.w;
        } else {
            const float2 s = unpack2(s2), w = unpack2(w2);
            a.s = s.x + s.y;
            a.w = w.x + w.y;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            a.s += __shfl_xor_sync(kAll, a.s, o);
            a.w += __shfl_xor_sync(kAll, a.w, o);
        }
        return a;
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

// The list of groups to one of elements: lanes with `group` hold theirs in `raw`
// (vectors at + 32 u, no warp's beyond 32 u >= left), others the key of a group of
// one element or 0 in `single`.
template <typename T, bool LONG>
__device__ __forceinline__ void list_elements(Warp<true, LONG> &st, const Row<T> &r, const uint4 (&raw)[U], uint32_t at,
                                              bool group, uint64_t single, int lane, uint32_t left = 32 * U) {
    const uint64_t mine = group ? r.best_key(raw, Row<T>::best(raw), at) : single;
    st.list = 0;
    st.insert(mine, kAll, lane);  // the best of each group first
    // then what else reaches the k-th, an element a lane at a time, read again by
    // its index (the loop's body once per element in the code took longer than
    // the rows' memory: instruction cache)
    uint32_t todo = 0;
#pragma unroll
    for (int j = 0; j < Row<T>::N; j += 2) {
        if (32 * (j / Row<T>::VN) >= left) break;
        const float2 p = Row<T>::pair(raw[j / Row<T>::VN], j % Row<T>::VN / 2);
        todo |= (!(p.x < st.thr) ? 1u : 0u) << j | (!(p.y < st.thr) ? 1u : 0u) << (j + 1);
    }
    if (!group) todo = 0;
    while (__any_sync(kAll, todo != 0)) {
        const int j = todo ? __ffs(todo) - 1 : 0;
        const uint32_t idx = r.index(at, j);
        bool want = todo && at + 32 * (j / Row<T>::VN) < r.nvec;
        todo &= todo - 1;
        const uint64_t key = want ? make_key(to_f32(r.x[idx]), idx) : 0;
        want = want && key > st.kth && key != mine;
        const unsigned lanes = __ballot_sync(kAll, want);
        if (lanes) st.insert(key, lanes, lane);
    }
}
template <typename T, bool LONG>
__device__ __forceinline__ void list_elements(Warp<true, LONG> &st, const Row<T> &r, int lane) {
    // an element outside the vectors is a group of its own
    const uint32_t i = ~(uint32_t)st.list - r.head, vec = i / Row<T>::VN;
    const bool in = lane < st.k && st.list, group = in && ~(uint32_t)st.list >= r.head && vec < r.nvec;
    const uint32_t at = vec / (32 * U) * (32 * U) + vec % 32;
    uint4 raw[U];
    r.load(raw, group ? at : r.nvec);
    list_elements(st, r, raw, at, group, in ? st.list : 0, lane);
}

// The row's answer from its sums and list of elements: one warp, every lane with
// the same `a`.
template <typename T, bool TOP, bool LONG>
__device__ __forceinline__ void finish(const Args &g, const Row<T> &r, int64_t row, const Softmax &a,
                                       const Warp<TOP, LONG> &st, int lane) {
    const bool none = a.s == 0.0f;  // every logit -inf: no token has any probability
    const float log_s = logf(a.s);
    if (lane == 0) {
        if (g.targets) {
            const int64_t t = g.targets[row];
            const bool valid = t < (int64_t)g.vocab;
            if (!valid) atomicExch(g.flags + lonnx::FLAG_TARGET, 1);
            if (g.logprob) {
                float lp = __uint_as_float(0x7fc00000u);
                if (valid) lp = none ? -INFINITY : fmaf(to_f32(r.x[t]) - a.m, g.inv_t, -log_s);
                g.logprob[row] = lp;
            }
        }
        if (g.entropy) g.entropy[row] = none ? 0.0f : fmaf(a.w / a.s, -0.69314718055994530942f, log_s);
    }
    if constexpr (TOP) {
        if (lane < g.k) {
            g.top_id[row * g.k + lane] = (int64_t)(uint32_t)~(uint32_t)st.list;
            g.top_logprob[row * g.k + lane] =
                none ? -INFINITY : fmaf(unordered((uint32_t)(st.list >> 32)) - a.m, g.inv_t, -log_s);
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

// the elements outside the vectors, one a lane
template <typename T, bool TOP, bool LONG>
__device__ __forceinline__ void edges(Warp<TOP, LONG> &st, const Row<T> &r, int lane) {
    if (r.head + r.tail == 0) return;
    const bool in = lane < r.head || (lane >= 16 && lane - 16 < r.tail);
    const uint32_t idx = lane < 16 ? lane : r.head + r.nvec * Row<T>::VN + lane - 16;
    const float x = in ? to_f32(r.x[idx]) : -INFINITY;
    // the head's indices are below the list's: equal values enter, too
    if (TOP && in && x == st.thr) st.thr = __uint_as_float(0x7fc00000u);
    st.offer(x, in, -INFINITY, lane, idx, [&] { return make_key(x, idx); });
    st.add(x, -INFINITY);
}

// Warp `w` of `nw` over one row: chunk i to warp i % nw, the elements outside
// the vectors to the last warp.
//
// `reached` (null: none): for each of the CTA's NW warps the value of its best
// ceil(k / NW)-th group so far.  Their least is reached by k groups of the row,
// so groups below it cannot be in the answer: the warps' lists together then
// take in about as many groups as one list over the whole CTA would.
template <int NW, typename T, bool TOP, bool LONG>
__device__ __forceinline__ void scan(Warp<TOP, LONG> &st, const Row<T> &r, int w, int nw, int lane, uint32_t *reached) {
    const uint32_t step = nw * 32 * U;
    constexpr uint32_t FOLD = 64 / (U * Row<T>::VN / 2);  // chunks: 64 terms in each half
    uint32_t v0 = w * 32 * U;
    uint4 next[U];
    if (v0 < r.nvec) r.load(next, v0 + lane);
    while (v0 < r.nvec) {
        const uint32_t at = v0 + lane, left = r.nvec - v0;
        uint4 raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u) raw[u] = next[u];
        v0 += step;
        if (v0 < r.nvec) r.load(next, v0 + lane);
        float floor = -INFINITY;
        if (TOP && reached) {
            const uint32_t o = __reduce_min_sync(kAll, *(volatile uint32_t *)(reached + lane % NW));
            if (o) floor = unordered(o);
        }
        const float best = Row<T>::best(raw);
        const bool changed = st.offer(best, at < r.nvec, floor, lane, r.index(at, 0), [&] { return r.best_key(raw, best, at); });
        if (TOP && reached && changed && lane == (st.k + NW - 1) / NW - 1) *(volatile uint32_t *)(reached + w % NW) = (uint32_t)(st.list >> 32);
        st.sum(r, raw, left);
        if (LONG && !(v0 & step * (FOLD - 1))) st.fold();  // (step is a power of two)
    }
    if (w == nw - 1) edges(st, r, lane);
}

// A warp per row (LONG: of more than kShortRow bytes)
constexpr int kShortRow = 8192;
template <typename T, bool TOP, bool LONG>
__global__ void __launch_bounds__(256, 4) k_logprobs_warp(const T *__restrict__ x, Args g) {
    const int lane = threadIdx.x & 31;
    for (int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); row < g.rows; row += (int64_t)gridDim.x * 8) {
        if (padding(g, row)) {
            finish_padding<TOP>(g, row, lane);
            continue;
        }
        const Row<T> r(x + row * g.ld, g.vocab);
        const float c = g.inv_t * 1.44269504088896340736f;
        Warp<TOP, LONG> st;
        st.reset(c, g.k);
        if (TOP && r.nvec <= 32 * U) {
            // one chunk: its groups are here, so the list is of elements at once
            if constexpr (TOP) {
                uint4 raw[U];
                r.load(raw, lane);
                const float best = Row<T>::best(raw);
                if (__any_sync(kAll, best > st.m)) st.raise(best);
                list_elements(st, r, raw, lane, lane < r.nvec, 0, lane, r.nvec);
                st.sum(r, raw, r.nvec);
                edges(st, r, lane);
            }
        } else {
            scan<1>(st, r, 0, 1, lane, nullptr);
            if constexpr (TOP) list_elements(st, r, lane);
        }
        finish(g, r, row, st.total(), st, lane);
    }
}

// The CTA's warps' sums and lists, joined in halves into warp 0's: in round h
// warps under h take those of warps h above.
template <int NW>
struct Joint {
    Softmax sums[NW];
    uint64_t lists[NW][32];
};
template <int NW, bool TOP>
__device__ __forceinline__ void join_warps(Joint<NW> &j, Softmax &a, uint64_t &list, int n, int w, int lane, float c) {
    for (int h = n >> 1; h > 0; h >>= 1) {
        if (w >= h && w < 2 * h) {
            if (lane == 0) j.sums[w] = a;
            if constexpr (TOP) j.lists[w][lane] = list;
        }
        __syncthreads();
        if (w < h) {
            join(a, j.sums[w + h], c);
            if constexpr (TOP) list = merge_desc(list, j.lists[w + h][lane], lane);
        }
    }
}

// A cluster of CTAs per row (1, 2, 4, 8 or 16): the warps' sums and lists meet in
// the CTA's shared memory, the CTAs' in the first CTA's warps, which read the
// others' over distributed shared memory.  No workspace.
template <int NW, typename T, bool TOP>
__global__ void __launch_bounds__(32 * NW, (TOP ? 32 : 24) / NW) k_logprobs_cta(const T *__restrict__ x, Args g) {
    __shared__ Joint<NW> joint;
    __shared__ Softmax cta_sums;
    __shared__ uint64_t cta_list[32];
    __shared__ uint32_t reached[NW];
    auto cluster = cg::this_cluster();
    const int parts = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const float c = g.inv_t * 1.44269504088896340736f;
    for (int64_t row = blockIdx.x / parts; row < g.rows; row += gridDim.x / parts) {
        if (padding(g, row)) {
            if (part == 0 && w == 0) finish_padding<TOP>(g, row, lane);
            continue;
        }
        const Row<T> r(x + row * g.ld, g.vocab);
        if (TOP) {
            if (threadIdx.x < NW) reached[threadIdx.x] = 0;
            __syncthreads();
        }
        Warp<TOP, true> st;
        st.reset(c, g.k);
        scan<NW>(st, r, part * NW + w, parts * NW, lane, reached);
        Softmax a = st.total();
        join_warps<NW, TOP>(joint, a, st.list, NW, w, lane, c);
        if (parts > 1) {
            if (w == 0) {
                if (lane == 0) cta_sums = a;
                if constexpr (TOP) cta_list[lane] = st.list;
            }
            cluster.sync();
            if (part == 0) {
                // warp w: CTAs w, w + NW, ..
                if (w > 0 && w < parts) {
                    a = *cluster.map_shared_rank(&cta_sums, w);
                    if constexpr (TOP) st.list = cluster.map_shared_rank(cta_list, w)[lane];
                }
                for (int i = w + NW; i < parts; i += NW) {
                    join(a, *cluster.map_shared_rank(&cta_sums, i), c);
                    if constexpr (TOP) st.list = merge_desc(st.list, cluster.map_shared_rank(cta_list, i)[lane], lane);
                }
            }
            cluster.barrier_arrive();  // the others' shared memory is read until here
            if (part == 0) join_warps<NW, TOP>(joint, a, st.list, min(parts, NW), w, lane, c);
        }
        if (part == 0 && w == 0) {
            if constexpr (TOP) list_elements(st, r, lane);
            finish(g, r, row, a, st, lane);
        }
        if (parts > 1) cluster.barrier_wait();
        __syncthreads();  // the next row's sums go into the same shared memory
    }
}

template <int NW, typename T, bool TOP>
int launch_cta(lonnx_ctx *ctx, const T *x, const Args &g, int parts) {
    auto kernel = k_logprobs_cta<NW, T, TOP>;
    const unsigned grid = (unsigned)(std::min<int64_t>(g.rows, (1 << 30) / parts) * parts);
    if (parts == 1) {
        kernel<<<grid, 32 * NW, 0, ctx->stream>>>(x, g);
        LONNX_CHECK_LAUNCH(ctx);
        return LONNX_OK;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(32 * NW);
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)parts;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    static bool attr_set[64] = {false};
    if (!attr_set[ctx->device & 63]) {
        LONNX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        attr_set[ctx->device & 63] = true;
    }
    ctx->launches++;
    LONNX_CUDA(cudaLaunchKernelEx(&cfg, kernel, x, g));
    return LONNX_OK;
}

template <typename T, bool TOP>
int launch(lonnx_ctx *ctx, const void *xv, const Args &g) {
    const T *x = static_cast<const T *>(xv);
    const int64_t row_bytes = (int64_t)g.vocab * (int)sizeof(T);
    // A warp to a row for short rows, or for enough of them to fill the SMs with
    // warps (5000 x 20000 bfloat16, 5 alternatives: 67 us; when it was 73, 4 warps
    // to a row took 95 and 8 warps 127); 4 warps, as joining their lists leaves
    // fewer idle, while SMs get 4 rows each (1000 x 10000: 19 us, 8 warps 25; 300 x
    // 50000: 24 us, 8 warps 23).
    if (row_bytes <= kShortRow || g.rows >= 24 * ctx->num_sms) {
        const unsigned grid = (unsigned)std::min<int64_t>((g.rows + 7) / 8, 1 << 30);
        // (a short row: at most 4 chunks, 64 terms, and one element outside the vectors)
        const auto kernel = row_bytes <= kShortRow ? k_logprobs_warp<T, TOP, false> : k_logprobs_warp<T, TOP, true>;
        kernel<<<grid, 256, 0, ctx->stream>>>(x, g);
        LONNX_CHECK_LAUNCH(ctx);
        return LONNX_OK;
    }
    if (TOP && g.rows >= 4 * ctx->num_sms) return launch_cta<4, T, TOP>(ctx, x, g, 1);
    // Few rows: as many CTAs to a row as fill the SMs twice, while each still has 16 KB to read.
    int parts = 1;
    while (parts < 16 && g.rows * parts < 2 * ctx->num_sms && row_bytes / (parts * 2) >= 16384) parts *= 2;
    return launch_cta<8, T, TOP>(ctx, x, g, parts);
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
