// paged.cuh — what the paged-cache kernels share: element types, the device view of the
// cache and of the batch, and the checks of what they read from device memory.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"
#include "kernels.h"

namespace tqb200 {

// ---------------------------------------------------------------- element types
template <typename T>
__device__ __forceinline__ float el_to_f(T v);
template <>
__device__ __forceinline__ float el_to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float el_to_f<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float el_to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T el_from_f(float v);
template <>
__device__ __forceinline__ float el_from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half el_from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 el_from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N consecutive elements as one load or store of N * sizeof(T) <= 16 bytes (N = 8 fp32: two).
template <typename T, int N>
struct ElVec {
    static_assert(N * sizeof(T) <= 16 || N * sizeof(T) == 32, "vector size");
    static constexpr int W = N * sizeof(T) / 4;
    uint32_t w[W];
    __device__ __forceinline__ void load(const T *p) {
        if constexpr (W >= 4) {
#pragma unroll
            for (int i = 0; i < W; i += 4) {
                const uint4 v = *reinterpret_cast<const uint4 *>(reinterpret_cast<const uint32_t *>(p) + i);
                w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
            }
        } else if constexpr (W == 2) {
            const uint2 v = *reinterpret_cast<const uint2 *>(p);
            w[0] = v.x, w[1] = v.y;
        } else {
            w[0] = *reinterpret_cast<const uint32_t *>(p);
        }
    }
    __device__ __forceinline__ void store(T *p) const {
        if constexpr (W >= 4) {
#pragma unroll
            for (int i = 0; i < W; i += 4)
                *reinterpret_cast<uint4 *>(reinterpret_cast<uint32_t *>(p) + i) =
                    make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
        } else if constexpr (W == 2) {
            *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
        } else {
            *reinterpret_cast<uint32_t *>(p) = w[0];
        }
    }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
        else {
            const uint16_t b = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
            T t;
            memcpy(&t, &b, 2);
            return el_to_f<T>(t);
        }
    }
    __device__ __forceinline__ void set(const float *v) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < N; ++i) w[i] = __float_as_uint(v[i]);
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const T a = el_from_f<T>(v[2 * i]), b = el_from_f<T>(v[2 * i + 1]);
                uint16_t ua, ub;
                memcpy(&ua, &a, 2);
                memcpy(&ub, &b, 2);
                w[i] = (uint32_t)ua | ((uint32_t)ub << 16);
            }
        }
    }
};

// ---------------------------------------------------------------- device views
// x / d and x % d for 0 <= x < 2^31 by one multiplication: with s = ceil(log2 d) and
// m = ceil(2^(31+s) / d) (< 2^32), e = m d - 2^(31+s) < d <= 2^s, so x m / 2^(31+s) is
// above x / d by x e / (d 2^(31+s)) < 1 / d and its floor is that of x / d.
struct FastDiv {
    uint32_t d, m, s;
    __host__ static FastDiv of(uint32_t d) {
        uint32_t s = 0;
        while ((1ull << s) < d) ++s;
        return {d, (uint32_t)(((1ull << (31 + s)) + d - 1) / d), s};
    }
    __device__ __forceinline__ uint32_t div(uint32_t x) const {
        return (uint32_t)(((unsigned long long)x * m) >> (31 + s));
    }
};

struct PagedView {
    char *k, *v;
    long long page_stride, head_stride, slot_stride;  // elements
    int n_pages;
    FastDiv page;  // slots per page
    // Element offset of KV head h of position x, -1 for a page outside the cache.
    __device__ __forceinline__ long long offset(const int *row, int x, int h, int *page_bad) const {
        const uint32_t j = page.div((uint32_t)x);
        const int p = row[j];
        if ((unsigned)p >= (unsigned)n_pages) {
            *page_bad = 1;
            return -1;
        }
        return p * page_stride + h * head_stride + (long long)(x - (int)(j * page.d)) * slot_stride;
    }
};

struct BatchView {
    const int *q_start, *kv_len, *table;
    int n_seqs, table_stride, n_tokens, max_q_len;
    int max_len;  // table_stride * page_size (at most 2^31 - 1): the most positions
};

// A sequence's numbers, checked; ok == 0: to be skipped.
struct SeqInfo {
    int q0, n, len, ok;
};
__device__ __forceinline__ SeqInfo seq_check(const BatchView &b, int q0, int q1, int len) {
    SeqInfo r;
    r.q0 = q0;
    r.n = q1 - q0;
    r.len = len;
    r.ok = q0 >= 0 && q1 >= q0 && q1 <= b.n_tokens && q1 - q0 <= b.max_q_len && len >= 0 && len <= b.max_len;
    return r;
}
__device__ __forceinline__ SeqInfo seq_info(const BatchView &b, int s) {
    return seq_check(b, b.q_start[s], b.q_start[s + 1], b.kv_len[s]);
}

// The sequence that holds row t: the last s with q_start[s] <= t (32 candidates at a time by
// the whole warp; every index stays in [0, n_seqs) whatever the array holds).  The caller
// checks that the row lies inside it.
__device__ __forceinline__ int seq_of_row(const BatchView &b, int t) {
    const int lane = threadIdx.x & 31;
    int lo = 0, n = b.n_seqs;  // candidates lo .. lo + n - 1; lo itself always stands
    while (n > 1) {
        const int step = (n + 31) / 32;
        const int i = lo + lane * step;
        const bool le = lane == 0 || (lane * step < n && b.q_start[i] <= t);
        const unsigned m = __ballot_sync(0xffffffffu, le);
        const int last = 31 - __clz((int)m);
        n = min(step, n - last * step);
        lo += last * step;
    }
    return lo;
}

__device__ __forceinline__ void report(int *status, int code) {
    if (status) atomicExch(status, code);
}

// ---------------------------------------------------------------- launch arguments
struct RopeArgs {
    const void *q, *k, *v;
    void *q_out, *k_out;
    int type;              // TQB200_EL_* of q, k, v, q_out, k_out
    int n_tokens, n_heads, n_kv_heads, head_dim, rotary_dim;
    long long q_stride, k_stride, v_stride, q_out_stride, k_out_stride;
    const float *q_norm, *k_norm;
    float eps, theta;
    const int *positions;
};

struct PagedAttnArgs {
    const void *q;
    void *out;
    int type, n_heads, n_kv_heads, head_dim, cache_type;
    long long q_stride, out_stride;
    float scale;
    PagedView kv;
    BatchView b;
    bool aligned;          // every row of q, out, k and v starts on 16 bytes
    void *work;
    int *status;
};

// ---------------------------------------------------------------- attention, shared
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// One warp's pass over positions [x0, x1) for one row (its p >= x1 - 1): the running maximum
// of the scaled scores (base 2), the sum and, in lane l, elements l, l + 32, ... of the
// weighted values.  Every element type, head_dim up to 256 and alignment; positions on pages
// outside the cache are passed over.
template <typename T, typename C>
__device__ __noinline__ void row_pass(const PagedAttnArgs &A, const T *q, int seq, int kv_head, int x0, int x1,
                         float &m, float &l, float (&o)[8]) {
    const int lane = threadIdx.x & 31, D = A.head_dim;
    float qv[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        qv[j] = lane + 32 * j < D ? el_to_f<T>(q[lane + 32 * j]) : 0.0f;
        o[j] = 0.0f;
    }
    m = -INFINITY;
    l = 0.0f;
    const float c = A.scale * kLog2e;
    const int *row = A.b.table + (long long)seq * A.b.table_stride;
    int bad = 0;
    for (int x = x0; x < x1; ++x) {
        const long long at = A.kv.offset(row, x, kv_head, &bad);
        if (at < 0) continue;  // warp-uniform
        const C *k = (const C *)A.kv.k + at, *v = (const C *)A.kv.v + at;
        float s = 0.0f, vv[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const bool in = lane + 32 * j < D;
            s = fmaf(qv[j], in ? el_to_f<C>(k[lane + 32 * j]) : 0.0f, s);
            vv[j] = in ? el_to_f<C>(v[lane + 32 * j]) : 0.0f;
        }
        s = warp_sum(s) * c;
        const float mn = fmaxf(m, s);
        const float base = mn == -INFINITY ? 0.0f : mn;
        const float f = exp2f(m - base), p = exp2f(s - base);
        m = mn;
        l = fmaf(l, f, p);
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = fmaf(o[j], f, p * vv[j]);
    }
    if (bad && lane == 0) report(A.status, TQB200_PAGED_BAD_PAGE);
}

// ---------------------------------------------------------------- split attention
// The work of a call is one line of tiles: for every sequence with rows, for every KV head,
// (for every block of query rows,) the tiles of positions it reads.  CTA c takes tiles
// [c quota, (c+1) quota), so every CTA reads equally many whatever the lengths are; the parts
// of a (sequence, head, rows) item that lies in several CTAs are joined by the last of them
// to arrive, in the order of the line (the result does not depend on who is last).  The item's
// first CTA names its ticket; a CTA leaves at most two parts: that of the item it begins in
// the middle of (slot 2c) and that of the item it ends in the middle of (slot 2c + 1).
constexpr int kSplitMaxCtas = 1024;
constexpr size_t kSplitTicketBytes = kSplitMaxCtas * 4;  // head of the workspace, zero between calls

int launch_qk_norm_rope(const RopeArgs &a, cudaStream_t st);
int launch_paged_append(const RopeArgs &a, const PagedView &kv, int cache_type, const BatchView &b,
                        int *status, cudaStream_t st);
int launch_paged_attention(const PagedAttnArgs &a, cudaStream_t st);
// At most 16 query rows per KV head, head_dim 64 or 128, 16-byte aligned rows.
int launch_paged_decode(const PagedAttnArgs &a, int rows, cudaStream_t st);
size_t paged_decode_work_bytes(int rows, int head_dim);
constexpr int kDecodeRows = 16;
size_t paged_attention_work_bytes(int n_seqs, int n_tokens, int max_q_len, int n_heads,
                                  int n_kv_heads, int head_dim);

}  // namespace tqb200
