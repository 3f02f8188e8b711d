// paged.cuh — what the paged-cache kernels share: element types, the device view of the
// cache and of the batch, and the checks of what they read from device memory.
#pragma once

#include <cuda_bf16.h>

#include <type_traits>

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

// two fp32 in one register pair: one instruction for both
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    return v;
}
__device__ __forceinline__ void unpair(uint64_t v, float &a, float &b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
    return v;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t v;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t v;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}

// N consecutive elements as one load or store of N * sizeof(T) <= 16 bytes (N = 8 fp32: two).
template <typename T, int N>
struct ElVec {
    static_assert(N * sizeof(T) == 8 || N * sizeof(T) == 16 || N * sizeof(T) == 32, "vector size");
    static constexpr int W = N * sizeof(T) / 4;
    uint32_t w[W];
    __device__ __forceinline__ void load(const T *p) {
        if constexpr (W >= 4) {
#pragma unroll
            for (int i = 0; i < W; i += 4) {
                const uint4 v = *reinterpret_cast<const uint4 *>(reinterpret_cast<const uint32_t *>(p) + i);
                w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
            }
        } else {
            const uint2 v = *reinterpret_cast<const uint2 *>(p);
            w[0] = v.x, w[1] = v.y;
        }
    }
    __device__ __forceinline__ void store(T *p) const {
        if constexpr (W >= 4) {
#pragma unroll
            for (int i = 0; i < W; i += 4)
                *reinterpret_cast<uint4 *>(reinterpret_cast<uint32_t *>(p) + i) =
                    make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
        } else {
            *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
        }
    }
    // elements 2 i and 2 i + 1
    __device__ __forceinline__ uint64_t get2(int i) const {
        if constexpr (sizeof(T) == 4) return pair(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
        else if constexpr (sizeof(T) == 2) {
            if constexpr (std::is_same<T, __half>::value) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
                return pair(f.x, f.y);
            } else {
                return pair(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
            }
        }
    }
    __device__ __forceinline__ void set2(int i, uint64_t v) {
        float a, b;
        unpair(v, a, b);
        if constexpr (sizeof(T) == 4) w[2 * i] = __float_as_uint(a), w[2 * i + 1] = __float_as_uint(b);
        else if constexpr (std::is_same<T, __half>::value) {
            const __half2 h = __floats2half2_rn(a, b);
            w[i] = *reinterpret_cast<const uint32_t *>(&h);
        } else {
            const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
            w[i] = *reinterpret_cast<const uint32_t *>(&h);
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
    int max_len;  // table_stride * page_size (at most 0x7fff0000: a tile past it stays an int): the most positions
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

__device__ __forceinline__ void report(int *status, int code) {
    if (status) atomicExch(status, code);
}

// Reports sequences whose numbers do not fit; a whole CTA, which has nothing else to do.
static __device__ __noinline__ void check_seqs(const BatchView &b, int *status) {
    bool bad = false;
#pragma unroll 4
    for (int s = threadIdx.x; s < b.n_seqs; s += blockDim.x) bad |= !seq_info(b, s).ok;
    if (bad) report(status, TQB200_PAGED_BAD_SEQ);
}

// The first sequence that fits and holds row t, -1: none; by the whole warp, 128 at a time.
static __device__ __noinline__ int scan_for_row(const BatchView &b, int t) {
    const int lane = threadIdx.x & 31;
    for (int s0 = 0; s0 < b.n_seqs; s0 += 128) {
        unsigned in = 0;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = s0 + 32 * u + lane;
            if (i < b.n_seqs && b.q_start[i] <= t && b.q_start[i + 1] > t) in |= 1u << u;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = s0 + 32 * u;
            const unsigned m = __ballot_sync(0xffffffffu, ((in >> u) & 1u) && seq_info(b, i + lane).ok);
            if (m) return i + __ffs((int)m) - 1;
        }
    }
    return -1;
}

// The sequence that holds row t, by the whole warp; ok == 0: none (a row behind the last, or of a
// sequence to be skipped).
__device__ __forceinline__ SeqInfo seq_of_row(const BatchView &b, int t, int &s) {
    const int lane = threadIdx.x & 31;
    // the last s with q_start[s] <= t, 32 candidates at a time (every index stays in [0, n_seqs)
    // whatever the array holds)
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
    s = lo;
    SeqInfo q = seq_info(b, s);
    if (q.ok && t >= q.q0 && t - q.q0 < q.n) return q;
    const bool behind = q.ok && t >= q.q0 && s == b.n_seqs - 1;
    q.ok = 0;
    if (!behind) {
        // An entry that decreases led the search astray: the rows of the sequences that fit must not be
        // lost with the one that does not, so all of them are looked at.
        s = scan_for_row(b, t);
        if (s >= 0) q = seq_info(b, s);
    }
    return q;
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
// weighted values (E of them: head_dim at most 32 E).  Every element type and alignment;
// positions on pages outside the cache are passed over.  The next position's loads go out
// before the present one is used (0.42 us a position for head_dim 96, 0.52 without).
template <typename T, typename C, int E>
__device__ __forceinline__ void row_pass(const PagedAttnArgs &A, const T *q, int seq, int kv_head, int x0, int x1,
                                         float &m, float &l, float (&o)[E]) {
    const int lane = threadIdx.x & 31, D = A.head_dim;
    const PagedView kv = A.kv;
    float qv[E];
    int e[E];  // lanes past the end read its last element, so that no load hangs on a condition
#pragma unroll
    for (int j = 0; j < E; ++j) {
        e[j] = min(lane + 32 * j, D - 1);
        qv[j] = lane + 32 * j < D ? el_to_f<T>(q[e[j]]) : 0.0f;
        o[j] = 0.0f;
    }
    m = -INFINITY;
    l = 0.0f;
    const float c = A.scale * kLog2e;
    const int *row = A.b.table + (long long)seq * A.b.table_stride;
    int bad = 0;
    C kr[E], vr[E], kn[E], vn[E];
    // position x's key and value, or (none, a bad page) the cache's first; its place, -1: none
    auto load = [&](int x, C (&k)[E], C (&v)[E]) {
        const long long at = x < x1 ? kv.offset(row, x, kv_head, &bad) : -1;
        const C *kp = (const C *)kv.k + max(at, 0LL), *vp = (const C *)kv.v + max(at, 0LL);
#pragma unroll
        for (int j = 0; j < E; ++j) k[j] = kp[e[j]], v[j] = vp[e[j]];
        return at;
    };
    long long at = load(x0, kr, vr);
#pragma unroll 2  // the copies from next to present go
    for (int x = x0; x < x1; ++x) {
        const long long next = load(x + 1, kn, vn);
        if (at >= 0) {  // warp-uniform
            float s = 0.0f;
#pragma unroll
            for (int j = 0; j < E; ++j) s = fmaf(qv[j], lane + 32 * j < D ? el_to_f<C>(kr[j]) : 0.0f, s);
            s = warp_sum(s) * c;
            const float mn = fmaxf(m, s);
            const float base = mn == -INFINITY ? 0.0f : mn;
            const float f = exp2f(m - base), p = exp2f(s - base);
            m = mn;
            l = fmaf(l, f, p);
#pragma unroll
            for (int j = 0; j < E; ++j) o[j] = fmaf(o[j], f, p * el_to_f<C>(vr[j]));
        }
        at = next;
#pragma unroll
        for (int j = 0; j < E; ++j) kr[j] = kn[j], vr[j] = vn[j];
    }
    if (bad && lane == 0) report(A.status, TQB200_PAGED_BAD_PAGE);
}

// ---------------------------------------------------------------- split attention
// The work of a call is one line of tiles.  An item is a block of `tq` tokens of one sequence
// with the query heads of one KV head (or some of them: `heads` such sets per sequence); it
// reads KT positions per tile, up to its last token's own.  The line has the sequences in
// order, in each the head sets, in each the token blocks.  CTA c takes tiles
// [c quota, (c+1) quota), so every CTA reads equally many whatever the lengths are; an item
// that lies in several CTAs is joined by the last of them to arrive, in the order of the line
// (the result does not depend on who is last).  Such an item's first CTA names its ticket; a
// CTA leaves at most two parts: of the item that it begins in the middle of (slot 2c) and of
// the one that it ends in the middle of (slot 2c + 1).
// Beginning an item (its queries, the first tile's latency, its results) costs as much as `over`
// tiles, so the line counts as many units more at the front of each item.
// Joining an item's parts takes its last CTA `part` tiles for each, so an item of t tiles is not
// cut into shares below sqrt(t part) (the least of share + parts * part).
// Where joining at all (worth `join` tiles) would cost more than even shares save, the items
// are taken whole instead, the sequence's last blocks (its longest) first: CTA c of g takes
// items c, 2g - 1 - c, 2g + c, ...
constexpr int kSplitMaxCtas = 1024;
constexpr size_t kSplitTicketBytes = kSplitMaxCtas * 4;  // head of the workspace, zero between calls

struct LineShape {
    int tq, heads;
    int min_quota, over, join;
    float part;  // joining one part, in tiles
};

// Sum of floor((a i + b) / M) over 0 <= i < n, M a power of two, a > 0: a i + b less its residue,
// over M.  The residues repeat every M / g terms, g = gcd(a, M), and are b mod g + 0, g, 2 g, ...
// in some order; the terms behind the last whole round are added up.
template <int M>
__device__ inline long long floor_line_sum(uint32_t n, uint32_t a, uint32_t b) {
    static_assert((M & (M - 1)) == 0, "power of two");
    const uint32_t g = min((uint32_t)M, a & (0u - a)), shift = __ffs(g) - 1, per = (uint32_t)M >> shift;
    const uint32_t rest = n & (per - 1), round = per * (b & (g - 1)) + g * (per * (per - 1) / 2);
    uint32_t tail = 0;
#pragma unroll 4
    for (uint32_t i = 0; i < rest; ++i) tail += (a * i + b) & (M - 1);
    const unsigned long long all = (unsigned long long)n * (n - 1) / 2 * a + (unsigned long long)n * b;
    const unsigned long long residues = (unsigned long long)(n / per) * round + tail;
    return (long long)((all - residues) / M);
}

// a / b, mostly of 32-bit values
__device__ __forceinline__ long long quotient(long long a, long long b) {
    if (((a | b) >> 32) == 0) return (uint32_t)a / (uint32_t)b;
    return a / b;
}

// Adds 1 to a ticket, after everything that the CTA wrote (the barrier before the call puts the
// other threads' stores before this thread's release, which is cumulative) and before everything
// that it reads after the barrier behind the call.
__device__ __forceinline__ unsigned take_ticket(unsigned *p) {
    unsigned n;
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(n) : "l"(p) : "memory");
    return n;
}

template <int KT>
struct Line {
    // tiles of token block b of `nb`: positions up to its last token's, at least one tile
    __device__ static __forceinline__ int block_tiles(const SeqInfo &q, int tq, int nb, int b) {
        const int last = q.len - q.n + (b == nb - 1 ? q.n : (b + 1) * tq) - 1;
        return last < 0 ? 1 : last / KT + 1;
    }
    __device__ static __forceinline__ int blocks(const SeqInfo &q, int tq) { return (q.n + tq - 1) / tq; }
    // tiles of one head set
    __device__ static __forceinline__ long long head_tiles(const SeqInfo &q, int tq) {
        if (!q.ok || q.n == 0) return 0;
        const int nb = blocks(q, tq);
        long long sum = block_tiles(q, tq, nb, nb - 1);
        if (nb > 1) {
            const int p0 = q.len - q.n;
            // the blocks before it: those that end before position 0 have one tile each
            const int none = p0 < 0 ? min(nb - 1, (int)((uint32_t)(-p0) / (uint32_t)tq)) : 0;
            sum += nb - 1 + floor_line_sum<KT>((uint32_t)(nb - 1 - none), (uint32_t)tq,
                                               (uint32_t)((long long)p0 + (long long)none * tq + tq - 1));
        }
        return sum;
    }

    // ---- one warp's way along its CTA's part of the line (every warp walks it for itself)
    LineShape sh;
    SeqInfo q;
    long long quota, at, end, u0;  // units: per CTA; the next, the end of the range; the item's first tile
    int seq, head, b, nb, tiles, ta, tb;
    bool whole;                     // the items are taken whole: at, end, u0 count items, u0 the sequence's first

    __device__ __forceinline__ void enter(const SeqInfo &i, int s) {
        seq = s;
        q = i;
        head = 0;
        b = 0;
        nb = blocks(q, sh.tq);
        tiles = block_tiles(q, sh.tq, nb, 0);
    }
    __device__ __forceinline__ void enter_from(const BatchView &B, int s) {
        SeqInfo i{};
        for (; s < B.n_seqs; ++s) {
            i = seq_info(B, s);
            if (i.ok && i.n > 0) break;
        }
        enter(i, s);
    }
    // whole items: the item number `at`
    __device__ __forceinline__ void seek(const BatchView &B) {
        while (at < end && at >= u0 + (long long)nb * sh.heads && seq < B.n_seqs) {
            u0 += (long long)nb * sh.heads;
            enter_from(B, seq + 1);
        }
        const long long j = at - u0, back = quotient(j, sh.heads);
        b = nb - 1 - (int)back;
        head = (int)(j - back * sh.heads);
        tiles = block_tiles(q, sh.tq, nb, b);
    }
    // The present item's part [ta, tb) for this CTA; false: the range is done.
    __device__ __forceinline__ bool part(const BatchView &B) {
        if (at >= end || seq >= B.n_seqs) return false;
        ta = whole ? 0 : (int)max(0LL, at - u0);
        tb = whole ? tiles : (int)min((long long)tiles, end - u0);
        return tb > ta;  // a range may end in the units before an item's first tile
    }
    __device__ __forceinline__ void next(const BatchView &B) {
        if (whole) {
            // c, 2g - 1 - c, 2g + c, ...: the steps alternate, together 2g
            const long long g = gridDim.x, r = at - quotient(at, 2 * g) * 2 * g;
            at += r < g ? 2 * (g - r) - 1 : 2 * (2 * g - r) - 1;
            if (at < end) seek(B);
            return;
        }
        at = u0 + tiles;
        u0 = at + sh.over;
        if (at >= end) return;
        if (++b == nb) {
            b = 0;
            if (++head == sh.heads) {
                enter_from(B, seq + 1);
                return;
            }
        }
        tiles = block_tiles(q, sh.tq, nb, b);
    }
    // The CTAs that share the item: the first and the last.
    __device__ __forceinline__ int first_cta() const { return (int)quotient(u0, quota); }
    __device__ __forceinline__ int last_cta() const { return (int)quotient(u0 + tiles - 1, quota); }
    __device__ __forceinline__ bool all_mine() const { return ta == 0 && tb == tiles; }
    __device__ __forceinline__ long long slot_of(int cta) const {
        return 2 * (long long)cta + ((long long)cta * quota >= u0 ? 0 : 1);
    }

    // The range of CTA blockIdx.x from the line's totals; `before`, `mine`: units of the caller's
    // sequences and of those before them.  Leaves them as items where items are taken whole.
    __device__ __forceinline__ void range(long long total, long long items, int most) {
        const long long g = gridDim.x;
        quota = max(quotient(total + g - 1, g), (long long)max(sh.min_quota, (int)sqrtf((float)most * sh.part)));
        most += sh.over;
        whole = (items <= g ? most : quota + most / 2) <= quota + sh.join;
        at = whole ? (long long)blockIdx.x : blockIdx.x * quota;
        end = whole ? items : min(at + quota, total);
    }
    // Into sequence s, whose units (or items) begin at `first` and whose head sets have `hu` units.
    __device__ __forceinline__ void locate(const BatchView &B, const SeqInfo &i, int s, long long first, long long hu) {
        const int lane = threadIdx.x & 31;
        enter(i, s);
        if (whole) {
            u0 = first;
            seek(B);
            return;
        }
        // head set by division, token block by a scan of 32 blocks at a time
        head = (int)quotient(at - first, hu);
        u0 = first + head * hu;
        long long off = at - u0;
        if (nb == 1) {
            u0 += sh.over;
            return;
        }
        for (int b0 = 0; b0 < nb; b0 += 32) {
            const int n = b0 + lane < nb ? block_tiles(q, sh.tq, nb, b0 + lane) + sh.over : 0;
            int sum = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += u;
            }
            const unsigned past = __ballot_sync(0xffffffffu, off < sum);
            if (past) {
                const int l = __ffs((int)past) - 1;
                b = b0 + l;
                tiles = __shfl_sync(0xffffffffu, n, l) - sh.over;
                u0 += __shfl_sync(0xffffffffu, sum, l) - tiles;
                return;
            }
            off -= __shfl_sync(0xffffffffu, sum, 31);
            u0 += __shfl_sync(0xffffffffu, sum, 31);
        }
    }

    // Whole CTA (THREADS of it), once: the line's length, the range, the first item.
    template <int THREADS>
    __device__ void begin(const BatchView &B, const LineShape &shape, int *status) {
        sh = shape;
        const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
        if (B.n_seqs <= 32) {
            // every warp for itself, a lane per sequence: no barrier, one round of loads
            SeqInfo i{};
            if (lane < B.n_seqs) {
                i = seq_info(B, lane);
                if (!i.ok && t < 32 && blockIdx.x == 0) report(status, TQB200_PAGED_BAD_SEQ);
            }
            const bool has = i.ok && i.n > 0;
            const int n = has ? blocks(i, sh.tq) : 0;
            const long long hu = has ? head_tiles(i, sh.tq) + (long long)n * sh.over : 0;
            const long long mine = hu * sh.heads, mine_i = (long long)n * sh.heads;
            long long inc = mine, inc_i = mine_i;
            if (B.n_seqs > 1) {
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const long long u = __shfl_up_sync(0xffffffffu, inc, o), v = __shfl_up_sync(0xffffffffu, inc_i, o);
                    if (lane >= o) inc += u, inc_i += v;
                }
            }
            const int last = B.n_seqs - 1;
            const int most = __reduce_max_sync(0xffffffffu, has ? block_tiles(i, sh.tq, n, n - 1) : 0);
            range(__shfl_sync(0xffffffffu, inc, last), __shfl_sync(0xffffffffu, inc_i, last), most);
            const unsigned past = __ballot_sync(0xffffffffu, lane < B.n_seqs && at < (whole ? inc_i : inc));
            seq = B.n_seqs;
            if (at >= end || past == 0) {
                at = end;  // nothing for this CTA
                return;
            }
            const int s = __ffs((int)past) - 1;
            SeqInfo f;
            f.q0 = __shfl_sync(0xffffffffu, i.q0, s);
            f.n = __shfl_sync(0xffffffffu, i.n, s);
            f.len = __shfl_sync(0xffffffffu, i.len, s);
            f.ok = 1;
            locate(B, f, s, __shfl_sync(0xffffffffu, whole ? inc_i - mine_i : inc - mine, s), __shfl_sync(0xffffffffu, hu, s));
            return;
        }
        constexpr int WARPS = THREADS / 32;
        __shared__ long long s_units[WARPS], s_items[WARPS], s_first, s_hu;
        __shared__ int s_most[WARPS], s_seq;
        const int per = (B.n_seqs + THREADS - 1) / THREADS;
        const int s0 = min(B.n_seqs, t * per), s1 = min(B.n_seqs, s0 + per);
        auto units_of = [&](const SeqInfo &i, long long &hu, long long &items) {
            items = 0;
            hu = 0;
            if (!i.ok || i.n == 0) return;
            const int n = blocks(i, sh.tq);
            items = (long long)n * sh.heads;
            hu = head_tiles(i, sh.tq) + (long long)n * sh.over;
        };
        long long mine = 0, mine_i = 0, hu = 0, n = 0;
        int most = 0;
        for (int s = s0; s < s1; ++s) {
            const SeqInfo i = seq_info(B, s);
            if (!i.ok && blockIdx.x == 0) report(status, TQB200_PAGED_BAD_SEQ);
            units_of(i, hu, n);
            mine += hu * sh.heads;
            mine_i += n;
            if (n) most = max(most, block_tiles(i, sh.tq, blocks(i, sh.tq), blocks(i, sh.tq) - 1));
        }
        long long inc = mine, inc_i = mine_i;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long u = __shfl_up_sync(0xffffffffu, inc, o), v = __shfl_up_sync(0xffffffffu, inc_i, o);
            if (lane >= o) inc += u, inc_i += v;
        }
        most = __reduce_max_sync(0xffffffffu, most);
        if (lane == 31) s_units[warp] = inc, s_items[warp] = inc_i, s_most[warp] = most;
        if (t == 0) s_seq = B.n_seqs;
        __syncthreads();
        long long before = inc - mine, total = 0, before_i = inc_i - mine_i, total_i = 0;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            if (w < warp) before += s_units[w], before_i += s_items[w];
            total += s_units[w];
            total_i += s_items[w];
            most = max(most, s_most[w]);
        }
        range(total, total_i, most);
        if (whole) before = before_i, mine = mine_i;
        if (at < end && at >= before && at < before + mine) {  // one thread
            for (int s = s0; s < s1; ++s) {
                if (s1 - s0 > 1) units_of(seq_info(B, s), hu, n);
                const long long u = whole ? n : hu * sh.heads;
                if (at < before + u) {
                    s_seq = s;
                    s_first = before;
                    s_hu = hu;
                    break;
                }
                before += u;
            }
        }
        __syncthreads();
        seq = s_seq;
        if (at >= end || seq >= B.n_seqs) {
            at = end;  // nothing for this CTA
            return;
        }
        locate(B, seq_info(B, seq), seq, s_first, s_hu);
    }
};

// A driver function by name, looked up at run time; null where there is none.
void *driver_entry(const char *name);
int launch_qk_norm_rope(const RopeArgs &a, cudaStream_t st);
int launch_paged_append(const RopeArgs &a, const PagedView &kv, int cache_type, const BatchView &b,
                        int *status, cudaStream_t st);
int launch_paged_attention(const PagedAttnArgs &a, cudaStream_t st);
// head_dim 64 or 128, 16-byte aligned rows; blocks of up to 16 query rows.
int launch_paged_decode(const PagedAttnArgs &a, cudaStream_t st);
size_t paged_decode_work_bytes(int head_dim);
constexpr int kDecodeRows = 16;
// The same with a 16-bit cache; blocks of 128 or 256 query rows.
int launch_paged_chunk(const PagedAttnArgs &a, cudaStream_t st);
size_t paged_chunk_work_bytes(int head_dim);
size_t paged_attention_work_bytes(int head_dim);

}  // namespace tqb200
