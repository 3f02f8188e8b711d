// paged_chunk.cu — causal attention of many new rows (chunks of prompts, alone or in one batch
// with single tokens) over a paged 16-bit KV cache, on the sm_100a tensor cores (tcgen05.mma,
// accumulators in TMEM).
//
// An item is QT tiles of 128 query rows (token, query head of one KV head) that share every
// tile of KT keys and values:
//   S = Q K^T (128 x KT, fp32 in TMEM);  P = 2^(c S - m) in 16 bits, written over S in TMEM;
//   O += P V (128 x D, fp32 in TMEM), P as the A operand from TMEM.
// Bound: the tensor pipe for long chunks (4 D operations per row, key and value).  Beside it
// runs one exponential per score on 16 lanes per clock, which takes as long as the products
// of 16-bit operands at the pipe's rate (128 x 64 scores of D 128: 512 clocks either way), so two
// query tiles alternate and each has two score buffers: the next tile's scores are formed while
// this one's softmax runs.  As issued the products take 640 clocks: one of N = 64 (Q K^T) comes
// every 48 clocks from its thread, where the pipe needs 32, one of N = 128 (P V) every 64.
// Roles (warps): QT groups of 4 softmax warps (thread = query row = TMEM lane), 2 QT warps that
// fetch keys and values, QT warps that each issue one query tile's products.
//  * A ring of slots holds whole K or V tiles in the order they are used, K0 K1 V0 K2 V1 ...
//    Whole tiles come by TMA from the pages (any order of heads and slots: the tensor map has
//    the cache's strides), the others (a sequence's last, odd page sizes) by 16-byte cp.async
//    with positions that do not exist filled with zeros; a bitmap per tile marks those.
//  * Shared memory holds rows of 128 bytes (64 dimensions of a position or query row) in the
//    128-byte swizzle, as K-major A and B operands for Q K^T and MN-major B operand for P V.
//  * Softmax: the row's maximum is raised only when a score passes it by 2^8 (then the warp
//    rescales its rows of O in TMEM); weights carry a factor 2^6 against fp16's subnormals,
//    so they stay below 2^14.  Of 16-bit activations they go into P V in the cache's type, off by
//    at most half a step, their sum as it was: the chunk below comes out 2.3e-3 off 64 bits, 1.7e-3
//    of it the results' own rounding; a second part for the weights would double P V.
//  * fp32 activations over an fp16 cache: Q (scaled per row by a power of two) and P are
//    split into fp16 hi + lo, two products each: 22 bits of either operand.
//  * fp32 results: the tensor core cuts its sums, so after every 8 tiles O moves to an fp32 sum
//    in the workspace and starts at zero (2000 rows over up to 8000 positions: 450 to 500 us by
//    the clock's state, 430 without; error against 64 bits 2e-6 of the result instead of 6e-6).
//  * Rows that come out not finite are computed again after the CTA's last item (redo_rows).
//  * Every wait is bounded; after one runs out the roles go on without waiting or issuing, the
//    issued copies and products are waited for (bounded), TMEM is freed and the error stored.
//
// Measured on one B200 (device time): 2048 rows of 32 heads over 8 KV heads of 128 and 16384
// bf16 positions (515 GFLOP) 470 to 550 us by the clock's state, 0.94 to 1.09 PFLOP/s; 512 rows
// of 32 heads over 4 KV heads, fp32 over fp16, 19.3 us.  A tile of 64 keys takes about 2400 clocks
// for both query tiles, of which the products as issued need 1280; the softmax warps' own chain
// (TMEM load, maximum, exponential, TMEM store) is what is left.  Whole tiles by 16-byte copies take
// 640 us at the first shape, by TMA 519; by pages of 16 it takes 544 us, by pages of 8 573.  An item's
// beginning and end (12000 of 29000 clocks for the 512 rows) run once, so their code is kept short.
#include <cuda.h>
#include <string.h>

#include <algorithm>
#include <numeric>
#include <type_traits>

#include "paged.cuh"

namespace tqb200 {
namespace {

constexpr float kRaise = 8.0f;
constexpr float kLift = 6.0f;
constexpr int kFold = 8;          // tiles per sum in TMEM where results are fp32
constexpr int kBehind = 3;        // tiles whose copies a fetching warp leaves in flight
constexpr int kRows = 128;        // query rows per tile: TMEM lanes
constexpr int kMaxSlots = 12;
constexpr int kUnread = -2147483647;  // a page number not read yet (bad if it were one)
constexpr int kMarks = 16;        // tiles whose bitmaps are kept (more than the ring holds)
constexpr int KT = 64;            // positions per tile (two words of a bitmap)
constexpr int kMeta = 1024;

struct ChunkParams {
    PagedAttnArgs A;
    unsigned *tickets;
    float *parts;     // [2 grid]: [D / 4][rows][4] accumulators, [rows] maxima, [rows] sums
    float *kept;      // [grid][D / 4][rows][4]: sums of earlier tiles (fp32 results)
    LineShape line;
    int sets, g_set;
    int slots;
    int box_rows;               // slots of a page per tensor copy, 0: no tensor copies
    alignas(64) uint8_t map_k[128], map_v[128];
};

// ---------------------------------------------------------------- tcgen05
// Operand in rows of 128 bytes (64 elements), 16-byte piece p of row r at p ^ (r & 7): swizzle
// mode 2.  Eight rows are 1024 bytes (the stride offset); `lead` is the way from 64 elements to
// the next 64 along the contiguous dimension of an MN-major operand.
__device__ __forceinline__ uint64_t row_desc(uint32_t saddr, uint32_t lead) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           (1ull << 46) | (2ull << 61);
}
// kind::f16, fp32 accumulator, M = 128; bv: the B operand is MN-major
template <typename C>
__device__ __forceinline__ constexpr uint32_t idesc_of(int n, bool bv) {
    const uint32_t f = std::is_same<C, __half>::value ? 0u : 1u;
    return (1u << 4) | (f << 7) | (f << 10) | (bv ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
        "r"((uint32_t)acc)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc),
        "r"((uint32_t)acc)
        : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 columns of this warp's lanes, 32 (fp32 words) or 16 registers a thread
__device__ __forceinline__ void tm_ld32(uint32_t a, float *v) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(a)
        : "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tm_ld16(uint32_t a, float (&v)[16]) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(a)
        : "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tm_st16(uint32_t a, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(a),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

__device__ __forceinline__ void tm_st16(uint32_t a, const float (&v)[16]) {
    uint32_t r[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(v[i]);
    tm_st16(a, r);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float v;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(v) : "f"(a), "f"(b), "f"(c));
    return v;
}

__device__ __forceinline__ bool elect_one() {
    uint32_t e;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(e));
    return e != 0;
}
__device__ __forceinline__ void arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool test_once(uint64_t *bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(done) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return done != 0;
}
__device__ __forceinline__ void copy16(uint32_t dst, const char *src, bool live) {  // not live: zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void box_load(uint32_t dst, const void *map, int x, int y, int z, int w, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
        : "memory");
}
template <int N>
__device__ __forceinline__ void copies_left() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <typename C>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (std::is_same<C, __half>::value) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}
__device__ __forceinline__ void split2(float a, float b, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&l);
}

template <typename T, int D, int QT>
struct ChunkShape {
    static constexpr int QS = std::is_same<T, float>::value ? 2 : 1;
    static constexpr int SOFT = QT * 128;                       // softmax threads
    static constexpr int FETCH = 2 * QT;                        // warps that fetch
    static constexpr int THREADS = SOFT + FETCH * 32 + QT * 32;  // QT 2: 14 warps, 128 registers a thread
    static constexpr int ROWS = QT * kRows;
    static constexpr uint32_t QBYTES = kRows * D * 2;           // one operand of one query tile
    static constexpr uint32_t TBYTES = KT * D * 2;              // one slot: a K or a V tile
    static constexpr uint32_t COLS = QT * (2 * KT + D) <= 256 ? 256 : 512;  // TMEM columns
    static_assert(QT * (2 * KT + D) <= 512, "TMEM");
};

// One row of an item from the parts of its CTAs, in order (thread = row).
template <typename T, int D, int ROWS>
__device__ __forceinline__ void join_row(const ChunkParams &P, const Line<KT> &it, int row, T *dst) {
    const int c0 = it.first_cta(), c1 = it.last_cta();
    auto part_of = [&](int cta) { return P.parts + it.slot_of(cta) * ROWS * (D + 2); };
    // statistics, then 32 values at a time: two parts' loads in flight
    float M = -INFINITY, L = 0.0f;
#pragma unroll 4
    for (int i = c0; i <= c1; ++i) M = fmaxf(M, __ldcg(part_of(i) + ROWS * D + row));
    const float b = M == -INFINITY ? 0.0f : M;
#pragma unroll 4
    for (int i = c0; i <= c1; ++i) {
        const float *pp = part_of(i) + ROWS * D + row;
        L = fmaf(ex2(__ldcg(pp) - b), __ldcg(pp + ROWS), L);
    }
    const float li = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll 1
    for (int d = 0; d < D; d += 32) {
        float o[32];
#pragma unroll
        for (int k = 0; k < 32; ++k) o[k] = 0.0f;
#pragma unroll 1
        for (int i = c0; i <= c1; i += 2) {
            const bool two = i < c1;
            const float *p0 = part_of(i), *p1 = part_of(two ? i + 1 : i);
            const float f0 = ex2(__ldcg(p0 + ROWS * D + row) - b);
            const float f1 = two ? ex2(__ldcg(p1 + ROWS * D + row) - b) : 0.0f;
            float4 x[8], y[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = __ldcg(reinterpret_cast<const float4 *>(p0 + ((d / 4 + k) * ROWS + row) * 4));
#pragma unroll
            for (int k = 0; k < 8; ++k) y[k] = __ldcg(reinterpret_cast<const float4 *>(p1 + ((d / 4 + k) * ROWS + row) * 4));
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                o[4 * k] = fmaf(f0, x[k].x, o[4 * k]), o[4 * k + 1] = fmaf(f0, x[k].y, o[4 * k + 1]);
                o[4 * k + 2] = fmaf(f0, x[k].z, o[4 * k + 2]), o[4 * k + 3] = fmaf(f0, x[k].w, o[4 * k + 3]);
            }
            if (two) {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    o[4 * k] = fmaf(f1, y[k].x, o[4 * k]), o[4 * k + 1] = fmaf(f1, y[k].y, o[4 * k + 1]);
                    o[4 * k + 2] = fmaf(f1, y[k].z, o[4 * k + 2]), o[4 * k + 3] = fmaf(f1, y[k].w, o[4 * k + 3]);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < 32; ++k) o[k] *= li;
#pragma unroll
        for (int k = 0; k < 32; k += 16 / sizeof(T)) {
            ElVec<T, 16 / sizeof(T)> v;
            v.set(o + k);
            v.store(dst + d + k);
        }
    }
}

// Whole CTA, after its last item: rows that came out not finite are computed again, each by a
// warp's pass over what the row sees.  A weight of 0 does not hide an infinity or NaN among values
// that the row does not see, and the split of an operand makes a NaN of its own from an infinity.
// Such passes (256 rows of 32 heads of 128 over 8192: 15 ms) may over a long context outlast
// the limits of the roles' waits; here nothing waits for them.  whole:
// items that are this CTA's alone; later: its parts (bit: slot) whose tickets are still to be taken.
template <typename T, typename C, int D, int QT>
__device__ __noinline__ void redo_rows(const ChunkParams &P, bool whole, int later) {
    using Sh = ChunkShape<T, D, QT>;
    constexpr int ROWS = Sh::ROWS;
    const PagedAttnArgs &A = P.A;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, G = A.n_heads / A.n_kv_heads;
    __shared__ unsigned s_join;
    Line<KT> it{};
    it.template begin<Sh::THREADS>(A.b, P.line, nullptr);
    for (; it.part(A.b); it.next(A.b)) {
        const bool mine = it.all_mine();
        const long long slot = it.slot_of(blockIdx.x);
        if (mine ? !whole : !((later >> (slot & 1)) & 1)) continue;
        const SeqInfo &q = it.q;
        const int head = it.head / P.sets, h0 = (it.head - head * P.sets) * P.g_set;
        const int gs = min(P.g_set, G - h0), tok0 = it.b * P.line.tq;
        const int rows = min(P.line.tq, q.n - tok0) * gs;
        auto at = [&](int row, long long stride) {
            const int t = row / gs;
            return (long long)(q.q0 + tok0 + t) * stride + (long long)(head * G + h0 + row - t * gs) * D;
        };
        float *part = P.parts + slot * ROWS * (D + 2);
        for (int row = warp; row < rows; row += Sh::THREADS / 32) {
            T *out = (T *)A.out + at(row, A.out_stride);
            float naught = 0.0f;
#pragma unroll
            for (int e = lane; e < D; e += 32)
                naught = fmaf(mine ? el_to_f<T>(out[e]) : part[(e / 4 * ROWS + row) * 4 + (e & 3)], 0.0f, naught);
            if (!__any_sync(0xffffffffu, naught != 0.0f)) continue;  // NaN is not 0 either
            float m, l, o[D / 32];
            row_pass<T, C, D / 32>(A, (const T *)A.q + at(row, A.q_stride), it.seq, head, it.ta * KT,
                                   min(it.tb * KT, q.len - q.n + tok0 + row / gs + 1), m, l, o);
            const float f = mine ? (l == 0.0f ? 0.0f : 1.0f / l) : exp2f(kLift);
#pragma unroll
            for (int j = 0; j < D / 32; ++j) {
                const int e = lane + 32 * j;
                if (mine) out[e] = el_from_f<T>(o[j] * f);
                else part[(e / 4 * ROWS + row) * 4 + (e & 3)] = o[j] * f;
            }
            if (!mine && lane == 0) part[ROWS * D + row] = m, part[ROWS * D + ROWS + row] = l * f;
        }
        if (mine) continue;
        __syncthreads();
        const int c0 = it.first_cta();
        if (tid == 0) {
            s_join = take_ticket(&P.tickets[c0]) == (unsigned)(it.last_cta() - c0);
            if (s_join) P.tickets[c0] = 0;
        }
        __syncthreads();
        if (s_join && tid < rows) join_row<T, D, ROWS>(P, it, tid, (T *)A.out + at(tid, A.out_stride));
        __syncthreads();  // s_join is read before it is written again
    }
}

// ---------------------------------------------------------------- the kernel
template <typename T, typename C, int D, int QT>
__global__ void __launch_bounds__(ChunkShape<T, D, QT>::THREADS, 1)
    paged_chunk_kernel(const __grid_constant__ ChunkParams P) {
    using Sh = ChunkShape<T, D, QT>;
    constexpr int QS = Sh::QS, ROWS = Sh::ROWS;
    constexpr uint32_t QHALF = kRows * 128, THALF = KT * 128;  // 64 dimensions of a query tile, of a slot
    extern __shared__ __align__(1024) uint8_t smem[];
    const PagedAttnArgs &A = P.A;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint64_t *full = reinterpret_cast<uint64_t *>(smem);   // [slots] tile landed (every fetch warp)
    uint64_t *empty = full + kMaxSlots;                    // [slots] tile read by every query tile's products
    uint64_t *sfull = empty + kMaxSlots;                   // [QT][2] scores in TMEM
    uint64_t *pready = sfull + 2 * QT;                     // [QT][2] weights in TMEM (4 warps)
    uint64_t *odone = pready + 2 * QT;                     // [QT][2] P V complete
    uint64_t *qready = odone + 2 * QT;                       // [QT] queries in shared memory, O free (4 warps)
    uint64_t *done = qready + QT;                          // [QT] every product of the issuing warp complete
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(done + QT);
    uint8_t *marks = smem + 512;                           // [kMarks][KT / 8]: positions that exist
    static_assert(kMarks * KT / 8 <= kMeta - 512 && 8 * (2 * kMaxSlots + 8 * QT) + 4 <= 512, "meta");
    uint8_t *sq = smem + kMeta;
    uint8_t *ring = sq + QT * QS * Sh::QBYTES;
    __shared__ int s_err, s_odd, s_again, s_later;  // a part, a whole row is not finite; parts left to redo_rows
    __shared__ unsigned s_last;

    if (tid == 0) {
        for (int i = 0; i < P.slots; ++i) {
            mbar_init(&full[i], Sh::FETCH);
            mbar_init(&empty[i], QT);
        }
        for (int i = 0; i < 2 * QT; ++i) {
            mbar_init(&sfull[i], 1);
            mbar_init(&pready[i], 4);
            mbar_init(&odone[i], 1);
        }
        for (int i = 0; i < QT; ++i) {
            mbar_init(&qready[i], 4);
            mbar_init(&done[i], 1);
        }
        fence_mbar_init();
        s_err = s_odd = s_again = s_later = 0;
    }
    Line<KT> it{};
    it.template begin<Sh::THREADS>(A.b, P.line, A.status);
    if (it.at >= it.end) return;  // uniform: nothing allocated yet
    constexpr int kIssue = Sh::SOFT / 32 + Sh::FETCH;  // first issuing warp
    if (warp == kIssue) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(Sh::COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_slot;
    const int G = A.n_heads / A.n_kv_heads;
    bool bad = false;  // warp-uniform: a wait ran out
    auto wait = [&](uint64_t *bar, uint32_t parity) {
        if (!bad && !__all_sync(0xffffffffu, mbar_wait_sleep(bar, parity, kWaitCycles))) {
            bad = true;
            if (lane == 0) s_err = 1;
        }
    };
    // Tiles of this CTA so far, over all its items.  Tile n uses the second of each pair of
    // barriers when n is odd, in their phase n / 2: the softmax runs up to two tiles ahead of
    // the products, and a parity tells only one phase from the next.
    uint32_t tiles_done = 0;
    uint32_t items_done = 0;

    if (warp < 4 * QT) {
        // ================================================================ softmax
        const int qt = warp >> 2, r = tid & 127;
        auto wait_product = [&](uint32_t n) { wait(&odone[2 * qt + (n & 1u)], (n >> 1) & 1u); };
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t s_of = tmem + lanes + (uint32_t)(qt * 2 * KT), o_at = tmem + lanes + (uint32_t)(QT * 2 * KT + qt * D);
        for (; it.part(A.b); it.next(A.b), ++items_done) {
            const SeqInfo &q = it.q;
            const int head = it.head / P.sets, h0 = (it.head - head * P.sets) * P.g_set;
            const int gs = min(P.g_set, G - h0), tok0 = it.b * P.line.tq;
            const int rows = min(P.line.tq, q.n - tok0) * gs;
            const int p0 = q.len - q.n + tok0;
            const int row = qt * kRows + r;
            const bool live = row < rows;
            // row / gs for row < 256: error of the reciprocal below 256 * 255 / 65536 < 1
            const uint32_t recip = (65535u + (uint32_t)gs) / (uint32_t)gs;
            auto token_of = [&](int x) { return (int)(((uint32_t)x * recip) >> 16); };
            const int tok = token_of(row);
            const long long q_row = (long long)(q.q0 + tok0 + tok);
            const long long h_off = (long long)(head * G + h0 + row - tok * gs) * D;
            const int see = live ? p0 + tok : -1;
            // every row of the warp sees up to here (rows that are not there see all)
            const int see_all = __reduce_min_sync(0xffffffffu, live ? see : 0x7fffffff);
            float c = A.scale * kLog2e;
            // ---- the warp's 32 rows to shared memory: 8 lanes take the 8 pieces of 64 dimensions
            // of one row, 4 rows at a time
            {
                const int g = lane >> 3, p = lane & 7;
                uint8_t *const mine = sq + qt * QS * Sh::QBYTES + (warp & 3) * 32 * 128;
                auto row_of = [&](int i) { return qt * kRows + 32 * (warp & 3) + 4 * i + g; };
                auto source = [&](int x) {
                    const int tx = token_of(x);
                    return (const T *)A.q + (long long)(q.q0 + tok0 + tx) * A.q_stride + (long long)(head * G + h0 + x - tx * gs) * D +
                           p * (16 / (int)sizeof(T));
                };
                auto target = [&](int i, int h, int piece) {
                    const int xw = 4 * i + g;
                    return mine + h * QHALF + xw * 128 + ((piece ^ (xw & 7)) * 16);
                };
                // all the loads of a batch before its first store: one latency
                if constexpr (QS == 1) {
                    uint4 v[8][D / 64];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const T *src = source(row_of(i));
#pragma unroll
                        for (int h = 0; h < D / 64; ++h)
                            v[i][h] = row_of(i) < rows ? *reinterpret_cast<const uint4 *>(src + h * 64) : make_uint4(0, 0, 0, 0);
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i)
#pragma unroll
                        for (int h = 0; h < D / 64; ++h) *reinterpret_cast<uint4 *>(target(i, h, p)) = v[i][h];
                } else {
                    // a lane takes 4 dimensions of every 32: whole lines per load
                    constexpr int B = 4, N = D / 32;
                    float scaled = 1.0f;  // this lane's row
#pragma unroll 1
                    for (int i0 = 0; i0 < 8; i0 += B) {
                        float4 v[B][N];
#pragma unroll
                        for (int j = 0; j < B; ++j) {
                            const T *src = source(row_of(i0 + j));
#pragma unroll
                            for (int k = 0; k < N; ++k)
                                v[j][k] = row_of(i0 + j) < rows ? *reinterpret_cast<const float4 *>(src + k * 32)
                                                                : make_float4(0, 0, 0, 0);
                        }
                        float most[B];
#pragma unroll
                        for (int j = 0; j < B; ++j) {
                            most[j] = 0.0f;
#pragma unroll
                            for (int k = 0; k < N; ++k)
                                most[j] = fmaxf(most[j], fmaxf(fmaxf(fabsf(v[j][k].x), fabsf(v[j][k].y)),
                                                               fmaxf(fabsf(v[j][k].z), fabsf(v[j][k].w))));
                        }
#pragma unroll
                        for (int d = 1; d < 8; d <<= 1)
#pragma unroll
                            for (int j = 0; j < B; ++j) most[j] = fmaxf(most[j], __shfl_xor_sync(0xffffffffu, most[j], d));
#pragma unroll
                        for (int j = 0; j < B; ++j) {
                            // the row's largest value goes to [2^13, 2^14)
                            const int e = max(14, min(254, (int)(__float_as_uint(most[j]) >> 23)));
                            const float up = __uint_as_float((uint32_t)(254 + 13 - e) << 23);
                            const float of_row = __shfl_sync(0xffffffffu, up, (lane & 3) * 8);  // of row 4 i + lane % 4
                            scaled = (lane >> 2) == i0 + j ? of_row : scaled;
#pragma unroll
                            for (int k = 0; k < N; ++k) {
                                uint2 hi, lo;
                                split2(v[j][k].x * up, v[j][k].y * up, hi.x, lo.x);
                                split2(v[j][k].z * up, v[j][k].w * up, hi.y, lo.y);
                                uint8_t *dst = target(i0 + j, k / 2, (k & 1) * 4 + p / 2) + (p & 1) * 8;
                                *reinterpret_cast<uint2 *>(dst) = hi;
                                *reinterpret_cast<uint2 *>(dst + Sh::QBYTES) = lo;
                            }
                        }
                    }
                    c = c / scaled;
                }
                fence_proxy_async_smem();
                fence_before();  // the previous item's reads of O are complete
                __syncwarp();
                if (lane == 0) arrive(&qready[qt]);
            }
            float m = -INFINITY, l = 0.0f, m_kept = -INFINITY;
            float *const kept = P.kept + ((long long)blockIdx.x * ROWS * D + row * 4);
            for (int tile = it.ta; tile < it.tb; ++tile, ++tiles_done) {
                // A tensor-core sum is cut, not rounded, at every product: over 12000 positions the results
                // came out 6e-6 short.  For fp32 results the sums start anew every kFold tiles, and what
                // they reached is added to a copy in the workspace, which this thread alone touches.
                const bool fold = QS == 2 && tile > it.ta && (tile - it.ta) % kFold == 0;
                if (fold) {
                    wait_product(tiles_done - 1);
                    fence_after();
                    const bool first = tile - it.ta == kFold;
                    const float f = first || m_kept == -INFINITY ? 0.0f : ex2(m_kept - m);
                    m_kept = m;
#pragma unroll 1
                    for (int d = 0; d < D; d += 32) {
                        float o[32];
                        tm_ld32(o_at + d, o);
                        float4 x[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            x[k] = first ? make_float4(0, 0, 0, 0) : *reinterpret_cast<const float4 *>(kept + ((d / 4 + k) * ROWS) * 4);
                        wait_ld();
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            *reinterpret_cast<float4 *>(kept + ((d / 4 + k) * ROWS) * 4) =
                                make_float4(fmaf(f, x[k].x, o[4 * k]), fmaf(f, x[k].y, o[4 * k + 1]), fmaf(f, x[k].z, o[4 * k + 2]),
                                            fmaf(f, x[k].w, o[4 * k + 3]));
                    }
                    fence_before();
                }
                const int buf = tiles_done & 1;
                const uint32_t s_at = s_of + (uint32_t)(buf * KT);
                wait(&sfull[2 * qt + buf], (tiles_done >> 1) & 1u);
                fence_after();
                // ---- which of the tile's positions the row sees: bit k of word w is position 32 w + k
                const uint2 mk = *reinterpret_cast<const uint2 *>(marks + (tiles_done % kMarks) * (KT / 8));
                const bool all = (mk.x & mk.y) == 0xffffffffu && tile * KT + KT - 1 <= see_all;  // warp-uniform
                // ---- the row's scores and their maximum
                float s[KT];
#pragma unroll
                for (int w = 0; w < KT / 32; ++w) tm_ld32(s_at + 32 * w, s + 32 * w);
                wait_ld();
                if (!all) {
                    auto seen = [&](uint32_t m, int first) {
                        const int n = see - first + 1;
                        return m & (n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u);
                    };
                    const uint32_t vis[2] = {seen(mk.x, tile * KT), seen(mk.y, tile * KT + 32)};
#pragma unroll
                    for (int k = 0; k < KT; ++k) s[k] = (vis[k / 32] >> (k & 31)) & 1u ? s[k] : -INFINITY;
                }
                float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int k = 0; k < KT; k += 2) m4[(k / 2) & 3] = max3(m4[(k / 2) & 3], s[k], s[k + 1]);
                const float mx = fmaxf(max3(m4[0], m4[1], m4[2]), m4[3]) * c;
                const bool raise = mx > m + kRaise;
                if (__any_sync(0xffffffffu, raise)) {
                    const float f = raise ? ex2(m - mx) : 1.0f;  // 0 from -inf
                    if (raise) m = mx;
                    l *= f;
                    if (tile > it.ta && !fold) {  // O holds something, once the product before is complete
                        wait_product(tiles_done - 1);
                        fence_after();
#pragma unroll 1
                        for (int d = 0; d < D; d += 16) {
                            float o[16];
                            tm_ld16(o_at + d, o);
                            wait_ld();
#pragma unroll
                            for (int k = 0; k < 16; ++k) o[k] *= f;
                            tm_st16(o_at + d, o);
                        }
                    }
                }
                // ---- weights, over the scores
                const float base = m == -INFINITY ? 0.0f : kLift - m;
                const uint64_t c2 = pair(c, c), base2 = pair(base, base);
                uint64_t sum2[2] = {pair(0.0f, 0.0f), pair(0.0f, 0.0f)};
#pragma unroll
                for (int w = 0; w < KT / 32; ++w) {
                    uint32_t hi[16], lo[QS == 2 ? 16 : 1];
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        float a, b;
                        unpair(fma2(pair(s[32 * w + 2 * k], s[32 * w + 2 * k + 1]), c2, base2), a, b);
                        a = ex2(a);
                        b = ex2(b);
                        sum2[k & 1] = add2(sum2[k & 1], pair(a, b));
                        if constexpr (QS == 1) hi[k] = pack2<C>(a, b);
                        else split2(a, b, hi[k], lo[k]);
                    }
                    tm_st16(s_at + 32 * w, hi);
                    if constexpr (QS == 2) tm_st16(s_at + 32 * w + 16, lo);
                }
                {
                    float a, b;
                    unpair(add2(sum2[0], sum2[1]), a, b);
                    l += a + b;
                }
                wait_st();
                fence_before();
                __syncwarp();
                if (lane == 0) arrive(&pready[2 * qt + buf]);
            }
            // ---- the item's end: O of this part
            wait_product(tiles_done - 1);
            fence_after();
            const bool whole = it.all_mine();
            float *part = P.parts + it.slot_of(blockIdx.x) * ROWS * (D + 2);
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            T *dst = (T *)A.out + q_row * A.out_stride + h_off;
            uint64_t naught[2] = {pair(0.0f, 0.0f), pair(0.0f, 0.0f)};  // NaN once a value is not finite
            // whole rows pass through the warp's part of the query buffer (every product of
            // queries is complete), 128 bytes of each at a time, so that 8 lanes store one row's;
            // piece p of row x lies at p ^ (x & 7): no bank conflicts either way
            uint8_t *const turn = sq + qt * QS * Sh::QBYTES + (warp & 3) * 32 * 128;
            constexpr int PIECE = 128 / sizeof(T);  // elements of a row per round
#pragma unroll 1  // the code of a round is fetched once, which takes as long as running it
            for (int d = 0; d < D; d += PIECE) {
                float o[PIECE];
#pragma unroll
                for (int k = 0; k < PIECE; k += 32) tm_ld32(o_at + d + k, o + k);
                wait_ld();
                if (QS == 2 && it.tb - it.ta > kFold) {
                    const float f = m_kept == -INFINITY ? 0.0f : ex2(m_kept - m);
#pragma unroll
                    for (int k = 0; k < PIECE; k += 4) {
                        const float4 x = *reinterpret_cast<const float4 *>(kept + ((d + k) / 4 * ROWS) * 4);
                        o[k] = fmaf(f, x.x, o[k]), o[k + 1] = fmaf(f, x.y, o[k + 1]);
                        o[k + 2] = fmaf(f, x.z, o[k + 2]), o[k + 3] = fmaf(f, x.w, o[k + 3]);
                    }
                }
#pragma unroll
                for (int k = 0; k < PIECE; k += 2)
                    naught[(k / 2) & 1] = fma2(pair(o[k], o[k + 1]), pair(0.0f, 0.0f), naught[(k / 2) & 1]);
                if (whole) {
#pragma unroll
                    for (int k = 0; k < PIECE; k += 2) unpair(mul2(pair(o[k], o[k + 1]), pair(inv, inv)), o[k], o[k + 1]);
                    constexpr int N = 16 / sizeof(T);
#pragma unroll
                    for (int p = 0; p < 8; ++p) {
                        ElVec<T, N> v;
                        v.set(o + p * N);
                        v.store(reinterpret_cast<T *>(turn + lane * 128 + ((p ^ (lane & 7)) * 16)));
                    }
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int x = 4 * i + (lane >> 3), p = lane & 7;
                        const int xr = qt * kRows + 32 * (warp & 3) + x, tx = token_of(xr);
                        const uint4 v = *reinterpret_cast<const uint4 *>(turn + x * 128 + ((p ^ (x & 7)) * 16));
                        if (xr < rows)
                            *reinterpret_cast<uint4 *>((T *)A.out + (long long)(q.q0 + tok0 + tx) * A.out_stride +
                                                       (long long)(head * G + h0 + xr - tx * gs) * D + d + p * N) = v;
                    }
                    __syncwarp();
                } else if (live) {
#pragma unroll
                    for (int k = 0; k < PIECE; k += 4)
                        *reinterpret_cast<float4 *>(part + ((d + k) / 4 * ROWS + row) * 4) =
                            make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
                }
            }
            if (!whole && live) {
                part[ROWS * D + row] = m;
                part[ROWS * D + ROWS + row] = l;
            }
            // Rows that are not finite are computed again once the CTA's pipeline has ended (redo_rows): a
            // part's ticket is left until then.
            float n0, n1;
            unpair(add2(naught[0], naught[1]), n0, n1);
            if (__any_sync(0xffffffffu, live && !(n0 + n1 == 0.0f)) && lane == 0) *(whole ? &s_again : &s_odd) = 1;
            if (!whole) {
                // ---- the last of the item's CTAs joins the parts, in order
                const int c0 = it.first_cta(), c1 = it.last_cta();
                asm volatile("bar.sync 1, %0;" ::"n"(Sh::SOFT) : "memory");
                if (tid == 0) {
                    if (s_odd) s_odd = 0, s_last = 0, s_later |= 1 << (it.slot_of(blockIdx.x) & 1);
                    else s_last = take_ticket(&P.tickets[c0]) == (unsigned)(c1 - c0);
                }
                asm volatile("bar.sync 1, %0;" ::"n"(Sh::SOFT) : "memory");
                if (s_last) {
                    if (tid == 0) P.tickets[c0] = 0;
                    if (live) join_row<T, D, ROWS>(P, it, row, dst);
                }
                // s_last is read by every thread before it is written again: the next write
                // follows the next item's first bar.sync
            }
        }
    } else if (warp < kIssue) {
        // ================================================================ keys and values
        const int fw = warp - 4 * QT;
        // A tile whose positions all exist comes by tensor copies, one box of 64 dimensions of a
        // page's slots (as many as divide a tile) per copy, each completing on the slot's barrier.
        // The others (a sequence's end, where what lies behind it must read as zeros; pages that
        // are not groups of 8 slots; bad pages) come by 16-byte copies, a row's 8 pieces by 8 lanes.
        constexpr int MINE = KT / Sh::FETCH;        // positions per warp: rows fw MINE + lane / 8 + 4 i
        constexpr int GRP = MINE / 4;
        const uint32_t ring0 = smem_u32(ring);
        int slot = 0, old = 0, pending = 0;         // next slot; the oldest not yet announced
        uint32_t lap = 0;                           // times round the ring
        uint32_t boxed = 0, boxed_par = 0;          // slots last filled by tensor copies, their parities
        bool bad_page = false;
        auto announce = [&]() {  // the caller waited for the copies
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) arrive(&full[old]);
            if (++old == P.slots) old = 0;
            --pending;
        };
        auto drain = [&]() {
            if (pending > 0) {
                copies_left<0>();
                while (pending > 0) announce();
            }
        };
        const int box_rows = P.box_rows, boxes = box_rows ? KT / box_rows : 1;  // boxes of 64 dimensions
        for (; it.part(A.b); it.next(A.b)) {
            const int head = it.head / P.sets, len = it.q.len;
            const int *table = A.b.table + (long long)it.seq * A.b.table_stride;
            // page of the tile's box `lane`, read a tile ahead
            auto box_page = [&](int tile) {
                const int x = tile * KT + (lane & (boxes - 1)) * box_rows;
                return box_rows && tile < it.tb && x < len ? __ldg(table + A.kv.page.div((uint32_t)x)) : -1;
            };
            auto mark = [&](uint32_t have, int i) {  // positions fw MINE + 4 i .. + 3, two i per byte
                if (lane == 0) marks[(tiles_done % kMarks) * (KT / 8) + (fw * MINE + 4 * i) / 8] = (uint8_t)have;
            };
            auto boxed_tile = [&](int tile, int page) {
                return box_rows && (tile + 1) * KT <= len && __all_sync(0xffffffffu, (unsigned)page < (unsigned)A.kv.n_pages);
            };
            auto claim = [&]() {  // the slot is free
                if (lap > 0 && !bad) {
                    const uint32_t par = (lap - 1) & 1u;
                    if (!__all_sync(0xffffffffu, test_once(&empty[slot], par))) {
                        drain();
                        wait(&empty[slot], par);
                    }
                }
            };
            auto fetch_boxes = [&](const void *map, int tile, int page) {
                drain();
                claim();
                if (!bad) {
                    // copy j of boxes x D / 64 by warp j % FETCH: a thread issues them one by one
                    constexpr int H = D / 64;
                    const int mine = (boxes * H - fw + Sh::FETCH - 1) / Sh::FETCH;
                    if (lane == 0) {
                        if (mine > 0) mbar_arrive_expect_tx(&full[slot], (uint32_t)(mine * box_rows) * 128);
                        else arrive(&full[slot]);
                    }
                    __syncwarp();
                    const int j = fw + lane * Sh::FETCH, i = j / H, h = j % H;
                    const int at = __shfl_sync(0xffffffffu, page, i & 31);
                    const int x = tile * KT + i * box_rows;
                    if (lane < mine)
                        box_load(ring0 + (uint32_t)slot * Sh::TBYTES + h * THALF + (uint32_t)(i * box_rows) * 128, map, h * 64,
                                 x - (int)(A.kv.page.div((uint32_t)x) * A.kv.page.d), head, at, &full[slot]);
                    if (mine > 0) {
                        boxed |= 1u << slot;
                        boxed_par = (boxed_par & ~(1u << slot)) | ((lap & 1u) << slot);
                    }
                    if (++old == P.slots) old = 0;
                }
                if (++slot == P.slots) slot = 0, ++lap;
            };
            // a tile that cannot be boxed: the pages of its positions, read a tile ahead too
            auto row_pages = [&](int tile, int (&pg)[GRP]) {
                const bool rows = tile < it.tb && !(box_rows && (tile + 1) * KT <= len);
#pragma unroll
                for (int i = 0; i < GRP; ++i) {
                    const int x = tile * KT + fw * MINE + 4 * i + (lane >> 3);
                    pg[i] = rows && x < len ? __ldg(table + A.kv.page.div((uint32_t)x)) : kUnread;
                }
            };
            auto offsets = [&](int tile, const int (&pg)[GRP], long long (&off)[GRP]) {  // of the lane's piece; -1: none
                uint32_t have = 0;
#pragma unroll
                for (int i = 0; i < GRP; ++i) {
                    const int x = tile * KT + fw * MINE + 4 * i + (lane >> 3);
                    off[i] = -1;
                    if (x < len) {
                        const uint32_t j = A.kv.page.div((uint32_t)x);
                        const int page = pg[i] == kUnread ? __ldg(table + j) : pg[i];
                        if ((unsigned)page < (unsigned)A.kv.n_pages)
                            off[i] = (page * A.kv.page_stride + head * A.kv.head_stride + (x - (int)(j * A.kv.page.d)) * A.kv.slot_stride) *
                                         (long long)sizeof(C) + (lane & 7) * 16;
                        else bad_page = true;
                    }
                    const unsigned b = __ballot_sync(0xffffffffu, off[i] >= 0);  // bits 0, 8, 16, 24: rows
                    have |= ((b & 1u) | ((b >> 7) & 2u) | ((b >> 14) & 4u) | ((b >> 21) & 8u)) << (4 * (i & 1));
                    if (i & 1) {
                        mark(have, i - 1);
                        have = 0;
                    }
                }
            };
            auto fetch_rows = [&](const char *base, const long long (&off)[GRP]) {
                claim();
                if (!bad) {
                    const uint32_t dst = ring0 + (uint32_t)slot * Sh::TBYTES;
#pragma unroll
                    for (int i = 0; i < GRP; ++i) {
                        const int r = fw * MINE + 4 * i + (lane >> 3);
#pragma unroll
                        for (int h = 0; h < D / 64; ++h)
                            copy16(dst + h * THALF + r * 128 + (((lane & 7) ^ (r & 7)) * 16), off[i] >= 0 ? base + off[i] + h * 128 : base,
                                   off[i] >= 0);
                    }
                    asm volatile("cp.async.commit_group;" ::: "memory");
                    if (++pending > kBehind) {
                        copies_left<kBehind>();
                        announce();
                    }
                }
                if (++slot == P.slots) slot = 0, ++lap;
            };
            // K of tile ta, then K of the next tile before V of each
            int page = box_page(it.ta), page1 = -1;
            long long off[GRP], ahead[GRP] = {};
            bool box = false, box1 = false;
            int pages1[GRP];
            auto keys = [&](int tile, int pg, long long (&o)[GRP]) {
                const bool bx = boxed_tile(tile, pg);
                if (bx) {
#pragma unroll
                    for (int i = 0; i < GRP; i += 2) mark(0xffu, i);
                    fetch_boxes(P.map_k, tile, pg);
                } else {
                    offsets(tile, pages1, o);
                    fetch_rows(A.kv.k, o);
                }
                ++tiles_done;
                return bx;
            };
            page1 = box_page(it.ta + 1);
            row_pages(it.ta, pages1);
            box = keys(it.ta, page, off);
            row_pages(it.ta + 1, pages1);
            for (int tile = it.ta; tile < it.tb; ++tile) {
                const int page2 = box_page(tile + 2);
                if (tile + 1 < it.tb) box1 = keys(tile + 1, page1, ahead);
                row_pages(tile + 2, pages1);
                if (box) fetch_boxes(P.map_v, tile, page);
                else fetch_rows(A.kv.v, off);
#pragma unroll
                for (int i = 0; i < GRP; ++i) off[i] = ahead[i];
                box = box1;
                page = page1;
                page1 = page2;
            }
        }
        drain();
        // tensor copies that nothing will wait for any more, after a wait ran out
        if (bad)
            for (int i = 0; i < P.slots; ++i)
                if ((boxed >> i) & 1u) mbar_wait_sleep(&full[i], (boxed_par >> i) & 1u, kWaitCycles / 8);
        if (__any_sync(0xffffffffu, bad_page) && lane == 0) report(A.status, TQB200_PAGED_BAD_PAGE);
    } else {
        // ================================================================ products of query tile qt
        // Every operand of an MMA is made warp-uniform (by shuffles) and one elected lane issues:
        // 64 clocks per 128 x 128 x 16 product, the pipe's own rate; from a branch on the lane
        // number, with the descriptors in per-thread registers, each took 96 to 130.
        auto uniform = [](uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); };
        const int qt = (int)uniform((uint32_t)(warp - kIssue));
        const bool one = elect_one();
        const uint32_t s_of = uniform(tmem) + (uint32_t)(qt * 2 * KT), o_at = uniform(tmem) + (uint32_t)(QT * 2 * KT + qt * D);
        const uint32_t q_at = uniform(smem_u32(sq)) + qt * QS * Sh::QBYTES, ring0 = uniform(smem_u32(ring));
        constexpr uint32_t id_qk = idesc_of<C>(KT, false), id_pv = idesc_of<C>(D, true);
        int slot = 0;
        uint32_t lap = 0, scored = 0;  // tiles whose scores were issued
        // S[scored % 2] = Q K^T of the next K slot
        auto scores = [&]() {
            wait(&full[slot], lap & 1u);
            if (!bad) {
                fence_after();
                const uint64_t qd = row_desc(q_at, 16);
                const uint64_t kd = row_desc(uniform(ring0 + (uint32_t)slot * Sh::TBYTES), 16);
                const int buf = (int)uniform(scored & 1u);
                if (one) {
#pragma unroll
                    for (int sp = QS - 1; sp >= 0; --sp)  // the small terms first: less is cut from them
#pragma unroll
                        for (int ks = 0; ks < D / 16; ++ks)
                            mma_ss(s_of + buf * KT, qd + (sp * Sh::QBYTES + (ks / 4) * QHALF + (ks % 4) * 32) / 16,
                                   kd + ((ks / 4) * THALF + (ks % 4) * 32) / 16, id_qk, ks > 0 || sp < QS - 1);
                    mma_commit(&sfull[2 * qt + buf]);
                    mma_commit(&empty[slot]);
                }
            }
            __syncwarp();
            ++scored;
            if (++slot == P.slots) slot = 0, ++lap;
        };
        auto wait_product = [&](uint32_t n) { wait(&odone[2 * qt + (n & 1u)], (n >> 1) & 1u); };
        for (; qt < QT && it.part(A.b); it.next(A.b), ++items_done) {
            wait(&qready[qt], items_done & 1u);
            scores();
            for (int tile = it.ta; tile < it.tb; ++tile, ++tiles_done) {
                if (tile + 1 < it.tb) {
                    // The buffer holds the weights of the tile before: the product that reads
                    // them has another shape than this one, and only products of one shape and
                    // accumulator are ordered by their issue, so its end is waited for.
                    if (tile > it.ta) wait_product(tiles_done - 1);
                    scores();  // runs while the softmax of this tile does
                }
                const int buf = (int)uniform(tiles_done & 1u);
                wait(&pready[2 * qt + buf], (tiles_done >> 1) & 1u);
                wait(&full[slot], lap & 1u);
                if (!bad) {
                    fence_after();
                    const uint64_t vd = row_desc(uniform(ring0 + (uint32_t)slot * Sh::TBYTES), THALF);
                    const bool more = uniform(tile > it.ta && !(QS == 2 && (tile - it.ta) % kFold == 0)) != 0;
                    const uint32_t p_at = s_of + buf * KT;
                    if (one) {
#pragma unroll
                        for (int kk = 0; kk < KT / 16; ++kk)
#pragma unroll
                            for (int sp = QS - 1; sp >= 0; --sp)
                                mma_ts(o_at, p_at + 32 * (kk >> 1) + 8 * (kk & 1) + 16 * sp, vd + kk * 2 * (1024 / 16), id_pv,
                                       kk > 0 || sp < QS - 1 || more);
                        mma_commit(&odone[2 * qt + buf]);
                        mma_commit(&empty[slot]);
                    }
                }
                __syncwarp();
                if (++slot == P.slots) slot = 0, ++lap;
            }
        }
        if (qt < QT) {  // everything issued above is complete before shared memory and TMEM go
            if (one) mma_commit(&done[qt]);
            if (!mbar_wait_sleep(&done[qt], 0u, kWaitCycles)) s_err = 1;
        }
        __syncwarp();
    }
    fence_before();
    __syncthreads();
    if (warp == kIssue) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Sh::COLS) : "memory");
    }
    if (tid == 0 && s_err) report(A.status, TQB200_PAGED_TIMEOUT);
    if (s_again | s_later) redo_rows<T, C, D, QT>(P, s_again != 0, s_later);
}

// Two parts of up to 256 rows for each of the grid's CTAs, one per SM.
size_t parts_floats(int head_dim) { return (size_t)std::min(4 * num_sms(), 2 * kSplitMaxCtas) * kRows * (size_t)(head_dim + 2); }

// Tensor map over (dimension, slot, head, page) of one of the cache's arrays, boxes of 64
// dimensions x `rows` slots; false: it cannot be mapped.
bool encode_pages(const char *base, const PagedAttnArgs &a, int rows, void *map128) {
    const cuuint64_t dims[4] = {(cuuint64_t)a.head_dim, a.kv.page.d, (cuuint64_t)a.n_kv_heads, (cuuint64_t)a.kv.n_pages};
    const long long in[3] = {a.kv.slot_stride, a.kv.head_stride, a.kv.page_stride};
    cuuint64_t strides[3];
    for (int i = 0; i < 3; ++i) {
        // a dimension of one element may have any stride: a valid one in its place
        strides[i] = (cuuint64_t)(dims[i + 1] == 1 ? a.head_dim : in[i]) * 2;
        if (strides[i] >= (1ull << 40) || strides[i] % 16 != 0) return false;
    }
    const cuuint32_t box[4] = {64u, (cuuint32_t)rows, 1u, 1u}, elem[4] = {1u, 1u, 1u, 1u};
    using Encode = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Encode encode = reinterpret_cast<Encode>(driver_entry("cuTensorMapEncodeTiled"));
    if (!encode) return false;
    CUtensorMap m;
    if (encode(&m, CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, const_cast<char *>(base), dims, strides, box, elem,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return false;
    memcpy(map128, &m, sizeof(m));
    return true;
}

template <typename T, typename C, int D, int QT>
int launch_chunk_t(const PagedAttnArgs &a, cudaStream_t st) {
    using Sh = ChunkShape<T, D, QT>;
    auto k = paged_chunk_kernel<T, C, D, QT>;
    static KernelSmem once;
    int limit = 0;
    TQ_CUDA_TRY(smem_limit_once(k, once, &limit));
    const int fixed = kMeta + QT * Sh::QS * (int)Sh::QBYTES;
    const int slots = std::min(kMaxSlots, (limit - fixed) / (int)Sh::TBYTES);
    TQ_CHECK_ARG(slots >= kBehind + 1, "paged_attention: %d bytes of shared memory hold %d tiles", limit, slots);
    ChunkParams P{};
    P.A = a;
    P.tickets = (unsigned *)a.work;
    P.parts = (float *)((char *)a.work + kSplitTicketBytes);
    P.kept = P.parts + parts_floats(D);
    const int G = a.n_heads / a.n_kv_heads;
    P.sets = (G + Sh::ROWS - 1) / Sh::ROWS;
    P.g_set = (G + P.sets - 1) / P.sets;
    P.line = {Sh::ROWS / P.g_set, a.n_kv_heads * P.sets, 1, 4, 10, 0.6f * QT * D / 128};
    P.slots = slots;
    // boxes that lie in one page and start on the swizzle's groups of 8 rows
    const int rows = std::gcd((int)a.kv.page.d, KT);
    if (rows % 8 == 0) {
        if (encode_pages(a.kv.k, a, rows, P.map_k) && encode_pages(a.kv.v, a, rows, P.map_v)) P.box_rows = rows;
    }
    const long long items = (long long)P.line.heads * (a.b.n_seqs + (long long)a.b.n_tokens / P.line.tq);
    const long long most = items * ((std::max(1, a.b.max_len) + KT - 1) / KT);
    const int grid = (int)std::min<long long>({(long long)num_sms(), most, kSplitMaxCtas});
    k<<<grid, Sh::THREADS, fixed + slots * Sh::TBYTES, st>>>(P);
    TQ_CUDA_TRY(cudaGetLastError());
    return TQB200_OK;
}

template <typename T, typename C>
int launch_chunk_c(const PagedAttnArgs &a, cudaStream_t st) {
    // Two query tiles per item: they take turns at the tensor pipe and halve the reads of the
    // cache.  The products of fp32 queries and weights (two operands each) of head_dim 128 keep the
    // pipe so long that one tile per item, whose blocks of 128 rows reach more SMs, is quicker up to
    // 5 G rows x positions x head_dim: 512 rows of 32 heads over 512 positions (1.1 G) 19.1 us
    // against 24.2, 64 over 6064 (1.6 G) 46 and 60, 1000 over 1000 (4.1 G) 40.5 and 43.3; but 1200
    // over 1200 (5.9 G) 63 and 60, 512 over 4512 (9.5 G) 115 and 91.  Elsewhere two are: 1500 bf16
    // rows over 1500 48.0 us against 56.6, 1000 fp32 rows of head_dim 64 23.9 against 29.9.  (The
    // positions are the page table's width, here that of the longest sequence; with a table of 32768
    // the first takes two tiles and 24.8 us.)
    if (a.head_dim == 64) return launch_chunk_t<T, C, 64, 2>(a, st);
    if constexpr (std::is_same<T, float>::value) {
        const double work = (double)a.b.n_tokens * a.n_heads * a.b.max_len * a.head_dim;
        if (work < 5e9) return launch_chunk_t<T, C, 128, 1>(a, st);
    }
    return launch_chunk_t<T, C, 128, 2>(a, st);
}

}  // namespace

size_t paged_chunk_work_bytes(int head_dim) {
    return kSplitTicketBytes + parts_floats(head_dim) * 4 + (size_t)num_sms() * 2 * kRows * head_dim * 4;
}

int launch_paged_chunk(const PagedAttnArgs &a, cudaStream_t st) {
    if (a.type == TQB200_EL_F32) return launch_chunk_c<float, __half>(a, st);
    if (a.type == TQB200_EL_F16) return launch_chunk_c<__half, __half>(a, st);
    return launch_chunk_c<__nv_bfloat16, __nv_bfloat16>(a, st);
}

}  // namespace tqb200
