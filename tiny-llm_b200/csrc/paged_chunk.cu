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
// of 16-bit operands (128 x 128 scores: 1024 clocks either way), so two query tiles alternate:
// while one is in its softmax the other's products run.
// Roles (warps): QT groups of 4 softmax warps (thread = query row = TMEM lane), 2 QT warps that
// fetch keys and values, QT warps that each issue one query tile's products.
//  * Keys and values come by 16-byte cp.async, one page lookup per position, so any page size
//    and any layout of 16-byte aligned rows is read alike; a ring of slots holds whole K or V
//    tiles in the order K0 V0 K1 V1 ...  A warp's 32 copies are 4 chunks of 8 positions, whose
//    16-byte pieces are adjacent in shared memory (no bank conflicts).  Positions past the end
//    and on bad pages are filled with zeros and marked in a bitmap.
//  * Shared memory holds the canonical layout without swizzle: 8 x 16-byte core matrices, the
//    D / 8 of 8 positions adjacent.  It serves K as the K-major and V as the MN-major B operand.
//  * Softmax: the row's maximum is raised only when a score passes it by 2^8 (then the warp
//    rescales its rows of O in TMEM); weights carry a factor 2^6 against fp16's subnormals,
//    so they stay below 2^14.
//  * fp32 activations over an fp16 cache: Q (scaled per row by a power of two) and P are
//    split into fp16 hi + lo, two products each: 22 bits of either operand.
//  * Every wait is bounded; after one runs out the roles go on without waiting or issuing, the
//    issued copies and products are waited for (bounded), TMEM is freed and the error stored.
#include <algorithm>
#include <type_traits>

#include "paged.cuh"

namespace tqb200 {
namespace {

constexpr float kRaise = 8.0f;
constexpr float kLift = 6.0f;
constexpr int kRows = 128;        // query rows per tile: TMEM lanes
constexpr int kMaxSlots = 8;
constexpr int kMarks = 16;        // tiles whose bitmaps are kept (more than the ring holds)
constexpr int kMeta = 1024;

struct ChunkParams {
    PagedAttnArgs A;
    unsigned *tickets;
    float *parts;     // [2 grid]: [D / 4][rows][4] accumulators, [rows] maxima, [rows] sums
    LineShape line;
    int sets, g_set;
    int slots;
};

// ---------------------------------------------------------------- tcgen05
__device__ __forceinline__ uint64_t core_desc(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(sbo >> 4) << 32) |
           (1ull << 46);
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
__device__ __forceinline__ void tm_ld32(uint32_t a, float (&v)[32]) {
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
__device__ __forceinline__ void tm_st32(uint32_t a, const float (&v)[32]) {
    uint32_t r[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(v[i]);
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(a),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tm_st16(uint32_t a, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(a),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
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

template <typename T, int D, int QT, int KT>
struct ChunkShape {
    static constexpr int QS = std::is_same<T, float>::value ? 2 : 1;
    static constexpr int SOFT = QT * 128;                       // softmax threads
    static constexpr int FETCH = 2 * QT;                        // warps that fetch
    // whole groups of 4 warps; 16 warps per SM either way: 128 registers a thread at launch
    static constexpr int THREADS = 256 * QT;
    static constexpr int ROWS = QT * kRows;
    static constexpr uint32_t QBYTES = kRows * D * 2;           // one operand of one query tile
    static constexpr uint32_t TBYTES = KT * D * 2;              // one slot: a K or a V tile
    static constexpr uint32_t COLS = QT * (KT + D) <= 256 ? 256 : 512;  // TMEM columns
    // per SM: two where the queries leave room for it
    static constexpr int CTAS = QT == 1 && QS * QBYTES <= 32768 ? 2 : 1;
    static_assert(QT * (KT + D) <= 512, "TMEM");
};

// ---------------------------------------------------------------- the kernel
template <typename T, typename C, int D, int QT, int KT>
__global__ void __launch_bounds__(ChunkShape<T, D, QT, KT>::THREADS, ChunkShape<T, D, QT, KT>::CTAS)
    paged_chunk_kernel(const __grid_constant__ ChunkParams P) {
    using Sh = ChunkShape<T, D, QT, KT>;
    constexpr int QS = Sh::QS, ROWS = Sh::ROWS;
    constexpr uint32_t LINE8 = D / 8 * 128;  // bytes of 8 positions (or query rows)
    extern __shared__ __align__(1024) uint8_t smem[];
    const PagedAttnArgs &A = P.A;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint64_t *full = reinterpret_cast<uint64_t *>(smem);   // [slots] tile landed (every fetch warp)
    uint64_t *empty = full + kMaxSlots;                    // [slots] tile read by every query tile's products
    uint64_t *sfull = empty + kMaxSlots;                   // [QT] scores in TMEM
    uint64_t *pready = sfull + QT;                         // [QT] weights in TMEM (4 warps)
    uint64_t *odone = pready + QT;                         // [QT] P V complete
    uint64_t *qready = odone + QT;                         // [QT] queries in shared memory, O free (4 warps)
    uint64_t *done = qready + QT;                          // [QT] every product of the issuing warp complete
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(done + QT);
    uint8_t *marks = smem + 512;                           // [kMarks][KT / 8]: positions that exist
    static_assert(kMarks * KT / 8 <= kMeta - 512, "marks");
    uint8_t *sq = smem + kMeta;
    uint8_t *ring = sq + QT * QS * Sh::QBYTES;
    __shared__ int s_err;
    __shared__ unsigned s_last;

    if (tid == 0) {
        for (int i = 0; i < P.slots; ++i) {
            mbar_init(&full[i], Sh::FETCH);
            mbar_init(&empty[i], QT);
        }
        for (int i = 0; i < QT; ++i) {
            mbar_init(&sfull[i], 1);
            mbar_init(&pready[i], 4);
            mbar_init(&odone[i], 1);
            mbar_init(&qready[i], 4);
            mbar_init(&done[i], 1);
        }
        fence_mbar_init();
        s_err = 0;
    }
    Line<KT> it;
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
    uint32_t tiles_done = 0;  // of this CTA, over all its items: phase of the per-tile barriers
    uint32_t items_done = 0;

    if (warp < 4 * QT) {
        // ================================================================ softmax
        if constexpr (QT == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");  // 8 x 184 + 8 x 72 = 16 x 128
        const int qt = warp >> 2, r = tid & 127;
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t s_at = tmem + lanes + (uint32_t)(qt * KT), o_at = tmem + lanes + (uint32_t)(QT * KT + qt * D);
        for (; it.part(A.b); it.next(A.b), ++items_done) {
            const SeqInfo &q = it.q;
            const int head = it.head / P.sets, h0 = (it.head - head * P.sets) * P.g_set;
            const int gs = min(P.g_set, G - h0), tok0 = it.b * P.line.tq;
            const int rows = min(P.line.tq, q.n - tok0) * gs;
            const int p0 = q.len - q.n + tok0;
            const int row = qt * kRows + r;
            const bool live = row < rows;
            const int tok = row / gs;
            const long long q_row = (long long)(q.q0 + tok0 + tok);
            const long long h_off = (long long)(head * G + h0 + row - tok * gs) * D;
            const int see = live ? p0 + tok : -1;
            float c = A.scale * kLog2e;
            // ---- the row to shared memory
            {
                uint8_t *dst = sq + qt * QS * Sh::QBYTES + (r >> 3) * LINE8 + (r & 7) * 16;
                const T *src = (const T *)A.q + q_row * A.q_stride + h_off;
                if constexpr (QS == 1) {
#pragma unroll
                    for (int j = 0; j < D / 8; ++j)
                        *reinterpret_cast<uint4 *>(dst + j * 128) =
                            live ? *reinterpret_cast<const uint4 *>(src + j * 8) : make_uint4(0, 0, 0, 0);
                } else {
                    float most = 0.0f;
                    if (live) {
#pragma unroll 8
                        for (int j = 0; j < D / 4; ++j) {
                            const float4 f = *reinterpret_cast<const float4 *>(src + j * 4);
                            most = fmaxf(most, fmaxf(fmaxf(fabsf(f.x), fabsf(f.y)), fmaxf(fabsf(f.z), fabsf(f.w))));
                        }
                    }
                    // the row's largest value goes to [2^13, 2^14)
                    const int e = max(14, min(254, (int)(__float_as_uint(most) >> 23)));
                    const float up = __uint_as_float((uint32_t)(254 + 13 - e) << 23);
                    c = c / up;
#pragma unroll 4
                    for (int j = 0; j < D / 8; ++j) {
                        float4 f = make_float4(0, 0, 0, 0), h = f;
                        if (live) {
                            f = *reinterpret_cast<const float4 *>(src + j * 8);
                            h = *reinterpret_cast<const float4 *>(src + j * 8 + 4);
                        }
                        uint4 hi, lo;
                        split2(f.x * up, f.y * up, hi.x, lo.x);
                        split2(f.z * up, f.w * up, hi.y, lo.y);
                        split2(h.x * up, h.y * up, hi.z, lo.z);
                        split2(h.z * up, h.w * up, hi.w, lo.w);
                        *reinterpret_cast<uint4 *>(dst + j * 128) = hi;
                        *reinterpret_cast<uint4 *>(dst + Sh::QBYTES + j * 128) = lo;
                    }
                }
                fence_proxy_async_smem();
                fence_before();  // the previous item's reads of O are complete
                __syncwarp();
                if (lane == 0) arrive(&qready[qt]);
            }
            float m = -INFINITY, l = 0.0f;
            for (int tile = it.ta; tile < it.tb; ++tile, ++tiles_done) {
                const uint32_t ph = tiles_done & 1u;
                wait(&sfull[qt], ph);
                fence_after();
                // ---- which of the tile's positions the row sees: bit k of word w is position 32 w + k
                uint32_t vis[KT / 32];
                bool all = true;
                {
                    const uint32_t *mk = reinterpret_cast<const uint32_t *>(marks + (tiles_done % kMarks) * (KT / 8));
#pragma unroll
                    for (int w = 0; w < KT / 32; ++w) {
                        const int n = see - (tile * KT + 32 * w) + 1;
                        vis[w] = mk[w] & (n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u);
                        all = all && vis[w] == 0xffffffffu;
                    }
                    all = __all_sync(0xffffffffu, all);
                }
                // ---- the row's maximum
                float mx = -INFINITY;
#pragma unroll
                for (int w = 0; w < KT / 32; ++w) {
                    float s[32];
                    tm_ld32(s_at + 32 * w, s);
                    wait_ld();
                    float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                    if (all) {
#pragma unroll
                        for (int k = 0; k < 32; ++k) m4[k & 3] = fmaxf(m4[k & 3], s[k]);
                    } else {
#pragma unroll
                        for (int k = 0; k < 32; ++k) m4[k & 3] = fmaxf(m4[k & 3], (vis[w] >> k) & 1u ? s[k] : -INFINITY);
                    }
                    mx = fmaxf(mx, fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])));
                }
                mx *= c;
                const bool raise = mx > m + kRaise;
                if (__any_sync(0xffffffffu, raise)) {
                    const float f = raise ? ex2(m - mx) : 1.0f;  // 0 from -inf
                    if (raise) m = mx;
                    l *= f;
                    if (tile > it.ta) {  // O holds something, once the product before is complete
                        wait(&odone[qt], ph ^ 1u);
                        fence_after();
#pragma unroll
                        for (int d = 0; d < D; d += 32) {
                            float o[32];
                            tm_ld32(o_at + d, o);
                            wait_ld();
#pragma unroll
                            for (int k = 0; k < 32; ++k) o[k] *= f;
                            tm_st32(o_at + d, o);
                        }
                    }
                }
                // ---- weights, over the scores
                const float base = m == -INFINITY ? 0.0f : kLift - m;
                float sum4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int w = 0; w < KT / 32; ++w) {
                    float s[32];
                    tm_ld32(s_at + 32 * w, s);
                    wait_ld();
#pragma unroll
                    for (int k = 0; k < 32; ++k) s[k] = ex2(fmaf(s[k], c, base));
                    if (!all) {
#pragma unroll
                        for (int k = 0; k < 32; ++k) s[k] = (vis[w] >> k) & 1u ? s[k] : 0.0f;
                    }
#pragma unroll
                    for (int k = 0; k < 32; ++k) sum4[k & 3] += s[k];
                    uint32_t hi[16];
                    if constexpr (QS == 1) {
#pragma unroll
                        for (int k = 0; k < 16; ++k) hi[k] = pack2<C>(s[2 * k], s[2 * k + 1]);
                    } else {
                        uint32_t lo[16];
#pragma unroll
                        for (int k = 0; k < 16; ++k) split2(s[2 * k], s[2 * k + 1], hi[k], lo[k]);
                        tm_st16(s_at + 32 * w + 16, lo);
                    }
                    tm_st16(s_at + 32 * w, hi);
                }
                l += (sum4[0] + sum4[1]) + (sum4[2] + sum4[3]);
                wait_st();
                fence_before();
                __syncwarp();
                if (lane == 0) arrive(&pready[qt]);
            }
            // ---- the item's end: O of this part
            wait(&odone[qt], (tiles_done - 1) & 1u);
            fence_after();
            const bool whole = it.all_mine();
            float *part = P.parts + it.slot_of(blockIdx.x) * ROWS * (D + 2);
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            T *dst = (T *)A.out + q_row * A.out_stride + h_off;
            bool odd = false;
#pragma unroll
            for (int d = 0; d < D; d += 32) {
                float o[32];
                tm_ld32(o_at + d, o);
                wait_ld();
#pragma unroll
                for (int k = 0; k < 32; ++k) odd |= (__float_as_uint(o[k]) & 0x7f800000u) == 0x7f800000u;
                if (!live) continue;
                if (whole) {
#pragma unroll
                    for (int k = 0; k < 32; ++k) o[k] *= inv;
#pragma unroll
                    for (int k = 0; k < 32; k += 16 / sizeof(T)) {
                        ElVec<T, 16 / sizeof(T)> v;
                        v.set(o + k);
                        v.store(dst + d + k);
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < 32; k += 4)
                        *reinterpret_cast<float4 *>(part + ((d + k) / 4 * ROWS + row) * 4) =
                            make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
                }
            }
            if (!whole && live) {
                part[ROWS * D + row] = m;
                part[ROWS * D + ROWS + row] = l;
            }
            // A weight of 0 does not hide an infinity or NaN among values that the row does not
            // see: rows that are not finite are computed again by a pass over what they see.
            unsigned again = __ballot_sync(0xffffffffu, odd && live);
            while (again) {  // warp-uniform
                const int src = __ffs((int)again) - 1;
                again &= again - 1;
                const long long rr = __shfl_sync(0xffffffffu, q_row, src), hh = __shfl_sync(0xffffffffu, h_off, src);
                const int ss = __shfl_sync(0xffffffffu, see, src), rw = __shfl_sync(0xffffffffu, row, src);
                float mr, lr, orow[8];
                row_pass<T, C>(A, (const T *)A.q + rr * A.q_stride + hh, it.seq, head, it.ta * KT, min(it.tb * KT, ss + 1), mr,
                               lr, orow);
                const float f = whole ? (lr == 0.0f ? 0.0f : 1.0f / lr) : exp2f(kLift);
#pragma unroll
                for (int j = 0; j < D / 32; ++j) {
                    const int e = lane + 32 * j;
                    if (whole) ((T *)A.out + rr * A.out_stride + hh)[e] = el_from_f<T>(orow[j] * f);
                    else part[(e / 4 * ROWS + rw) * 4 + (e & 3)] = orow[j] * f;
                }
                if (!whole && lane == 0) {
                    part[ROWS * D + rw] = mr;
                    part[ROWS * D + ROWS + rw] = lr * f;
                }
            }
            if (!whole) {
                // ---- the last of the item's CTAs joins the parts, in order
                const int c0 = it.first_cta(), c1 = it.last_cta();
                __threadfence();
                asm volatile("bar.sync 1, %0;" ::"n"(Sh::SOFT) : "memory");
                if (tid == 0) s_last = atomicAdd(&P.tickets[c0], 1u) == (unsigned)(c1 - c0);
                asm volatile("bar.sync 1, %0;" ::"n"(Sh::SOFT) : "memory");
                if (s_last) {
                    __threadfence();
                    if (tid == 0) P.tickets[c0] = 0;
                    if (live) {
                        float M = -INFINITY, L = 0.0f;
                        for (int i = c0; i <= c1; ++i)
                            M = fmaxf(M, __ldcg(P.parts + it.slot_of(i) * ROWS * (D + 2) + ROWS * D + row));
                        const float b = M == -INFINITY ? 0.0f : M;
                        for (int i = c0; i <= c1; ++i) {
                            const float *pp = P.parts + it.slot_of(i) * ROWS * (D + 2) + ROWS * D + row;
                            L = fmaf(ex2(__ldcg(pp) - b), __ldcg(pp + ROWS), L);
                        }
                        const float li = L == 0.0f ? 0.0f : 1.0f / L;
                        for (int d = 0; d < D; d += 32) {
                            float o[32];
#pragma unroll
                            for (int k = 0; k < 32; ++k) o[k] = 0.0f;
                            for (int i = c0; i <= c1; ++i) {
                                const float *pp = P.parts + it.slot_of(i) * ROWS * (D + 2);
                                const float f = ex2(__ldcg(pp + ROWS * D + row) - b);
#pragma unroll
                                for (int k = 0; k < 32; k += 4) {
                                    const float4 x = __ldcg(reinterpret_cast<const float4 *>(pp + ((d + k) / 4 * ROWS + row) * 4));
                                    o[k] = fmaf(f, x.x, o[k]), o[k + 1] = fmaf(f, x.y, o[k + 1]);
                                    o[k + 2] = fmaf(f, x.z, o[k + 2]), o[k + 3] = fmaf(f, x.w, o[k + 3]);
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
                }
                // s_last is read by every thread before it is written again: the next write
                // follows the next item's first bar.sync
            }
        }
    } else if (warp < kIssue) {
        // ================================================================ keys and values
        if constexpr (QT == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        const int fw = warp - 4 * QT;
        constexpr int GRP = KT / 8 / Sh::FETCH;     // groups of 8 positions per warp
        const uint32_t ring0 = smem_u32(ring);
        const uint32_t my = (uint32_t)(fw * GRP) * LINE8 + (uint32_t)(lane >> 3) * 128 + (uint32_t)(lane & 7) * 16;
        int slot = 0, old = 0, pending = 0;         // next slot; the oldest not yet announced
        uint32_t lap = 0;                           // times round the ring
        bool bad_page = false;
        auto announce = [&]() {  // the caller waited for the copies
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) arrive(&full[old]);
            if (++old == P.slots) old = 0;
            --pending;
        };
        for (; it.part(A.b); it.next(A.b)) {
            const int head = it.head / P.sets, len = it.q.len;
            const int *table = A.b.table + (long long)it.seq * A.b.table_stride;
            auto place_of = [&](int tile, int i) { return tile * KT + (fw * GRP + i) * 8 + (lane & 7); };
            int page[GRP];
#pragma unroll
            for (int i = 0; i < GRP; ++i) {
                const int x = place_of(it.ta, i);
                page[i] = x < len ? __ldg(table + A.kv.page.div((uint32_t)x)) : -1;
            }
            for (int tile = it.ta; tile < it.tb; ++tile, ++tiles_done) {
                long long off[GRP];
#pragma unroll
                for (int i = 0; i < GRP; ++i) {
                    const int x = place_of(tile, i);
                    off[i] = -1;
                    if (x < len) {
                        if ((unsigned)page[i] < (unsigned)A.kv.n_pages) {
                            const int in = x - (int)(A.kv.page.div((uint32_t)x) * A.kv.page.d);
                            off[i] = (page[i] * A.kv.page_stride + head * A.kv.head_stride + in * A.kv.slot_stride) * (long long)sizeof(C) +
                                     (lane >> 3) * 16;
                        } else {
                            bad_page = true;
                        }
                    }
                    const unsigned have = __ballot_sync(0xffffffffu, off[i] >= 0);
                    if (lane == 0) marks[(tiles_done % kMarks) * (KT / 8) + fw * GRP + i] = (uint8_t)have;
                    const int xn = place_of(tile + 1, i);
                    page[i] = tile + 1 < it.tb && xn < len ? __ldg(table + A.kv.page.div((uint32_t)xn)) : -1;
                }
#pragma unroll
                for (int kv = 0; kv < 2; ++kv) {
                    if (lap > 0 && !bad) {
                        const uint32_t par = (lap - 1) & 1u;
                        if (!__all_sync(0xffffffffu, test_once(&empty[slot], par))) {
                            copies_left<0>();
                            while (pending > 0) announce();
                            wait(&empty[slot], par);
                        }
                    }
                    if (!bad) {
                        const char *base = kv ? A.kv.v : A.kv.k;
                        const uint32_t dst = ring0 + (uint32_t)slot * Sh::TBYTES + my;
#pragma unroll
                        for (int i = 0; i < GRP; ++i)
#pragma unroll
                            for (int j = 0; j < D / 32; ++j)
                                copy16(dst + i * LINE8 + j * 512, off[i] >= 0 ? base + off[i] + j * 64 : base, off[i] >= 0);
                        asm volatile("cp.async.commit_group;" ::: "memory");
                        ++pending;
                        if (pending > 2) {
                            copies_left<2>();
                            announce();
                        }
                    }
                    if (++slot == P.slots) slot = 0, ++lap;
                }
            }
        }
        copies_left<0>();
        while (pending > 0) announce();
        if (__any_sync(0xffffffffu, bad_page) && lane == 0) report(A.status, TQB200_PAGED_BAD_PAGE);
    } else {
        // ================================================================ products of query tile qt
        if constexpr (QT == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        const int qt = warp - kIssue;
        const uint32_t s_at = tmem + (uint32_t)(qt * KT), o_at = tmem + (uint32_t)(QT * KT + qt * D);
        const uint32_t q_at = smem_u32(sq) + qt * QS * Sh::QBYTES, ring0 = smem_u32(ring);
        constexpr uint32_t id_qk = idesc_of<C>(KT, false), id_pv = idesc_of<C>(D, true);
        int slot = 0;
        uint32_t lap = 0;
        auto advance = [&]() {
            if (++slot == P.slots) slot = 0, ++lap;
        };
        for (; qt < QT && it.part(A.b); it.next(A.b), ++items_done) {
            wait(&qready[qt], items_done & 1u);
            for (int tile = it.ta; tile < it.tb; ++tile, ++tiles_done) {
                // scores; the slots of K and V alternate, so K of the next tile follows V of this one
                wait(&full[slot], lap & 1u);
                if (!bad && lane == 0) {
                    fence_after();
                    const uint32_t k_at = ring0 + (uint32_t)slot * Sh::TBYTES;
#pragma unroll
                    for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
                        for (int sp = QS - 1; sp >= 0; --sp)
                            mma_ss(s_at, core_desc(q_at + sp * Sh::QBYTES + ks * 256, 128, LINE8),
                                   core_desc(k_at + ks * 256, 128, LINE8), id_qk, ks > 0 || sp < QS - 1);
                    mma_commit(&sfull[qt]);
                    mma_commit(&empty[slot]);
                }
                __syncwarp();
                advance();
                wait(&pready[qt], tiles_done & 1u);
                wait(&full[slot], lap & 1u);
                if (!bad && lane == 0) {
                    fence_after();
                    const uint32_t v_at = ring0 + (uint32_t)slot * Sh::TBYTES;
#pragma unroll
                    for (int kk = 0; kk < KT / 16; ++kk)
#pragma unroll
                        for (int sp = QS - 1; sp >= 0; --sp)
                            mma_ts(o_at, s_at + 32 * (kk >> 1) + 8 * (kk & 1) + 16 * sp,
                                   core_desc(v_at + kk * 2 * LINE8, LINE8, 128), id_pv, tile > it.ta || kk > 0 || sp < QS - 1);
                    mma_commit(&odone[qt]);
                    mma_commit(&empty[slot]);
                }
                __syncwarp();
                advance();
            }
        }
        if (qt < QT && lane == 0) {  // everything issued above is complete before shared memory and TMEM go
            mma_commit(&done[qt]);
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
}

template <typename T, typename C, int D, int QT, int KT>
int launch_chunk_t(const PagedAttnArgs &a, cudaStream_t st) {
    using Sh = ChunkShape<T, D, QT, KT>;
    auto k = paged_chunk_kernel<T, C, D, QT, KT>;
    static KernelSmem once;
    int limit = 0;
    TQ_CUDA_TRY(smem_limit_once(k, once, &limit));
    if (Sh::CTAS == 2) limit = std::min(limit, 112 * 1024);  // of the SM's 228 KB, 1 KB per CTA reserved
    const int fixed = kMeta + QT * Sh::QS * (int)Sh::QBYTES;
    const int slots = std::min(kMaxSlots, (limit - fixed) / (int)Sh::TBYTES);
    TQ_CHECK_ARG(slots >= 3, "paged_attention: %d bytes of shared memory hold %d tiles", limit, slots);
    ChunkParams P{};
    P.A = a;
    P.tickets = (unsigned *)a.work;
    P.parts = (float *)((char *)a.work + kSplitTicketBytes);
    const int G = a.n_heads / a.n_kv_heads;
    P.sets = (G + Sh::ROWS - 1) / Sh::ROWS;
    P.g_set = (G + P.sets - 1) / P.sets;
    P.line = {Sh::ROWS / P.g_set, a.n_kv_heads * P.sets, 1, 8};
    P.slots = slots;
    const long long items = (long long)P.line.heads * (a.b.n_seqs + (long long)a.b.n_tokens / P.line.tq);
    const long long most = items * ((std::max(1, a.b.max_len) + KT - 1) / KT);
    const int grid = (int)std::min<long long>({(long long)num_sms() * Sh::CTAS, most, kSplitMaxCtas});
    k<<<grid, Sh::THREADS, fixed + slots * Sh::TBYTES, st>>>(P);
    TQ_CUDA_TRY(cudaGetLastError());
    return TQB200_OK;
}

template <typename T, typename C>
int launch_chunk_c(const PagedAttnArgs &a, cudaStream_t st) {
    constexpr bool split = std::is_same<T, float>::value;
    const bool big = (long long)a.b.n_tokens * a.n_heads >= 256LL * num_sms();
    if (a.head_dim == 64)
        return big ? launch_chunk_t<T, C, 64, 2, 128>(a, st) : launch_chunk_t<T, C, 64, 1, 64>(a, st);
    if constexpr (split) return big ? launch_chunk_t<T, C, 128, 2, 64>(a, st) : launch_chunk_t<T, C, 128, 1, 64>(a, st);
    else return big ? launch_chunk_t<T, C, 128, 2, 128>(a, st) : launch_chunk_t<T, C, 128, 1, 64>(a, st);
}

}  // namespace

size_t paged_chunk_work_bytes(int head_dim) {
    const size_t slots = std::min(4 * num_sms(), 2 * kSplitMaxCtas);  // 2 per CTA of 128 rows: 2 CTAs per SM
    return kSplitTicketBytes + slots * kRows * (size_t)(head_dim + 2) * 4;
}

int launch_paged_chunk(const PagedAttnArgs &a, cudaStream_t st) {
    if (a.type == TQB200_EL_F32) return launch_chunk_c<float, __half>(a, st);
    if (a.type == TQB200_EL_F16) return launch_chunk_c<__half, __half>(a, st);
    return launch_chunk_c<__nv_bfloat16, __nv_bfloat16>(a, st);
}

}  // namespace tqb200
