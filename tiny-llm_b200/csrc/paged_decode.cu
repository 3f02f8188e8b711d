// paged_decode.cu — causal attention of few new rows (single tokens, short chunks) over a paged
// KV cache on mma.sync, in blocks of up to 8 or 16 query rows; every chunk over an fp32 cache.
// sm_100a.
//
// Bound: HBM (every key and value is read once per block of rows), or latency for short
// contexts.  A tcgen05 tile would spend 128 rows on these few, and its
// operands would have to pass through shared memory; here keys and values go from global
// memory into the registers of the warp that uses them, 16 bytes a lane, and never touch
// shared memory.  The products run on mma.sync with the KEYS as the 16 rows and the queries as
// the 8 columns (transposed products):
//   S^T [16 keys x 8 rows] = K [16 x D] Q^T [D x 8],   O^T [D x 8] += V^T [D x 16] P^T [16 x 8].
//  * A dot product does not care about the order of its terms, so lane (g, t) of the A operand
//    (row g, columns 2t, 2t+1, 2t+8, 2t+9) takes dimensions 8(t + 4j) .. + 7 of key g: one
//    16-byte load feeds two products, and the queries are laid out alike.
//  * V^T as the A operand wants pairs of keys for one dimension: lane (g, t) loads dimensions
//    8g .. 8g+7 of keys 2t, 2t+1, 2t+8, 2t+9 and interleaves the halves of two keys' words.
//  * P^T as the B operand is the 8x8 transpose of the S^T accumulator (movmatrix).
//  * fp32 activations over an fp16 cache: q is scaled per row by a power of two (its largest
//    value to 2^13..2^14) and split into two fp16 (hi + lo: 22 bits), the weights likewise.
//  * fp32 cache: tf32 products of operands split in two (hi hi + hi lo + lo hi: 2^-21 of the
//    product), the accumulators transposed by shuffles.
// Softmax: each warp keeps its own running maximum per row (shared by the warp's lanes),
// raised only when a score passes it by 2^4 (one vote per 16 keys; else no shuffles), so
// weights are at most 2^4; they carry a factor 2^6 that keeps small ones out of fp16's
// subnormals.  Sums and accumulators are fp32.  Of 16-bit activations a weight goes into P V in the
// cache's type, off by at most half a step, its sum as it was: the results of 64 tokens over up
// to 8192 bf16 positions are 2.0e-3 off 64 bits, 1.7e-3 of it their own rounding; a second part
// for the weights would double the products.  The next 16 keys (and then values) are in
// flight while the present ones are used; page numbers are read one step further ahead.
//
// Measured on one B200 (device time): 64 single tokens of 32 heads over 8 KV heads of 128, 126
// thousand bf16 positions (516 MB): 88 us, 5.9 TB/s of the 6.5 of a copy; one token over 4096
// fp16 positions (16.8 MB) 15.6 us, of which planning takes 1.4, the queries and first keys
// 2.4, two steps of 64 keys 2.6, the join of 33 parts 4.5; 3 tokens over up to 40 fp32
// positions 6.0 us.  With one chain of sums for the scores a step took 530 clocks longer; with
// the planning in 64-bit divisions and two barriers every call took 4 us longer.  Where results
// are fp32, each step's sums start at zero in the tensor core and are added to the accumulators
// in fp32: the tensor core cuts its sums, which over 12000 positions came to 6e-6.  Over an
// fp32 cache a chunk of 2000 rows of 32 heads over up to 8000 positions takes 6.6 ms (5.4 with
// running sums), 35 TFLOP/s: three tf32 products per term, and each block of 16 rows reads the
// cache again from L2.
#include <algorithm>
#include <type_traits>

#include "paged.cuh"

namespace tqb200 {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kSub = 16;                // keys of a warp's step
constexpr int kTile = kSub * kWarps;    // keys of a CTA's step: the unit of the split
constexpr float kRaise = 4.0f;          // log2 by which a score may pass the running maximum
constexpr float kLift = 6.0f;           // log2 of the weights' common factor

struct DecodeParams {
    PagedAttnArgs A;
    unsigned *tickets;
    float *parts;     // [2 grid][rows][HD + 2]: accumulators, then maximum, sum
    LineShape line;
    int sets, g_set;  // sets of at most g_set query heads that a KV head's queries fall into
};

// ---------------------------------------------------------------- mma.sync
template <typename C>
__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                      uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<C, __half>::value)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
// tf32 keeps 10 bits after the point: hi is x cut there (exact), lo what is left, rounded there
// (to nearest; cut, it would be short of x more often than not)
__device__ __forceinline__ void tf32_split(float x, uint32_t &hi, uint32_t &lo) {
    hi = __float_as_uint(x) & 0xffffe000u;
    lo = (__float_as_uint(x - __uint_as_float(hi)) + 0x1000u) & 0xffffe000u;
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
// hi = the fp16 of (a, b), lo = the fp16 of what is left
__device__ __forceinline__ void split2(float a, float b, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&l);
}
__device__ __forceinline__ uint4 ld16(const char *p) {  // read once
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t word(const uint4 &v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// row_pass out of line: the kernel's registers are its own.
template <typename T, typename C, int E>
__device__ __noinline__ void row_again(const PagedAttnArgs &A, const T *q, int seq, int kv_head, int x0, int x1, float &m,
                                       float &l, float (&o)[E]) {
    row_pass<T, C, E>(A, q, seq, kv_head, x0, x1, m, l, o);
}

// ---------------------------------------------------------------- the kernel
// T activations, C cache, D head_dim, NB blocks of 8 query rows.
template <typename C, int D, int NB>
constexpr int kPerSm = D == 64 ? (NB == 1 ? 4 : std::is_same<C, float>::value ? 2 : 3)
                               : (NB == 1 && !std::is_same<C, float>::value ? 3 : 2);  // CTAs: by registers

template <typename T, typename C, int D, int NB>
__global__ void __launch_bounds__(kThreads, kPerSm<C, D, NB>) paged_decode_kernel(const __grid_constant__ DecodeParams P) {
    constexpr bool F32 = std::is_same<C, float>::value;
    constexpr bool SPLIT = !F32 && std::is_same<T, float>::value;  // hi + lo fp16 operands
    constexpr int QS = F32 || SPLIT ? 2 : 1;
    constexpr int ROWS = 8 * NB;
    constexpr int EL = 16 / sizeof(C);     // elements of a 16-byte load
    constexpr int KC = D / (4 * EL);       // loads per key
    constexpr int VC = D / (8 * EL);       // loads per value row
    constexpr int MT = D / 16;             // 16-dimension tiles of O^T
    constexpr bool QREG = NB * QS * KC <= 4;  // query operands kept in registers
    const PagedAttnArgs &A = P.A;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;

    // one buffer, in turn: the query operands while the item's tiles are read, the warps'
    // accumulators at its end, the weights of up to 128 parts when they are joined
    constexpr size_t kBuf = std::max({sizeof(float) * kWarps * ROWS * D, sizeof(uint4) * QS * NB * KC * 32,
                                      sizeof(float) * 2 * ROWS * kThreads});
    __shared__ __align__(16) char s_buf[kBuf];
    auto &s_o = *reinterpret_cast<float(*)[kWarps][ROWS][D]>(s_buf);
    auto &s_q = *reinterpret_cast<uint4(*)[QS * NB * KC][32]>(s_buf);
    auto &s_w = *reinterpret_cast<float(*)[ROWS][kThreads]>(s_buf);
    auto &s_p = *reinterpret_cast<float(*)[ROWS][kThreads]>(s_buf + sizeof(float) * ROWS * kThreads);
    __shared__ float s_m[kWarps][ROWS], s_l[kWarps][ROWS];
    __shared__ float s_c[ROWS];
    __shared__ unsigned s_last;

    Line<kTile> it;
    it.begin<kThreads>(A.b, P.line, A.status);
    const int G = A.n_heads / A.n_kv_heads;

    for (; it.part(A.b); it.next(A.b)) {
        // ---- the item: rows (token, query head) of one KV head, tokens tok0 ..
        const SeqInfo &q = it.q;
        const int head = it.head / P.sets, h0 = (it.head - head * P.sets) * P.g_set;
        const int gs = min(P.g_set, G - h0);  // query heads of this set
        const int ta = it.ta, tb = it.tb, tok0 = it.b * P.line.tq;
        const int rows = min(P.line.tq, q.n - tok0) * gs;
        const int p0 = q.len - q.n + tok0;  // position of the first row
        const int *table = A.b.table + (long long)it.seq * A.b.table_stride;
        const uint32_t recip = (65535u + (uint32_t)gs) / (uint32_t)gs;  // r / gs for r < 256
        auto token_of = [&](int r) { return (int)(((uint32_t)r * recip) >> 16); };
        auto row_at = [&](int r, long long stride) {
            const int t = token_of(r);
            return (long long)(q.q0 + tok0 + t) * stride + (long long)(head * G + h0 + r - t * gs) * D;
        };
        auto row_q = [&](int r) {
            return (const T *)A.q + row_at(r, A.q_stride);
        };

        // ---- page offsets of a step's 16 keys: lane l (mod 16) has key l
        auto page_of = [&](int tile) -> int {  // the page number, read ahead
            const int x = tile * kTile + warp * kSub + (lane & 15);
            return tile < tb && x < q.len ? __ldg(table + A.kv.page.div((uint32_t)x)) : -1;
        };
        int bad_page = 0;
        auto offset_of = [&](int tile, int page) -> long long {
            const int x = tile * kTile + warp * kSub + (lane & 15);
            if (tile >= tb || x >= q.len) return -1;
            if ((unsigned)page >= (unsigned)A.kv.n_pages) {
                bad_page = 1;
                return -1;
            }
            const int slot = x - (int)(A.kv.page.div((uint32_t)x) * A.kv.page.d);
            return (page * A.kv.page_stride + head * A.kv.head_stride + slot * A.kv.slot_stride) * (long long)sizeof(C);
        };
        uint4 kr[2][KC], vr[4][VC];
        // key g and g + 8 of 16
        auto load_k = [&](long long off) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const long long o = __shfl_sync(0xffffffffu, off, g + 8 * h);
                const char *p = A.kv.k + o + t4 * 16;
#pragma unroll
                for (int j = 0; j < KC; ++j) kr[h][j] = o >= 0 ? ld16(p + j * 64) : make_uint4(0, 0, 0, 0);
            }
        };
        // values of keys 2t, 2t+1, 2t+8, 2t+9 (16 bits), t, t+4, t+8, t+12 (fp32)
        auto v_key = [&](int i) { return F32 ? t4 + 4 * i : 2 * t4 + (i & 1) + 8 * (i >> 1); };
        auto load_v = [&](long long off) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const long long o = __shfl_sync(0xffffffffu, off, v_key(i));
                const char *p = A.kv.v + o + g * 16;
#pragma unroll
                for (int j = 0; j < VC; ++j) vr[i][j] = o >= 0 ? ld16(p + j * 128) : make_uint4(0, 0, 0, 0);
            }
        };
        int page1 = page_of(ta);
        // the queries' loads go out before the keys', which wait for their pages
        constexpr int QW = std::is_same<T, float>::value ? EL / 4 : 1;  // 16-byte loads per piece
        uint4 qraw[NB][KC][QW];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            if (!QREG && warp != (nb & (kWarps - 1))) continue;
            const int r = 8 * nb + g;
            const T *src = row_q(min(r, rows - 1)) + t4 * EL;
#pragma unroll
            for (int j = 0; j < KC; ++j)
#pragma unroll
                for (int e = 0; e < QW; ++e)
                    qraw[nb][j][e] = r < rows ? *reinterpret_cast<const uint4 *>(src + j * 4 * EL + e * 4) : make_uint4(0, 0, 0, 0);
        }
        long long off = offset_of(ta, page1);
        page1 = page_of(ta + 1);
        load_k(off);
        load_v(off);

        // ---- queries: lane (g, t) holds row 8 nb + g, dimensions EL (t + 4 j) .. of it
        uint4 qr[QREG ? QS * NB * KC : 1];
        float c[NB][2];   // log2(e) * scale (* 2^-row scale) of this lane's two columns per block
        int see[NB][2];   // last position that the column's row sees, -1: none
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const int r = 8 * nb + g;
            float up = 1.0f, c_row = A.scale * kLog2e;
            if (QREG || warp == (nb & (kWarps - 1))) {
                if constexpr (std::is_same<T, float>::value) {
                    float x[KC][EL];
                    float most = 0.0f;
#pragma unroll
                    for (int j = 0; j < KC; ++j)
#pragma unroll
                        for (int e = 0; e < EL; ++e) {
                            x[j][e] = __uint_as_float(word(qraw[nb][j][e / 4], e & 3));
                            most = fmaxf(most, fabsf(x[j][e]));
                        }
                    if constexpr (SPLIT) {
                        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                        // most in [2^(e-127), 2^(e-126)) goes to [2^13, 2^14)
                        const int e = max(14, min(254, (int)(__float_as_uint(most) >> 23)));
                        up = __uint_as_float((uint32_t)(254 + 13 - e) << 23);
                        c_row = c_row / up;
                    }
#pragma unroll
                    for (int j = 0; j < KC; ++j) {
                        uint32_t hi[4], lo[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if constexpr (F32) tf32_split(x[j][e], hi[e], lo[e]);
                            else split2(x[j][2 * e] * up, x[j][2 * e + 1] * up, hi[e], lo[e]);
                        }
                        const uint4 h4 = make_uint4(hi[0], hi[1], hi[2], hi[3]), l4 = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                        if constexpr (QREG) {
                            qr[nb * KC + j] = h4;
                            qr[(NB + nb) * KC + j] = l4;
                        } else {
                            s_q[nb * KC + j][lane] = h4;
                            s_q[(NB + nb) * KC + j][lane] = l4;
                        }
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < KC; ++j) {
                        const uint4 v = qraw[nb][j][0];
                        if constexpr (QREG) qr[nb * KC + j] = v;
                        else s_q[nb * KC + j][lane] = v;
                    }
                }
                if (!QREG && t4 == 0) s_c[r] = c_row;
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int col = 8 * nb + 2 * t4 + e;
                if (QREG) c[nb][e] = __shfl_sync(0xffffffffu, c_row, (2 * t4 + e) * 4);
                see[nb][e] = col < rows ? p0 + token_of(col) : -1;
            }
        }
        if (!QREG) {
            __syncthreads();
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int e = 0; e < 2; ++e) c[nb][e] = s_c[8 * nb + 2 * t4 + e];
        }
        auto q_op = [&](int s, int nb, int j) -> uint4 {
            if constexpr (QREG) return qr[(s * NB + nb) * KC + j];
            else return s_q[(s * NB + nb) * KC + j][lane];
        };

        float o[NB][MT][4];
        float m[NB][2], l[NB][2];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[nb][i][e] = 0.0f;
            m[nb][0] = m[nb][1] = -INFINITY;
            l[nb][0] = l[nb][1] = 0.0f;
        }

        for (int tile = ta; tile < tb; ++tile) {
            const int x0 = tile * kTile + warp * kSub;
            const long long next = offset_of(tile + 1, page1);
            page1 = page_of(tile + 2);
            const unsigned have = __ballot_sync(0xffffffffu, off >= 0);
            off = next;
            // ---- scores: s[0], s[1] key g with columns 2t, 2t+1; s[2], s[3] key g + 8
            // (two or three chains of sums each: the products' latency is theirs)
            float s[NB][4];
            if constexpr (F32) {
                float s2[NB][4], s3[NB][4];
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[nb][e] = s2[nb][e] = 0.0f;
#pragma unroll
                for (int j = 0; j < KC; ++j) {
                    // the large terms of 8 dimensions by themselves, added on by fp32 additions
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s3[nb][e] = 0.0f;
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        uint32_t hi[4], lo[4];
                        tf32_split(__uint_as_float(word(kr[0][j], 2 * u)), hi[0], lo[0]);
                        tf32_split(__uint_as_float(word(kr[1][j], 2 * u)), hi[1], lo[1]);
                        tf32_split(__uint_as_float(word(kr[0][j], 2 * u + 1)), hi[2], lo[2]);
                        tf32_split(__uint_as_float(word(kr[1][j], 2 * u + 1)), hi[3], lo[3]);
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            const uint4 qh = q_op(0, nb, j), ql = q_op(1, nb, j);
                            mma_tf32(s2[nb], lo, word(qh, 2 * u), word(qh, 2 * u + 1));
                            mma_tf32(s2[nb], hi, word(ql, 2 * u), word(ql, 2 * u + 1));
                            mma_tf32(s3[nb], hi, word(qh, 2 * u), word(qh, 2 * u + 1));
                        }
                    }
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[nb][e] += s3[nb][e];
                }
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[nb][e] += s2[nb][e];
            } else {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    float s2[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[nb][e] = s2[e] = 0.0f;
#pragma unroll
                    for (int j = 0; j < KC; ++j)
#pragma unroll
                        for (int sp = QS - 1; sp >= 0; --sp) {
                            const uint4 b = q_op(sp, nb, j);
                            mma16<C>(sp ? s2 : s[nb], kr[0][j].x, kr[1][j].x, kr[0][j].y, kr[1][j].y, b.x, b.y);
                            mma16<C>(QS == 1 || sp ? s2 : s[nb], kr[0][j].z, kr[1][j].z, kr[0][j].w, kr[1][j].w, b.z, b.w);
                        }
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[nb][e] += s2[e];
                }
            }
            load_k(off);
            // ---- masks and the running maximum
            bool raise = false;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int x = x0 + g + 8 * (e >> 1);
                    const bool ok = x <= see[nb][e & 1] && ((have >> (g + 8 * (e >> 1))) & 1u);
                    s[nb][e] = ok ? s[nb][e] * c[nb][e & 1] : -INFINITY;
                    raise |= s[nb][e] > m[nb][e & 1] + kRaise;
                }
            if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float mx = fmaxf(s[nb][e], s[nb][e + 2]);
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
                        if (mx > m[nb][e]) {
                            const float f = ex2(m[nb][e] - mx);  // 0 from -inf
                            m[nb][e] = mx;
                            l[nb][e] *= f;
#pragma unroll
                            for (int i = 0; i < MT; ++i) o[nb][i][e] *= f, o[nb][i][e + 2] *= f;
                        }
                    }
            }
            // ---- weights
            uint32_t pb[QS][NB][2][2];  // B operands: [split][block][k8 step (fp32)][b0, b1]; 16 bits: [..][0]
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                float p[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float base = m[nb][e & 1] == -INFINITY ? 0.0f : m[nb][e & 1] - kLift;
                    p[e] = ex2(s[nb][e] - base);
                    l[nb][e & 1] += p[e];
                }
                if constexpr (F32) {
#pragma unroll
                    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                        for (int b = 0; b < 2; ++b) {
                            const int src = (t4 + 4 * b) * 4 + (g >> 1);
                            const float v0 = __shfl_sync(0xffffffffu, p[2 * kk], src);
                            const float v1 = __shfl_sync(0xffffffffu, p[2 * kk + 1], src);
                            tf32_split((g & 1) ? v1 : v0, pb[0][nb][kk][b], pb[1][nb][kk][b]);
                        }
                } else if constexpr (SPLIT) {
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        uint32_t hi, lo;
                        split2(p[2 * b], p[2 * b + 1], hi, lo);
                        pb[0][nb][0][b] = transpose8x8(hi);
                        pb[1][nb][0][b] = transpose8x8(lo);
                    }
                } else {
#pragma unroll
                    for (int b = 0; b < 2; ++b) pb[0][nb][0][b] = transpose8x8(pack2<C>(p[2 * b], p[2 * b + 1]));
                }
            }
            // ---- values.  A product cuts its sum instead of rounding it, always towards zero: where the
            // results are fp32 a step's products are summed apart and added to the rest by fp32 additions.
            if constexpr (F32) {
#pragma unroll
                for (int j = 0; j < VC; ++j)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int kk = 0; kk < 2; ++kk) {
                            uint32_t hi[4], lo[4];
                            tf32_split(__uint_as_float(word(vr[2 * kk][j], 2 * i)), hi[0], lo[0]);
                            tf32_split(__uint_as_float(word(vr[2 * kk][j], 2 * i + 1)), hi[1], lo[1]);
                            tf32_split(__uint_as_float(word(vr[2 * kk + 1][j], 2 * i)), hi[2], lo[2]);
                            tf32_split(__uint_as_float(word(vr[2 * kk + 1][j], 2 * i + 1)), hi[3], lo[3]);
#pragma unroll
                            for (int nb = 0; nb < NB; ++nb) {
                                float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                                mma_tf32(d, lo, pb[0][nb][kk][0], pb[0][nb][kk][1]);
                                mma_tf32(d, hi, pb[1][nb][kk][0], pb[1][nb][kk][1]);
                                mma_tf32(d, hi, pb[0][nb][kk][0], pb[0][nb][kk][1]);
#pragma unroll
                                for (int e = 0; e < 4; ++e) o[nb][j * 2 + i][e] += d[e];
                            }
                        }
            } else {
#pragma unroll
                for (int j = 0; j < VC; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t wa = word(vr[0][j], i), wb = word(vr[1][j], i);
                        const uint32_t wc = word(vr[2][j], i), wd = word(vr[3][j], i);
                        const uint32_t a0 = __byte_perm(wa, wb, 0x5410), a1 = __byte_perm(wa, wb, 0x7632);
                        const uint32_t a2 = __byte_perm(wc, wd, 0x5410), a3 = __byte_perm(wc, wd, 0x7632);
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            if constexpr (QS == 1) {
                                mma16<C>(o[nb][j * 4 + i], a0, a1, a2, a3, pb[0][nb][0][0], pb[0][nb][0][1]);
                            } else {
                                float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                                mma16<C>(d, a0, a1, a2, a3, pb[1][nb][0][0], pb[1][nb][0][1]);
                                mma16<C>(d, a0, a1, a2, a3, pb[0][nb][0][0], pb[0][nb][0][1]);
#pragma unroll
                                for (int e = 0; e < 4; ++e) o[nb][j * 4 + i][e] += d[e];
                            }
                        }
                    }
            }
            load_v(off);
        }
        if (__any_sync(0xffffffffu, bad_page) && lane == 0) report(A.status, TQB200_PAGED_BAD_PAGE);

        // ---- the warps' parts, joined through shared memory
        // A weight of 0 does not hide an infinity or NaN among values that a row does not see, and the split
        // of an operand makes a NaN of its own from an infinity (lo = 0 or of the other sign beside hi):
        // results that are not finite are computed again by a pass over what the row sees.
        uint64_t naught[2] = {pair(0.0f, 0.0f), pair(0.0f, 0.0f)};  // NaN once a value is not finite
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int e = 0; e < 4; e += 2)
                    naught[e / 2] = fma2(pair(o[nb][i][e], o[nb][i][e + 1]), pair(0.0f, 0.0f), naught[e / 2]);
        float n0, n1;
        unpair(add2(naught[0], naught[1]), n0, n1);
        const bool odd = !(n0 + n1 == 0.0f);
        const bool slow = __syncthreads_or(odd);  // also: every warp is done with the query operands
        if (slow) {
            for (int r = warp; r < ROWS; r += kWarps) {
                float mr = -INFINITY, lr = 0.0f, orow[D / 32];
                if (r < rows) {
                    const int x1 = min(tb * kTile, p0 + token_of(r) + 1);
                    row_again<T, C, D / 32>(A, row_q(r), it.seq, head, ta * kTile, x1, mr, lr, orow);
                    const float lift = exp2f(kLift);
                    lr *= lift;
#pragma unroll
                    for (int j = 0; j < D / 32; ++j) orow[j] *= lift;
                }
                for (int w = 0; w < kWarps; ++w) {
                    if (lane == 0) s_m[w][r] = w ? -INFINITY : mr, s_l[w][r] = w ? 0.0f : lr;
#pragma unroll
                    for (int j = 0; j < D / 32; ++j) s_o[w][r][lane + 32 * j] = w || r >= rows ? 0.0f : orow[j];
                }
            }
        } else {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) l[nb][e] += __shfl_xor_sync(0xffffffffu, l[nb][e], d);
                    if (g == 0) {
                        s_m[warp][8 * nb + 2 * t4 + e] = m[nb][e];
                        s_l[warp][8 * nb + 2 * t4 + e] = l[nb][e];
                    }
                }
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    constexpr int TJ = F32 ? 2 : 4;  // tiles per load
                    const int d = (i / TJ) * 8 * EL + EL * g + 2 * (i % TJ);
                    *reinterpret_cast<float2 *>(&s_o[warp][8 * nb + 2 * t4][d]) = make_float2(o[nb][i][0], o[nb][i][2]);
                    *reinterpret_cast<float2 *>(&s_o[warp][8 * nb + 2 * t4 + 1][d]) = make_float2(o[nb][i][1], o[nb][i][3]);
                }
            }
        }
        __syncthreads();
        const bool whole = it.all_mine();
        float *part = P.parts + it.slot_of(blockIdx.x) * ROWS * (D + 2);
        for (int i = tid; i < rows * (D / 4); i += kThreads) {
            const int r = i / (D / 4), d = (i % (D / 4)) * 4;
            float M = s_m[0][r];
#pragma unroll
            for (int w = 1; w < kWarps; ++w) M = fmaxf(M, s_m[w][r]);
            const float base = M == -INFINITY ? 0.0f : M;
            float L = 0.0f;
            float4 v = make_float4(0, 0, 0, 0);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float f = ex2(s_m[w][r] - base);
                const float4 x = *reinterpret_cast<const float4 *>(&s_o[w][r][d]);
                L = fmaf(f, s_l[w][r], L);
                v.x = fmaf(f, x.x, v.x), v.y = fmaf(f, x.y, v.y), v.z = fmaf(f, x.z, v.z), v.w = fmaf(f, x.w, v.w);
            }
            if (whole) {
                const float inv = L == 0.0f ? 0.0f : 1.0f / L;
                const float y[4] = {v.x * inv, v.y * inv, v.z * inv, v.w * inv};
                ElVec<T, 4> ov;
                ov.set(y);
                ov.store((T *)A.out + row_at(r, A.out_stride) + d);
            } else {
                *reinterpret_cast<float4 *>(part + r * D + d) = v;
                if (d == 0) part[ROWS * D + r] = M, part[ROWS * D + ROWS + r] = L;
            }
        }
        if (!whole) {
            // ---- the item's parts from CTAs c0 .. c1; the last to arrive joins them in order
            const int c0 = it.first_cta(), c1 = it.last_cta();
            __syncthreads();
            if (tid == 0) s_last = take_ticket(&P.tickets[c0]) == (unsigned)(c1 - c0);
            __syncthreads();
            if (s_last) {  // uniform
                auto part_of = [&](int cta) { return P.parts + it.slot_of(cta) * ROWS * (D + 2); };
                constexpr int PER = ROWS * D / 4 / kThreads;  // float4 of the result per thread
                float4 acc[PER];
#pragma unroll
                for (int k = 0; k < PER; ++k) acc[k] = make_float4(0, 0, 0, 0);
                // 128 parts at a time: their maxima and sums to shared memory (thread = part), the
                // running maximum and sum of every row (warp = row), the weights, the values
                for (int b = c0; b <= c1; b += kThreads) {
                    const int cnt = min(kThreads, c1 + 1 - b);
                    if (tid < cnt) {
                        const float *pp = part_of(b + tid) + ROWS * D;
                        for (int r = 0; r < rows; ++r) s_w[r][tid] = __ldcg(pp + r), s_p[r][tid] = __ldcg(pp + ROWS + r);
                    }
                    __syncthreads();
                    for (int r = warp; r < rows; r += kWarps) {
                        const float m0 = b == c0 ? -INFINITY : s_m[0][r], l0 = b == c0 ? 0.0f : s_l[0][r];
                        float M = m0;
                        for (int i = lane; i < cnt; i += 32) M = fmaxf(M, s_w[r][i]);
#pragma unroll
                        for (int d = 16; d > 0; d >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
                        const float base = M == -INFINITY ? 0.0f : M;
                        float L = 0.0f;
                        for (int i = lane; i < cnt; i += 32) {
                            const float f = ex2(s_w[r][i] - base);
                            s_w[r][i] = f;
                            L = fmaf(f, s_p[r][i], L);
                        }
                        L = warp_sum(L);
                        const float old = ex2(m0 - base);
                        __syncwarp();
                        if (lane == 0) s_m[0][r] = M, s_l[0][r] = fmaf(old, l0, L), s_c[r] = old;
                    }
                    __syncthreads();
#pragma unroll
                    for (int k = 0; k < PER; ++k) {
                        const int i = tid + k * kThreads, r = i / (D / 4), d = (i % (D / 4)) * 4;
                        if (r < rows) {
                            const float old = s_c[r];
                            acc[k].x *= old, acc[k].y *= old, acc[k].z *= old, acc[k].w *= old;
#pragma unroll 16
                            for (int w = 0; w < cnt; ++w) {
                                const float4 x = __ldcg(reinterpret_cast<const float4 *>(part_of(b + w) + r * D + d));
                                const float f = s_w[r][w];
                                acc[k].x = fmaf(f, x.x, acc[k].x), acc[k].y = fmaf(f, x.y, acc[k].y);
                                acc[k].z = fmaf(f, x.z, acc[k].z), acc[k].w = fmaf(f, x.w, acc[k].w);
                            }
                        }
                    }
                    __syncthreads();
                }
#pragma unroll
                for (int k = 0; k < PER; ++k) {
                    const int i = tid + k * kThreads, r = i / (D / 4), d = (i % (D / 4)) * 4;
                    if (r < rows) {
                        const float L = s_l[0][r], inv = L == 0.0f ? 0.0f : 1.0f / L;
                        const float y[4] = {acc[k].x * inv, acc[k].y * inv, acc[k].z * inv, acc[k].w * inv};
                        ElVec<T, 4> ov;
                        ov.set(y);
                        ov.store((T *)A.out + row_at(r, A.out_stride) + d);
                    }
                }
                if (tid == 0) P.tickets[c0] = 0;  // ready for the next call
            }
        }
        __syncthreads();  // shared memory free for the next item
    }
}

template <typename T, typename C, int D, int NB>
int launch_decode_t(const PagedAttnArgs &a, cudaStream_t st) {
    static std::atomic<int> s_occ{0};
    int occ = s_occ.load();
    auto k = paged_decode_kernel<T, C, D, NB>;
    if (!occ) {
        TQ_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&occ, k, kThreads, 0));
        TQ_CHECK_ARG(occ >= 1, "paged_attention: the decode kernel does not fit an SM");
        s_occ.store(occ);
    }
    DecodeParams P{};
    P.A = a;
    P.tickets = (unsigned *)a.work;
    P.parts = (float *)((char *)a.work + kSplitTicketBytes);
    const int G = a.n_heads / a.n_kv_heads;
    P.sets = (G + 8 * NB - 1) / (8 * NB);
    P.g_set = (G + P.sets - 1) / P.sets;
    P.line = {8 * NB / P.g_set, a.n_kv_heads * P.sets, 2, 1, 2, 0.03f};
    // no more CTAs than there can be tiles
    const long long items = (long long)P.line.heads * (a.b.n_seqs + (long long)a.b.n_tokens / P.line.tq);
    const long long most = items * ((std::max(1, a.b.max_len) + kTile - 1) / kTile);
    const int grid = (int)std::min<long long>({(long long)num_sms() * std::min(occ, 4), most, kSplitMaxCtas});
    k<<<grid, kThreads, 0, st>>>(P);
    TQ_CUDA_TRY(cudaGetLastError());
    return TQB200_OK;
}

template <typename T, typename C>
int launch_decode_c(const PagedAttnArgs &a, cudaStream_t st) {
    const bool few = (long long)a.b.max_q_len * (a.n_heads / a.n_kv_heads) <= 8;
    if (a.head_dim == 64) return few ? launch_decode_t<T, C, 64, 1>(a, st) : launch_decode_t<T, C, 64, 2>(a, st);
    return few ? launch_decode_t<T, C, 128, 1>(a, st) : launch_decode_t<T, C, 128, 2>(a, st);
}

}  // namespace

size_t paged_decode_work_bytes(int head_dim) {
    const size_t ctas = std::min(4 * num_sms(), kSplitMaxCtas);
    return kSplitTicketBytes + 2 * ctas * kDecodeRows * (size_t)(head_dim + 2) * 4;
}

int launch_paged_decode(const PagedAttnArgs &a, cudaStream_t st) {
    if (a.type == TQB200_EL_F32)
        return a.cache_type == TQB200_EL_F32 ? launch_decode_c<float, float>(a, st) : launch_decode_c<float, __half>(a, st);
    if (a.type == TQB200_EL_F16) return launch_decode_c<__half, __half>(a, st);
    return launch_decode_c<__nv_bfloat16, __nv_bfloat16>(a, st);
}

}  // namespace tqb200
