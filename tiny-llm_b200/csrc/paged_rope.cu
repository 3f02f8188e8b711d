// paged_rope.cu — per-head RMSNorm of queries and keys with rotate-half RoPE, to other rows
// or (append) into the pages of a KV cache, sm_100a.
//
//   x~ = x * (mean(x^2) + eps)^-1/2 * w                       (w absent: x~ = x)
//   y_i = x~_i cos a_i - x~_{i+h} sin a_i,  y_{i+h} = x~_{i+h} cos a_i + x~_i sin a_i,
//   h = rotary_dim / 2, i < h, a_i = position * theta^(-i/h); y = x~ past rotary_dim.
//
// Bound: HBM for long chunks (every value is read and written once), latency for a few
// tokens.  A head's row is held by 2^k lanes, 16 bytes of activations each (head_dim 128:
// 16 lanes for 16-bit types, 32 for fp32), so a warp handles 32 / 2^k rows at a time.  The
// lane of element i + h is a fixed distance away, so the rotation is one shuffle of the raw
// words.  The angle depends on (token, lane) only: a warp keeps its token and folds w, cos
// and sin into two factors per element, held in registers over all the token's heads:
//   y = rsqrt(..) * (x * (w cos) + x_partner * (w_partner * +-sin)).
// Angles are formed in double (position * theta^(-i/h) / 2 pi, its fraction taken before it
// is rounded to fp32), so far positions keep their phase; one exp2 per lane, the
// neighbouring frequencies by multiplication.  A few tokens are spread over up to 16 warps
// per SM (heads split), many tokens get one warp each.
#include <algorithm>
#include <cmath>

#include "paged.cuh"

namespace tqb200 {
namespace {

constexpr int kRopeThreads = 128;
constexpr int kRopeUnroll = 4;  // row groups whose loads are in flight together

struct RopeParams {
    RopeArgs a;
    PagedView kv;
    BatchView b;
    int *status;
    int lane_bits;           // log2 of the lanes of a row
    int warps;               // warps per token
    double log2_step;        // log2(theta) / h: frequency i is 2^(-i log2_step)
    double ratio;            // 2^-log2_step
};

// The row's place in its sequence; false: the row is left as it is.
template <bool APPEND>
__device__ __forceinline__ bool row_place(const RopeParams &P, int tok, int *table_row, int *cache_pos,
                                          int *rope_pos) {
    *cache_pos = 0;
    *table_row = 0;
    if constexpr (APPEND) {
        const int s = seq_of_row(P.b, tok);
        const SeqInfo q = seq_info(P.b, s);
        if (!q.ok) {
            if ((threadIdx.x & 31) == 0) report(P.status, TQB200_PAGED_BAD_SEQ);
            return false;
        }
        if (tok < q.q0 || tok >= q.q0 + q.n) return false;
        *table_row = s;
        *cache_pos = q.len - q.n + (tok - q.q0);
    }
    *rope_pos = P.a.positions ? P.a.positions[tok] : *cache_pos;
    return true;
}

template <typename T, typename C, bool APPEND>
__global__ void __launch_bounds__(kRopeThreads) rope_vec_kernel(const __grid_constant__ RopeParams P) {
    constexpr int VEC = 16 / sizeof(T);
    const RopeArgs &a = P.a;
    const long long gw = (long long)blockIdx.x * (kRopeThreads / 32) + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    const long long tok_ll = gw / P.warps;
    if (tok_ll >= a.n_tokens) return;  // warp-uniform; no CTA barrier below
    const int tok = (int)tok_ll, part = (int)(gw - tok_ll * P.warps);
    int seq, pos, rpos;
    if (!row_place<APPEND>(P, tok, &seq, &pos, &rpos)) return;

    const int lpr = 1 << P.lane_bits, rpi = 32 >> P.lane_bits;
    const int sub = lane >> P.lane_bits, c = lane & (lpr - 1);
    const bool in_row = c * VEC < a.head_dim;
    const int hc = a.rotary_dim / 2 / VEC;  // lanes of one rotated half
    const bool rot = c < 2 * hc, low = c < hc;
    const int partner = lane + (rot ? (low ? hc : -hc) : 0);
    // row groups: n_q of queries, n_k of keys, then (append) n_k of values
    const int n_q = (a.n_heads + rpi - 1) / rpi, n_k = (a.n_kv_heads + rpi - 1) / rpi;
    const int n_it = n_q + (APPEND ? 2 : 1) * n_k;

    auto source = [&](int it, int &head, int &count) -> const T * {
        const char *base;
        long long stride;
        if (it < n_q) base = (const char *)a.q, stride = a.q_stride, count = a.n_heads;
        else if (it < n_q + n_k) it -= n_q, base = (const char *)a.k, stride = a.k_stride, count = a.n_kv_heads;
        else it -= n_q + n_k, base = (const char *)a.v, stride = a.v_stride, count = a.n_kv_heads;
        head = it * rpi + sub;
        return reinterpret_cast<const T *>(base) + tok * stride + (long long)head * a.head_dim + c * VEC;
    };
    ElVec<T, VEC> raw[kRopeUnroll];
    auto load_group = [&](int it0) {
#pragma unroll
        for (int u = 0; u < kRopeUnroll; ++u) {
            const int it = it0 + u * P.warps;
#pragma unroll
            for (int w = 0; w < 4; ++w) raw[u].w[w] = 0u;
            if (it < n_it) {
                int head, count;
                const T *p = source(it, head, count);
                if (head < count && in_row) raw[u].load(p);
            }
        }
    };
    load_group(part);

    // where this token's keys and values go, and its angles
    long long slot = -1;
    if constexpr (APPEND) {
        if (pos >= 0 && a.n_kv_heads > 0) {
            int bad = 0;
            slot = P.kv.offset(P.b.table + (long long)seq * P.b.table_stride, pos, 0, &bad);
            if (bad && lane == 0) report(P.status, TQB200_PAGED_BAD_PAGE);
        }
    }
    float fq[2][VEC], fk[2][VEC];  // factors of x and of its partner
    {
        float cs[VEC], sn[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) cs[j] = 1.0f, sn[j] = 0.0f;
        if (rot) {
            const int i0 = (low ? c : c - hc) * VEC;
            double f = exp2(-(double)i0 * P.log2_step) * 0.15915494309189533577;  // turns per position
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                double t = (double)rpos * f;
                t -= rint(t);
                float s_, c_;
                sincospif(2.0f * (float)t, &s_, &c_);
                cs[j] = c_;
                sn[j] = low ? -s_ : s_;
                f *= P.ratio;
            }
        }
        const int pc = c + (rot ? (low ? hc : -hc) : 0);  // the partner's lane in the row
        auto factors = [&](const float *w, float (&f)[2][VEC]) {
            if (w == nullptr || !in_row) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) f[0][j] = cs[j], f[1][j] = sn[j];
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    f[0][j] = w[c * VEC + j] * cs[j];
                    f[1][j] = w[pc * VEC + j] * sn[j];
                }
            }
        };
        factors(a.q_norm, fq);
        factors(a.k_norm, fk);
    }

    const float inv_n = 1.0f / (float)a.head_dim;
    auto turn = [&](const ElVec<T, VEC> &x, const float (&f)[2][VEC], bool norm, float (&y)[VEC]) {
        float r = 1.0f;
        if (norm) {
            float ss = 0.0f;
#pragma unroll
            for (int j = 0; j < VEC; ++j) ss = fmaf(x.get(j), x.get(j), ss);
            for (int o = lpr >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            r = rsqrtf(fmaf(ss, inv_n, a.eps));
        }
        ElVec<T, VEC> xp;
#pragma unroll
        for (int w = 0; w < 4; ++w) xp.w[w] = __shfl_sync(0xffffffffu, x.w[w], partner);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            // lanes without a rotation keep x alone: 0 * a partner's infinity would be NaN
            const float other = rot ? xp.get(j) * f[1][j] : 0.0f;
            y[j] = r * fmaf(x.get(j), f[0][j], other);
        }
    };

    for (int it0 = part; it0 < n_it; it0 += kRopeUnroll * P.warps) {
        if (it0 != part) load_group(it0);
#pragma unroll
        for (int u = 0; u < kRopeUnroll; ++u) {
            const int it = it0 + u * P.warps;
            if (it >= n_it) break;  // warp-uniform
            float y[VEC];
            if (it < n_q) {
                turn(raw[u], fq, a.q_norm != nullptr, y);
                const int head = it * rpi + sub;
                if (head < a.n_heads && in_row) {
                    ElVec<T, VEC> o;
                    o.set(y);
                    o.store((T *)a.q_out + tok * a.q_out_stride + (long long)head * a.head_dim + c * VEC);
                }
            } else if (it < n_q + n_k) {
                turn(raw[u], fk, a.k_norm != nullptr, y);
                const int head = (it - n_q) * rpi + sub;
                if (head < a.n_kv_heads && in_row) {
                    if constexpr (APPEND) {
                        ElVec<C, VEC> o;
                        o.set(y);
                        if (slot >= 0) o.store((C *)P.kv.k + slot + head * P.kv.head_stride + c * VEC);
                    } else {
                        ElVec<T, VEC> o;
                        o.set(y);
                        o.store((T *)a.k_out + tok * a.k_out_stride + (long long)head * a.head_dim + c * VEC);
                    }
                }
            } else if constexpr (APPEND) {
                const int head = (it - n_q - n_k) * rpi + sub;
                if (head < a.n_kv_heads && in_row && slot >= 0) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) y[j] = raw[u].get(j);
                    ElVec<C, VEC> o;
                    o.set(y);
                    o.store((C *)P.kv.v + slot + head * P.kv.head_stride + c * VEC);
                }
            }
        }
    }
}

// Any head_dim up to 256 and any alignment: one warp per row, lane l holds elements l, l + 32,
// ...; the partner's value is read again from memory (before any lane writes: q_out may be q).
template <typename T, typename C, bool APPEND>
__global__ void __launch_bounds__(kRopeThreads) rope_any_kernel(const __grid_constant__ RopeParams P) {
    const RopeArgs &a = P.a;
    const long long gw = (long long)blockIdx.x * (kRopeThreads / 32) + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    const int rows = a.n_heads + (APPEND ? 2 : 1) * a.n_kv_heads;
    const long long tok_ll = gw / rows;
    if (tok_ll >= a.n_tokens) return;
    const int tok = (int)tok_ll, row = (int)(gw - tok_ll * rows);
    int seq, pos, rpos;
    if (!row_place<APPEND>(P, tok, &seq, &pos, &rpos)) return;
    const int D = a.head_dim, half = a.rotary_dim / 2;
    const bool is_q = row < a.n_heads, is_v = row >= a.n_heads + a.n_kv_heads;
    const int head = is_q ? row : is_v ? row - a.n_heads - a.n_kv_heads : row - a.n_heads;
    const T *x = is_q ? (const T *)a.q + tok * a.q_stride
                      : is_v ? (const T *)a.v + tok * a.v_stride : (const T *)a.k + tok * a.k_stride;
    x += (long long)head * D;
    const float *w = is_q ? a.q_norm : is_v ? nullptr : a.k_norm;
    float v[8], o[8];
    float ss = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int e = lane + 32 * j;
        v[j] = e < D ? el_to_f<T>(x[e]) : 0.0f;
        ss = fmaf(v[j], v[j], ss);
    }
    float r = 1.0f;
    if (w) r = rsqrtf(fmaf(warp_sum(ss), 1.0f / (float)D, a.eps));
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int e = lane + 32 * j;
        o[j] = v[j];
        if (e >= D || is_v) continue;
        const float y = v[j] * (w ? w[e] : 1.0f);
        if (e < 2 * half) {
            const int i = e < half ? e : e - half, p = e < half ? e + half : e - half;
            double t = (double)rpos * (exp2(-(double)i * P.log2_step) * 0.15915494309189533577);
            t -= rint(t);
            float sn, cs;
            sincospif(2.0f * (float)t, &sn, &cs);
            const float yp = el_to_f<T>(x[p]) * (w ? w[p] : 1.0f);
            o[j] = r * fmaf(y, cs, yp * (e < half ? -sn : sn));
        } else {
            o[j] = r * y;
        }
    }
    __syncwarp();
    if (is_q || !APPEND) {
        T *y = is_q ? (T *)a.q_out + tok * a.q_out_stride : (T *)a.k_out + tok * a.k_out_stride;
        y += (long long)head * D;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (lane + 32 * j < D) y[lane + 32 * j] = el_from_f<T>(o[j]);
    } else if constexpr (APPEND) {
        if (pos < 0) return;
        int bad = 0;
        const long long at = P.kv.offset(P.b.table + (long long)seq * P.b.table_stride, pos, head, &bad);
        if (bad) {
            if (lane == 0) report(P.status, TQB200_PAGED_BAD_PAGE);
            return;
        }
        C *y = (C *)(is_v ? P.kv.v : P.kv.k) + at;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (lane + 32 * j < D) y[lane + 32 * j] = el_from_f<C>(o[j]);
    }
}

bool multiple(uintptr_t v, size_t n) { return v % n == 0; }

template <typename T, typename C, bool APPEND>
int launch_rope_t(RopeParams &P, cudaStream_t st) {
    const RopeArgs &a = P.a;
    constexpr int VEC = 16 / sizeof(T);
    P.log2_step = a.rotary_dim > 0 ? 2.0 * std::log2((double)a.theta) / a.rotary_dim : 0.0;
    P.ratio = std::exp2(-P.log2_step);
    int lanes = 1, bits = 0;
    while (lanes * VEC < a.head_dim) lanes *= 2, ++bits;
    bool vec = lanes <= 32 && a.head_dim % VEC == 0 && (a.rotary_dim / 2) % VEC == 0;
    vec = vec && multiple((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.q_out | (uintptr_t)a.k_out, 16);
    vec = vec && multiple((uintptr_t)(a.q_stride | a.k_stride | a.v_stride | a.q_out_stride | a.k_out_stride), VEC);
    if (APPEND)
        vec = vec && multiple((uintptr_t)P.kv.k | (uintptr_t)P.kv.v, 16) &&
              multiple((uintptr_t)(P.kv.page_stride | P.kv.head_stride | P.kv.slot_stride), VEC);
    constexpr int kWarps = kRopeThreads / 32;
    if (vec) {
        P.lane_bits = bits;
        const int rpi = 32 >> bits;
        const int n_it = (a.n_heads + rpi - 1) / rpi + (APPEND ? 2 : 1) * ((a.n_kv_heads + rpi - 1) / rpi);
        // warps per token: enough for 16 warps per SM, each with as many row groups as the others
        const int target = 16 * num_sms();
        int warps = std::min(n_it, (target + a.n_tokens - 1) / a.n_tokens);
        const int per = (n_it + warps - 1) / warps;
        P.warps = (n_it + per - 1) / per;
        const long long blocks = ((long long)a.n_tokens * P.warps + kWarps - 1) / kWarps;
        TQ_CHECK_ARG(blocks < (1LL << 31), "norm/rope: %d tokens", a.n_tokens);
        rope_vec_kernel<T, C, APPEND><<<(unsigned)blocks, kRopeThreads, 0, st>>>(P);
    } else {
        const int rows = a.n_heads + (APPEND ? 2 : 1) * a.n_kv_heads;
        const long long blocks = ((long long)a.n_tokens * rows + kWarps - 1) / kWarps;
        TQ_CHECK_ARG(blocks < (1LL << 31), "norm/rope: %d tokens of %d rows", a.n_tokens, rows);
        rope_any_kernel<T, C, APPEND><<<(unsigned)blocks, kRopeThreads, 0, st>>>(P);
    }
    TQ_CUDA_TRY(cudaGetLastError());
    return TQB200_OK;
}

}  // namespace

int launch_qk_norm_rope(const RopeArgs &a, cudaStream_t st) {
    if (a.n_tokens == 0 || a.n_heads + a.n_kv_heads == 0) return TQB200_OK;
    RopeParams P{};
    P.a = a;
    if (a.type == TQB200_EL_F32) return launch_rope_t<float, float, false>(P, st);
    if (a.type == TQB200_EL_F16) return launch_rope_t<__half, __half, false>(P, st);
    return launch_rope_t<__nv_bfloat16, __nv_bfloat16, false>(P, st);
}

int launch_paged_append(const RopeArgs &a, const PagedView &kv, int cache_type, const BatchView &b,
                        int *status, cudaStream_t st) {
    if (a.n_tokens == 0 || b.n_seqs == 0) return TQB200_OK;
    RopeParams P{};
    P.a = a;
    P.kv = kv;
    P.b = b;
    P.status = status;
    if (a.type == TQB200_EL_F32)
        return cache_type == TQB200_EL_F32 ? launch_rope_t<float, float, true>(P, st)
                                           : launch_rope_t<float, __half, true>(P, st);
    if (a.type == TQB200_EL_F16) return launch_rope_t<__half, __half, true>(P, st);
    return launch_rope_t<__nv_bfloat16, __nv_bfloat16, true>(P, st);
}

}  // namespace tqb200
