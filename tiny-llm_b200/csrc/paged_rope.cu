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
// is rounded to fp32), so far positions keep their phase; a lane forms one or two of the angles
// that it shares with the other lanes of its pair index and its frequencies stay in registers
// over all the warp's tokens.  Few tokens are cut into parts (heads dealt out to warps).
//
// Measured on one B200 (device time): 8192 rows of 32 + 8 + 8 heads of 128 into bf16 pages (201 MB)
// 46.6 us, 4.3 TB/s; 8191 fp16 rows of 32 + 8 heads, a quarter rotated (168 MB) 38.6 us; one row 3.1
// us.  It issues 2600 warp instructions a token of 48 heads (4900 while one loop served all
// kinds of rows) and waits on memory half the time: 4 CTAs per SM take 54 us; 6 spill registers,
// 57.  A ring of cp.async groups in shared memory instead of register loads gave 45.5 us but
// 15% more for few rows, and was left out.
#include <algorithm>
#include <cmath>

#include "paged.cuh"

namespace tqb200 {
namespace {

constexpr int kRopeThreads = 128;
constexpr int kRopeUnroll = 4;  // row groups whose loads are in flight together
constexpr int kRopePerSm = 5;   // CTAs per SM

struct RopeParams {
    RopeArgs a;
    PagedView kv;
    BatchView b;
    int *status;
    int lane_bits;           // log2 of the lanes of a row
    int warps;               // parts that a token is cut into, a warp each
    int blocks;              // CTAs that take tokens; append with a status word: one more checks the sequences
    double log2_step;        // log2(theta) / h: frequency i is 2^(-i log2_step)
    double ratio;            // 2^-log2_step
};

// The token's place in its sequence; live == false: its rows are left as they are.  A sequence
// once found serves the following tokens without a search.
struct Place {
    SeqInfo q{0, 0, 0, 0};
    int seq = 0, cache_pos = 0, rope_pos = 0;
    bool live = false;
    template <bool APPEND>
    __device__ __forceinline__ void find(const RopeParams &P, int tok) {
        live = true;
        cache_pos = 0;
        if constexpr (APPEND) {
            if (!q.ok || tok < q.q0 || tok >= q.q0 + q.n) {
                q = seq_of_row(P.b, tok, seq);
                live = q.ok;
            }
            cache_pos = q.len - q.n + (tok - q.q0);
        }
        rope_pos = P.a.positions && live ? P.a.positions[tok] : cache_pos;
    }
};

// LB: log2 of the lanes of a row, -1 where it is known at run time only.
template <typename T, typename C, bool APPEND, int LB>
__global__ void __launch_bounds__(kRopeThreads, kRopePerSm) rope_vec_kernel(const __grid_constant__ RopeParams P) {
    constexpr int VEC = 16 / sizeof(T), H = VEC / 2;
    constexpr int U = kRopeUnroll;
    const RopeArgs &a = P.a;
    const long long gw = (long long)blockIdx.x * (kRopeThreads / 32) + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    // warp gw: part `part` of tokens tok, tok + step, ... (step: whole tokens at a time)
    const int part = (int)(gw % P.warps);
    const long long step = (long long)P.blocks * (kRopeThreads / 32) / P.warps;
    long long tok = gw / P.warps;
    if constexpr (APPEND)
        if (blockIdx.x == (unsigned)P.blocks) return check_seqs(P.b, P.status);
    if (tok >= step || tok >= a.n_tokens) return;  // warp-uniform; no CTA barrier below

    const int bits = LB >= 0 ? LB : P.lane_bits;
    const int lpr = 1 << bits, rpi = 32 >> bits;
    const int sub = lane >> bits, c = lane & (lpr - 1);
    const bool in_row = c * VEC < a.head_dim;
    const int hc = a.rotary_dim / 2 / VEC;  // lanes of one rotated half
    const bool rot = c < 2 * hc, low = c < hc;
    const int partner = lane + (rot ? (low ? hc : -hc) : 0);
    // Row groups: n_q of queries, n_k of keys, then (append) n_k of values; group i of them all
    // belongs to part i % warps.  first_*: this part's first of each kind; lim_*: how many
    // groups hold a row for this lane.
    const int n_q = (a.n_heads + rpi - 1) / rpi, n_k = (a.n_kv_heads + rpi - 1) / rpi;
    const int first_q = part, first_k = (part + P.warps - n_q % P.warps) % P.warps;
    const int first_v = (part + P.warps - (n_q + n_k) % P.warps) % P.warps;
    const int lim_q = in_row ? (a.n_heads - sub + rpi - 1) / rpi : 0, lim_k = in_row ? (a.n_kv_heads - sub + rpi - 1) / rpi : 0;
    const int mine = sub * a.head_dim + c * VEC;        // the lane's elements in a group of rows
    const long long apart = (long long)P.warps * rpi * a.head_dim;  // from one of this part's groups to the next
    const T *const q0 = (const T *)a.q + mine + (long long)first_q * rpi * a.head_dim;
    const T *const k0 = (const T *)a.k + mine + (long long)first_k * rpi * a.head_dim;
    const T *const v0 = (const T *)a.v + mine + (long long)first_v * rpi * a.head_dim;
    T *const qo0 = (T *)a.q_out + mine + (long long)first_q * rpi * a.head_dim;
    T *const ko0 = (T *)a.k_out + mine + (long long)first_k * rpi * a.head_dim;

    // The lanes of one pair index (two halves of rpi rows) share its VEC angles: lane (sub, half)
    // forms `share` of them, from number slot * share on; their frequencies stay over the tokens.
    const int pc = c + (rot ? (low ? hc : -hc) : 0);  // the partner's lane in the row
    const int share = VEC / min(VEC, 2 * rpi);        // angles per lane
    const int slot = share > 2 ? 0 : (sub * 2 + (low ? 0 : 1)) % (VEC / share);
    double freq[2];                                   // turns per position
    {
        const double i0 = (low ? c : c - hc) * VEC + slot * share;
        freq[0] = rot ? exp2(-i0 * P.log2_step) * 0.15915494309189533577 : 0.0;
        freq[1] = freq[0] * P.ratio;
    }

    const float inv_n = 1.0f / (float)a.head_dim;
    auto turn = [&](const ElVec<T, VEC> &x, const uint64_t (&f)[2][H], bool norm, uint64_t (&y)[H]) {
        uint64_t r = pair(1.0f, 1.0f);
        uint64_t x2[H];
#pragma unroll
        for (int j = 0; j < H; ++j) x2[j] = x.get2(j);
        if (norm) {
            uint64_t ss2 = mul2(x2[0], x2[0]);
#pragma unroll
            for (int j = 1; j < H; ++j) ss2 = fma2(x2[j], x2[j], ss2);
            float ss, sb;
            unpair(ss2, ss, sb);
            ss += sb;
#pragma unroll
            for (int o = lpr >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            ss = rsqrtf(fmaf(ss, inv_n, a.eps));
            r = pair(ss, ss);
        }
        ElVec<T, VEC> xp;
        // lanes without a rotation take no partner: 0 * its infinity would be NaN
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            xp.w[w] = __shfl_sync(0xffffffffu, x.w[w], partner);
            if (!rot) xp.w[w] = 0u;
        }
#pragma unroll
        for (int j = 0; j < H; ++j) y[j] = mul2(r, fma2(xp.get2(j), f[1][j], mul2(x2[j], f[0][j])));
    };

    Place place;
    for (; tok < a.n_tokens; tok += step) {
        place.find<APPEND>(P, (int)tok);
        // where this token's keys and values go
        long long at = -1;
        if constexpr (APPEND) {
            if (place.live && place.cache_pos >= 0) {
                int bad = 0;
                at = P.kv.offset(P.b.table + (long long)place.seq * P.b.table_stride, place.cache_pos, 0, &bad);
                if (bad && lane == 0) report(P.status, TQB200_PAGED_BAD_PAGE);
            }
        }
        // its angles, and the factors of x and of the partner's x
        uint64_t fq[2][H], fk[2][H];
        {
            float cv[2], sv[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                double t = (double)place.rope_pos * freq[e];
                t -= rint(t);
                sincospif(2.0f * (float)t, &sv[e], &cv[e]);
            }
            float cs[VEC], sn[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                // angle j of this lane's pair indexes: formed by the lane of slot j / share among
                // those that share them
                if (share > 2) {
                    // few lanes share (wide rows): each forms its own, one by one
                    double f = freq[0];
                    for (int k = 0; k < j; ++k) f *= P.ratio;
                    double t = (double)place.rope_pos * f;
                    t -= rint(t);
                    sincospif(2.0f * (float)t, &sn[j], &cs[j]);
                } else {
                    const int from = j / share, s_ = from >> 1, h_ = from & 1;
                    const int src = rot ? (s_ << bits) + (low ? c : c - hc) + (h_ ? hc : 0) : lane;
                    cs[j] = __shfl_sync(0xffffffffu, cv[0], src);
                    sn[j] = __shfl_sync(0xffffffffu, sv[0], src);
                    if (share == 2) {
                        const float c1 = __shfl_sync(0xffffffffu, cv[1], src), s1 = __shfl_sync(0xffffffffu, sv[1], src);
                        if (j & 1) cs[j] = c1, sn[j] = s1;
                    }
                }
                if (!rot) cs[j] = 1.0f, sn[j] = 0.0f;
                else if (low) sn[j] = -sn[j];
            }
            auto factors = [&](const float *w, uint64_t (&f)[2][H]) {
                const bool has = w && in_row;
#pragma unroll
                for (int j = 0; j < H; ++j) {
                    const float2 own = has ? *reinterpret_cast<const float2 *>(w + c * VEC + 2 * j) : make_float2(1.0f, 1.0f);
                    const float2 his = has ? *reinterpret_cast<const float2 *>(w + pc * VEC + 2 * j) : make_float2(1.0f, 1.0f);
                    f[0][j] = pair(own.x * cs[2 * j], own.y * cs[2 * j + 1]);
                    f[1][j] = pair(his.x * sn[2 * j], his.y * sn[2 * j + 1]);
                }
            };
            factors(a.q_norm, fq);
            factors(a.k_norm, fk);
        }
        // One kind of rows: U groups' loads at a time, then what is done with each.
        auto rows = [&](const T *src, int it, int groups, int lim, auto &&use) {
            for (; it < groups; it += U * P.warps) {
                ElVec<T, VEC> raw[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
#pragma unroll
                    for (int w = 0; w < 4; ++w) raw[u].w[w] = 0u;
                    if (it + u * P.warps < lim) raw[u].load(src);
                    src += apart;
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (it + u * P.warps >= groups) break;  // warp-uniform
                    use(raw[u], it + u * P.warps < lim);
                }
            }
        };
        if (!place.live) continue;
        {
            T *to = qo0 + tok * a.q_out_stride;
            rows(q0 + tok * a.q_stride, first_q, n_q, lim_q, [&](const ElVec<T, VEC> &x, bool has) {
                uint64_t y[H];
                turn(x, fq, a.q_norm != nullptr, y);
                if (has) {
                    ElVec<T, VEC> o;
#pragma unroll
                    for (int j = 0; j < H; ++j) o.set2(j, y[j]);
                    o.store(to);
                }
                to += apart;
            });
        }
        if constexpr (!APPEND) {
            T *to = ko0 + tok * a.k_out_stride;
            rows(k0 + tok * a.k_stride, first_k, n_k, lim_k, [&](const ElVec<T, VEC> &x, bool has) {
                uint64_t y[H];
                turn(x, fk, a.k_norm != nullptr, y);
                if (has) {
                    ElVec<T, VEC> o;
#pragma unroll
                    for (int j = 0; j < H; ++j) o.set2(j, y[j]);
                    o.store(to);
                }
                to += apart;
            });
        } else if (at >= 0) {
            const long long heads_apart = (long long)P.warps * rpi * P.kv.head_stride;
            C *to = (C *)P.kv.k + at + (first_k * rpi + sub) * P.kv.head_stride + c * VEC;
            rows(k0 + tok * a.k_stride, first_k, n_k, lim_k, [&](const ElVec<T, VEC> &x, bool has) {
                uint64_t y[H];
                turn(x, fk, a.k_norm != nullptr, y);
                if (has) {
                    ElVec<C, VEC> o;
#pragma unroll
                    for (int j = 0; j < H; ++j) o.set2(j, y[j]);
                    o.store(to);
                }
                to += heads_apart;
            });
            to = (C *)P.kv.v + at + (first_v * rpi + sub) * P.kv.head_stride + c * VEC;
            rows(v0 + tok * a.v_stride, first_v, n_k, lim_k, [&](const ElVec<T, VEC> &x, bool has) {
                if (has) {
                    ElVec<C, VEC> o;
#pragma unroll
                    for (int j = 0; j < H; ++j) o.set2(j, x.get2(j));
                    o.store(to);
                }
                to += heads_apart;
            });
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
    if constexpr (APPEND)
        if (blockIdx.x == (unsigned)P.blocks) return check_seqs(P.b, P.status);
    if (tok_ll >= a.n_tokens) return;
    const int tok = (int)tok_ll, row = (int)(gw - tok_ll * rows);
    Place place;
    place.find<APPEND>(P, tok);
    if (!place.live) return;
    const int pos = place.cache_pos, rpos = place.rope_pos, seq = place.seq;
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
    vec = vec && multiple((uintptr_t)a.q_norm | (uintptr_t)a.k_norm, 8);
    vec = vec && multiple((uintptr_t)(a.q_stride | a.k_stride | a.v_stride | a.q_out_stride | a.k_out_stride), VEC);
    if (APPEND)
        vec = vec && multiple((uintptr_t)P.kv.k | (uintptr_t)P.kv.v, 16) &&
              multiple((uintptr_t)(P.kv.page_stride | P.kv.head_stride | P.kv.slot_stride), VEC);
    constexpr int kWarps = kRopeThreads / 32;
    const int check = APPEND && P.status ? 1 : 0;
    if (vec) {
        P.lane_bits = bits;
        const int rpi = 32 >> bits;
        const int n_it = (a.n_heads + rpi - 1) / rpi + (APPEND ? 2 : 1) * ((a.n_kv_heads + rpi - 1) / rpi);
        // The resident warps stay and take further tokens.  A token is cut into `parts` (its row
        // groups dealt out) so that few tokens still reach every warp, and so that the last
        // round is full: the cost of parts p is the rounds times a part's groups and its
        // set-up, worth about 3 of them.
        const long long resident = ((long long)kRopePerSm * num_sms() - check) * kWarps;
        int parts = 1;
        double best = 0.0;
        for (int p = 1; p <= std::min(n_it, 64); ++p) {
            const double rounds = std::ceil((double)a.n_tokens * p / (double)(resident / p * p));
            const double cost = rounds * ((n_it + p - 1) / p + 3);
            if (p == 1 || cost < best) best = cost, parts = p;
            if (p >= 4 && (long long)a.n_tokens * p >= resident) break;
        }
        P.warps = parts;
        P.blocks = (int)std::min(((long long)a.n_tokens * parts + kWarps - 1) / kWarps, resident / kWarps);
        const unsigned grid = P.blocks + check;
        if (bits == 3) rope_vec_kernel<T, C, APPEND, 3><<<grid, kRopeThreads, 0, st>>>(P);
        else if (bits == 4) rope_vec_kernel<T, C, APPEND, 4><<<grid, kRopeThreads, 0, st>>>(P);
        else if (bits == 5) rope_vec_kernel<T, C, APPEND, 5><<<grid, kRopeThreads, 0, st>>>(P);
        else rope_vec_kernel<T, C, APPEND, -1><<<grid, kRopeThreads, 0, st>>>(P);
    } else {
        const int rows = a.n_heads + (APPEND ? 2 : 1) * a.n_kv_heads;
        const long long blocks = ((long long)a.n_tokens * rows + kWarps - 1) / kWarps;
        TQ_CHECK_ARG(blocks < (1LL << 31) - 1, "norm/rope: %d tokens of %d rows", a.n_tokens, rows);
        P.blocks = (int)blocks;
        rope_any_kernel<T, C, APPEND><<<(unsigned)blocks + check, kRopeThreads, 0, st>>>(P);
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
