// paged_attention.cu — causal attention of new rows over a paged KV cache: the kernel for any
// shape, and the choice of kernel, sm_100a.
//
//   out[t, h] = sum_{x <= p} e^(scale q.K[x] - M) V[x] / sum_{x <= p} e^(scale q.K[x] - M),
// p the row's position, M any bound of the scores (the running maximum).
#include <algorithm>
#include <cfloat>

#include "paged.cuh"

namespace tqb200 {
namespace {

constexpr int kAnyThreads = 128;

// One warp per (row, head), head_dim at most 32 E; with a status word one more CTA checks the sequences.
template <typename T, typename C, int E>
__global__ void __launch_bounds__(kAnyThreads) paged_attn_any_kernel(const __grid_constant__ PagedAttnArgs A) {
    const long long gw = (long long)blockIdx.x * (kAnyThreads / 32) + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    const long long tok_ll = gw / A.n_heads;
    if (A.status && blockIdx.x == gridDim.x - 1) return check_seqs(A.b, A.status);
    if (tok_ll >= A.b.n_tokens) return;
    const int tok = (int)tok_ll, head = (int)(gw - tok_ll * A.n_heads);
    int s;
    const SeqInfo q = seq_of_row(A.b, tok, s);
    if (!q.ok) return;
    const int pos = q.len - q.n + (tok - q.q0);
    float m, l, o[E];
    row_pass<T, C, E>(A, (const T *)A.q + tok * A.q_stride + (long long)head * A.head_dim, s,
                      head / (A.n_heads / A.n_kv_heads), 0, pos + 1, m, l, o);
    T *out = (T *)A.out + tok * A.out_stride + (long long)head * A.head_dim;
    const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
#pragma unroll
    for (int j = 0; j < E; ++j)
        if (lane + 32 * j < A.head_dim) out[lane + 32 * j] = el_from_f<T>(o[j] * inv);
}

template <typename T, typename C>
int launch_any(const PagedAttnArgs &a, cudaStream_t st) {
    const long long blocks = ((long long)a.b.n_tokens * a.n_heads + kAnyThreads / 32 - 1) / (kAnyThreads / 32);
    TQ_CHECK_ARG(blocks < (1LL << 31) - 1, "paged_attention: %d tokens of %d heads", a.b.n_tokens, a.n_heads);
    const unsigned grid = (unsigned)blocks + (a.status ? 1 : 0);
    if (a.head_dim <= 128) paged_attn_any_kernel<T, C, 4><<<grid, kAnyThreads, 0, st>>>(a);
    else paged_attn_any_kernel<T, C, 8><<<grid, kAnyThreads, 0, st>>>(a);
    TQ_CUDA_TRY(cudaGetLastError());
    return TQB200_OK;
}

}  // namespace

void *driver_entry(const char *name) {
    void *fn = nullptr;
    cudaDriverEntryPointQueryResult q{};
    if (cudaGetDriverEntryPointByVersion(name, &fn, 12000, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess) {
        cudaGetLastError();
        return nullptr;
    }
    return fn;
}

// One size for chunks and single tokens, of any type: 59 MB for head_dim 128 on 148 SMs, most of it
// the tcgen05 kernel's, so that a workspace made for one batch serves them all.
size_t paged_attention_work_bytes(int head_dim) {
    return head_dim == 64 || head_dim == 128
               ? std::max(paged_decode_work_bytes(head_dim), paged_chunk_work_bytes(head_dim)) : 16;
}

int launch_paged_attention(const PagedAttnArgs &a, cudaStream_t st) {
    if (a.b.n_tokens == 0 || a.b.n_seqs == 0) return TQB200_OK;
    if (a.aligned && (a.head_dim == 64 || a.head_dim == 128)) {
        // The tcgen05 kernel needs a 16-bit cache and pays from some work on: its items cost
        // about 10 us before their first result.  Work is rows x positions x head_dim, the
        // positions bounded by the page table (the lengths are known on the device only):
        // 14 heads x 64 tokens over 564 positions (32 M) 14.6 us by mma.sync, 17.1 by tcgen05; 32
        // heads of 128, 64 tokens over 164 (43 M) 10.7 and 13.2, 128 over 128 (67 M) 10.0 and
        // 10.6, 48 over 448 (88 M) 20.9 and 16.5, 64 over 564 (148 M) 24.0 and 19.0, all with a page
        // table as wide as the longest sequence.  With a wider one the small ones go to tcgen05 too: a table of
        // 32768 positions costs the first 18.8 us against 15.9, the second 13.2 against 10.9.
        // Up to 16 rows of queries per KV head mma.sync reads no key twice.
        const long long rows = (long long)a.b.max_q_len * (a.n_heads / a.n_kv_heads);
        const double work = (double)a.b.n_tokens * a.n_heads * a.b.max_len * a.head_dim;
        if (a.cache_type != TQB200_EL_F32 && rows > kDecodeRows && work > 60e6) return launch_paged_chunk(a, st);
        return launch_paged_decode(a, st);
    }
    if (a.type == TQB200_EL_F32)
        return a.cache_type == TQB200_EL_F32 ? launch_any<float, float>(a, st) : launch_any<float, __half>(a, st);
    if (a.type == TQB200_EL_F16) return launch_any<__half, __half>(a, st);
    return launch_any<__nv_bfloat16, __nv_bfloat16>(a, st);
}

}  // namespace tqb200
