// paged_capi.cu — the extern "C" entry points of the paged-cache operators (declared in
// include/tqb200.h): argument checks on the host, then the launchers.
#include <cuda.h>

#include <algorithm>
#include <cmath>

#include "paged.cuh"

using namespace tqb200;

namespace {

#define TQ_TRY(expr)       \
    do {                   \
        int s_ = (expr);   \
        if (s_) return s_; \
    } while (0)

constexpr int kMaxHeads = 4096;

size_t el_size(int type) { return type == TQB200_EL_F32 ? 4 : 2; }
bool el_known(int type) { return type == TQB200_EL_F32 || type == TQB200_EL_F16 || type == TQB200_EL_BF16; }

// p: `align`-aligned memory that the current device reads (its own, managed or pinned host
// memory).  A host pointer or another device's would fault inside a kernel.
int check_ptr(const char *op, const char *name, const void *p, size_t align) {
    TQ_CHECK_ARG(p, "%s: %s is null", op, name);
    TQ_CHECK_ARG(((uintptr_t)p) % align == 0, "%s: %s is not %zu-byte aligned", op, name, align);
    return TQB200_OK;
}
// By the driver's attribute query: 50 ns a pointer against 90 for the runtime's.
int check_place(const char *op, const char *name, const void *p, int dev) {
    using Query = CUresult (*)(unsigned, CUpointer_attribute *, void **, CUdeviceptr);
    static const Query query = reinterpret_cast<Query>(driver_entry("cuPointerGetAttributes"));
    if (!query) return set_error(TQB200_ERR_NO_DEVICE, "%s: no CUDA driver", op);
    unsigned type = 0;
    int ordinal = 0;
    CUpointer_attribute what[2] = {CU_POINTER_ATTRIBUTE_MEMORY_TYPE, CU_POINTER_ATTRIBUTE_DEVICE_ORDINAL};
    void *where[2] = {&type, &ordinal};
    const CUresult r = query(2, what, where, (CUdeviceptr)p);
    TQ_CHECK_ARG(r == CUDA_SUCCESS && type != 0, "%s: %s is not device memory", op, name);
    TQ_CHECK_ARG(type != CU_MEMORYTYPE_DEVICE || ordinal == dev, "%s: %s is on device %d, the current device is %d", op, name,
                 ordinal, dev);
    return TQB200_OK;
}
int current_device(int *dev) {
    if (cudaGetDevice(dev) != cudaSuccess) {
        cudaGetLastError();
        return set_error(TQB200_ERR_NO_DEVICE, "no CUDA device visible");
    }
    return TQB200_OK;
}

int check_heads(const char *op, int n_heads, int n_kv_heads, int head_dim) {
    TQ_CHECK_ARG(n_heads >= 0 && n_heads <= kMaxHeads && n_kv_heads >= 0 && n_kv_heads <= kMaxHeads,
                 "%s: %d query and %d KV heads (0..%d)", op, n_heads, n_kv_heads, kMaxHeads);
    TQ_CHECK_ARG(head_dim >= 8 && head_dim <= 256 && head_dim % 8 == 0,
                 "%s: head_dim %d (a multiple of 8 up to 256)", op, head_dim);
    return TQB200_OK;
}

// Rows of `n` tokens, `width` elements each, `stride` apart; `distinct`: written, so not on
// one another.
int check_rows(const char *op, const char *name, const void *p, int n, long long stride, long long width,
               int type, bool distinct) {
    TQ_TRY(check_ptr(op, name, p, el_size(type)));
    TQ_CHECK_ARG(stride >= (distinct && n > 1 ? width : 0) && stride <= (1LL << 40),
                 "%s: %s row stride %lld (rows of %lld)", op, name, stride, width);
    return TQB200_OK;
}

int check_rotary(const char *op, int head_dim, int rotary_dim, float eps, float theta) {
    TQ_CHECK_ARG(rotary_dim >= 0 && rotary_dim <= head_dim && rotary_dim % 2 == 0,
                 "%s: rotary_dim %d (even, 0..head_dim %d)", op, rotary_dim, head_dim);
    TQ_CHECK_ARG(rotary_dim == 0 || (std::isfinite(theta) && theta > 0.0f), "%s: theta %g", op, theta);
    TQ_CHECK_ARG(std::isfinite(eps) && eps >= 0.0f, "%s: eps %g", op, eps);
    return TQB200_OK;
}

int check_types(const char *op, int type, int cache) {
    TQ_CHECK_ARG(el_known(type), "%s: unknown element type %d", op, type);
    TQ_CHECK_ARG(el_known(cache), "%s: unknown cache type %d", op, cache);
    TQ_CHECK_ARG(type == cache || (type == TQB200_EL_F32 && cache == TQB200_EL_F16),
                 "%s: activations of type %d over a cache of type %d", op, type, cache);
    return TQB200_OK;
}

int check_cache(const char *op, const tqb200_paged_cache *c) {
    TQ_CHECK_ARG(c, "%s: cache is null", op);
    TQ_CHECK_ARG(el_known(c->type), "%s: unknown cache type %d", op, c->type);
    TQ_TRY(check_ptr(op, "cache k", c->k, el_size(c->type)));
    TQ_TRY(check_ptr(op, "cache v", c->v, el_size(c->type)));
    TQ_CHECK_ARG(c->n_pages >= 1 && c->page_size >= 1, "%s: %d pages of %d slots", op, c->n_pages, c->page_size);
    TQ_CHECK_ARG(c->n_kv_heads >= 1, "%s: %d KV heads", op, c->n_kv_heads);
    TQ_TRY(check_heads(op, 0, c->n_kv_heads, c->head_dim));
    // rows of head_dim elements, no two on one another: from the smallest stride up, each
    // covers what lies inside it
    struct {
        long long stride, count;
    } dim[3] = {{c->slot_stride, c->page_size}, {c->head_stride, c->n_kv_heads}, {c->page_stride, c->n_pages}};
    std::sort(dim, dim + 3, [](const auto &a, const auto &b) { return a.stride < b.stride; });
    long long covered = c->head_dim;
    for (const auto &d : dim) {
        TQ_CHECK_ARG(d.stride >= 0 && d.stride <= (1LL << 46) / d.count, "%s: cache stride %lld", op, d.stride);
        if (d.count == 1) continue;
        TQ_CHECK_ARG(d.stride >= covered, "%s: cache stride %lld inside %lld elements", op, d.stride, covered);
        covered += (d.count - 1) * d.stride;
    }
    return TQB200_OK;
}

int check_batch(const char *op, const tqb200_paged_batch *b) {
    TQ_CHECK_ARG(b, "%s: batch is null", op);
    TQ_CHECK_ARG(b->n_seqs >= 0 && b->n_tokens >= 0 && b->max_q_len >= 0 && b->table_stride >= 0,
                 "%s: %d sequences, %d rows, at most %d each, %d pages each", op, b->n_seqs, b->n_tokens,
                 b->max_q_len, b->table_stride);
    TQ_CHECK_ARG(b->n_seqs <= (1 << 24), "%s: %d sequences", op, b->n_seqs);
    if (b->n_seqs == 0) return TQB200_OK;
    TQ_TRY(check_ptr(op, "q_start", b->q_start, 4));
    TQ_TRY(check_ptr(op, "kv_len", b->kv_len, 4));
    TQ_TRY(check_ptr(op, "page_table", b->page_table, 4));
    return TQB200_OK;
}

PagedView view_of(const tqb200_paged_cache *c) {
    PagedView v{};
    v.k = (char *)c->k;
    v.v = (char *)c->v;
    v.page_stride = c->page_stride;
    v.head_stride = c->head_stride;
    v.slot_stride = c->slot_stride;
    v.n_pages = c->n_pages;
    v.page = FastDiv::of((uint32_t)c->page_size);
    return v;
}
BatchView view_of(const tqb200_paged_batch *b, int page_size) {
    BatchView v{b->q_start, b->kv_len, b->page_table, b->n_seqs, b->table_stride, b->n_tokens, b->max_q_len, 0};
    const long long most = (long long)b->table_stride * page_size;
    v.max_len = (int)(most < 0x7fff0000LL ? most : 0x7fff0000LL);
    return v;
}

}  // namespace

extern "C" {

int tqb200_dev_qk_norm_rope(const void *q, const void *k, void *q_out, void *k_out, int type,
                            int n_tokens, int n_heads, int n_kv_heads, int head_dim,
                            int rotary_dim, long long q_stride, long long k_stride,
                            long long q_out_stride, long long k_out_stride, const float *q_norm,
                            const float *k_norm, float eps, float theta, const int *positions,
                            void *stream) {
    const char *op = "qk_norm_rope";
    TQ_CHECK_ARG(el_known(type), "%s: unknown element type %d", op, type);
    TQ_TRY(check_heads(op, n_heads, n_kv_heads, head_dim));
    TQ_TRY(check_rotary(op, head_dim, rotary_dim, eps, theta));
    TQ_CHECK_ARG(n_tokens >= 0, "%s: %d tokens", op, n_tokens);
    if (n_tokens == 0 || n_heads + n_kv_heads == 0) return TQB200_OK;
    struct {
        const char *name, *out_name;
        const void *in;
        void *out;
        int heads;
        long long stride, out_stride;
        const float *norm;
    } sides[2] = {{"q", "q_out", q, q_out, n_heads, q_stride, q_out_stride, q_norm},
                  {"k", "k_out", k, k_out, n_kv_heads, k_stride, k_out_stride, k_norm}};
    for (const auto &s : sides) {
        if (s.heads == 0) continue;
        const long long width = (long long)s.heads * head_dim;
        TQ_TRY(check_rows(op, s.name, s.in, n_tokens, s.stride, width, type, false));
        TQ_TRY(check_rows(op, s.out_name, s.out, n_tokens, s.out_stride, width, type, true));
        TQ_CHECK_ARG(s.in != s.out || n_tokens == 1 || s.stride == s.out_stride,
                     "%s: %s in place with another row stride", op, s.name);
        TQ_CHECK_ARG(((uintptr_t)s.norm) % 4 == 0, "%s: %s norm weights not 4-byte aligned", op, s.name);
    }
    TQ_CHECK_ARG(rotary_dim == 0 || positions, "%s: positions is null", op);
    TQ_CHECK_ARG(((uintptr_t)positions) % 4 == 0, "%s: positions not 4-byte aligned", op);
    int dev = 0;
    TQ_TRY(current_device(&dev));
    for (const auto &s : sides) {
        if (s.heads == 0) continue;
        TQ_TRY(check_place(op, s.name, s.in, dev));
        TQ_TRY(check_place(op, s.out_name, s.out, dev));
        if (s.norm) TQ_TRY(check_place(op, "norm weights", s.norm, dev));
    }
    if (positions) TQ_TRY(check_place(op, "positions", positions, dev));
    RopeArgs a{};
    a.type = type;
    a.n_tokens = n_tokens;
    a.n_heads = n_heads;
    a.n_kv_heads = n_kv_heads;
    a.head_dim = head_dim;
    a.rotary_dim = rotary_dim;
    if (n_heads) a.q = q, a.q_out = q_out, a.q_stride = q_stride, a.q_out_stride = q_out_stride, a.q_norm = q_norm;
    if (n_kv_heads) a.k = k, a.k_out = k_out, a.k_stride = k_stride, a.k_out_stride = k_out_stride, a.k_norm = k_norm;
    a.eps = eps;
    a.theta = theta;
    a.positions = positions;
    return launch_qk_norm_rope(a, (cudaStream_t)stream);
}

int tqb200_dev_paged_append(const void *q, const void *k, const void *v, void *q_out, int type,
                            int n_heads, int rotary_dim, long long q_stride, long long k_stride,
                            long long v_stride, long long q_out_stride, const float *q_norm,
                            const float *k_norm, float eps, float theta, const int *positions,
                            const tqb200_paged_cache *cache, const tqb200_paged_batch *batch,
                            int *status, void *stream) {
    const char *op = "paged_append";
    TQ_TRY(check_cache(op, cache));
    TQ_TRY(check_batch(op, batch));
    TQ_TRY(check_types(op, type, cache->type));
    const int D = cache->head_dim, n = batch->n_tokens;
    TQ_TRY(check_heads(op, n_heads, cache->n_kv_heads, D));
    TQ_TRY(check_rotary(op, D, rotary_dim, eps, theta));
    if (n == 0 || batch->n_seqs == 0) return TQB200_OK;
    const long long q_width = (long long)n_heads * D, k_width = (long long)cache->n_kv_heads * D;
    if (n_heads) {
        TQ_TRY(check_rows(op, "q", q, n, q_stride, q_width, type, false));
        TQ_TRY(check_rows(op, "q_out", q_out, n, q_out_stride, q_width, type, true));
        TQ_CHECK_ARG(q != q_out || n == 1 || q_stride == q_out_stride, "%s: q in place with another row stride", op);
        TQ_CHECK_ARG(((uintptr_t)q_norm) % 4 == 0, "%s: q norm weights not 4-byte aligned", op);
    }
    TQ_TRY(check_rows(op, "k", k, n, k_stride, k_width, type, false));
    TQ_TRY(check_rows(op, "v", v, n, v_stride, k_width, type, false));
    TQ_CHECK_ARG(((uintptr_t)k_norm) % 4 == 0, "%s: k norm weights not 4-byte aligned", op);
    TQ_CHECK_ARG(((uintptr_t)positions | (uintptr_t)status) % 4 == 0,
                 "%s: positions or status not 4-byte aligned", op);
    int dev = 0;
    TQ_TRY(current_device(&dev));
    if (n_heads) {
        TQ_TRY(check_place(op, "q", q, dev));
        TQ_TRY(check_place(op, "q_out", q_out, dev));
        if (q_norm) TQ_TRY(check_place(op, "q norm weights", q_norm, dev));
    }
    if (k_norm) TQ_TRY(check_place(op, "k norm weights", k_norm, dev));
    if (positions) TQ_TRY(check_place(op, "positions", positions, dev));
    if (status) TQ_TRY(check_place(op, "status", status, dev));
    TQ_TRY(check_place(op, "k", k, dev));
    TQ_TRY(check_place(op, "v", v, dev));
    TQ_TRY(check_place(op, "cache k", cache->k, dev));
    TQ_TRY(check_place(op, "cache v", cache->v, dev));
    TQ_TRY(check_place(op, "q_start", batch->q_start, dev));
    TQ_TRY(check_place(op, "kv_len", batch->kv_len, dev));
    TQ_TRY(check_place(op, "page_table", batch->page_table, dev));
    RopeArgs a{};
    a.type = type;
    a.n_tokens = n;
    a.n_heads = n_heads;
    a.n_kv_heads = cache->n_kv_heads;
    a.head_dim = D;
    a.rotary_dim = rotary_dim;
    if (n_heads) a.q = q, a.q_out = q_out, a.q_stride = q_stride, a.q_out_stride = q_out_stride, a.q_norm = q_norm;
    a.k = k, a.v = v, a.k_stride = k_stride, a.v_stride = v_stride, a.k_norm = k_norm;
    a.eps = eps;
    a.theta = theta;
    a.positions = positions;
    return launch_paged_append(a, view_of(cache), cache->type, view_of(batch, cache->page_size), status,
                               (cudaStream_t)stream);
}

size_t tqb200_paged_attention_workspace_bytes(const tqb200_paged_cache *cache,
                                              const tqb200_paged_batch *batch, int n_heads) {
    const char *op = "paged_attention";
    if (!cache || !batch || cache->n_kv_heads < 1 || n_heads < 1 || n_heads % cache->n_kv_heads != 0 ||
        check_heads(op, n_heads, cache->n_kv_heads, cache->head_dim) || batch->n_seqs < 0 ||
        batch->n_seqs > (1 << 24) || batch->n_tokens < 0 || batch->max_q_len < 0)
        return 0;
    return paged_attention_work_bytes(cache->head_dim);
}

int tqb200_dev_paged_attention(const void *q, void *out, int type, int n_heads, long long q_stride,
                               long long out_stride, float scale, const tqb200_paged_cache *cache,
                               const tqb200_paged_batch *batch, void *workspace,
                               size_t workspace_bytes, int *status, void *stream) {
    const char *op = "paged_attention";
    TQ_TRY(check_cache(op, cache));
    TQ_TRY(check_batch(op, batch));
    TQ_TRY(check_types(op, type, cache->type));
    const int D = cache->head_dim, n = batch->n_tokens;
    TQ_TRY(check_heads(op, n_heads, cache->n_kv_heads, D));
    TQ_CHECK_ARG(n_heads >= 1 && n_heads % cache->n_kv_heads == 0,
                 "%s: %d query heads over %d KV heads", op, n_heads, cache->n_kv_heads);
    TQ_CHECK_ARG(std::isfinite(scale) && scale > 0.0f, "%s: scale %g (positive)", op, scale);
    if (n == 0 || batch->n_seqs == 0) return TQB200_OK;
    const long long width = (long long)n_heads * D;
    TQ_TRY(check_rows(op, "q", q, n, q_stride, width, type, false));
    TQ_TRY(check_rows(op, "out", out, n, out_stride, width, type, true));
    TQ_CHECK_ARG(q != out, "%s: out is q", op);
    TQ_TRY(check_ptr(op, "workspace", workspace, 16));
    const size_t need = tqb200_paged_attention_workspace_bytes(cache, batch, n_heads);
    TQ_CHECK_ARG(workspace_bytes >= need, "%s: workspace of %zu bytes, %zu needed", op, workspace_bytes, need);
    TQ_CHECK_ARG(((uintptr_t)status) % 4 == 0, "%s: status not 4-byte aligned", op);
    int dev = 0;
    TQ_TRY(current_device(&dev));
    if (status) TQ_TRY(check_place(op, "status", status, dev));
    TQ_TRY(check_place(op, "q", q, dev));
    TQ_TRY(check_place(op, "out", out, dev));
    TQ_TRY(check_place(op, "workspace", workspace, dev));
    TQ_TRY(check_place(op, "cache k", cache->k, dev));
    TQ_TRY(check_place(op, "cache v", cache->v, dev));
    TQ_TRY(check_place(op, "q_start", batch->q_start, dev));
    TQ_TRY(check_place(op, "kv_len", batch->kv_len, dev));
    TQ_TRY(check_place(op, "page_table", batch->page_table, dev));
    PagedAttnArgs a{};
    a.q = q;
    a.out = out;
    a.type = type;
    a.n_heads = n_heads;
    a.n_kv_heads = cache->n_kv_heads;
    a.head_dim = D;
    a.cache_type = cache->type;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.scale = scale;
    a.kv = view_of(cache);
    a.b = view_of(batch, cache->page_size);
    const uintptr_t e = el_size(type), c = el_size(cache->type);
    a.aligned = (((uintptr_t)q | (uintptr_t)out | (uintptr_t)q_stride * e | (uintptr_t)out_stride * e |
                  (uintptr_t)cache->k | (uintptr_t)cache->v | (uintptr_t)cache->page_stride * c |
                  (uintptr_t)cache->head_stride * c | (uintptr_t)cache->slot_stride * c) &
                 15) == 0;
    a.work = workspace;
    a.status = status;
    return launch_paged_attention(a, (cudaStream_t)stream);
}

}  // extern "C"
