// extern "C" entry points of the operators over a paged cache in 16, 8 or 4 bits (declared
// in include/mlxq_b200.h): host-side validation, then the launches.
#include <cmath>
#include <cstdio>

#include "../../include/mlxq_b200.h"
#include "paged_ops.h"

namespace {

int fail(int code, const char* what, const char* msg) {
    char buf[256];
    snprintf(buf, sizeof(buf), "%s: %s", what, msg);
    return mlxq::set_last_error(code, buf);
}

int done(cudaError_t e, const char* what) {
    return e == cudaSuccess ? MLXQ_OK : fail(MLXQ_ERR_CUDA, what, cudaGetErrorString(e));
}

bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

constexpr int64_t kIntMax = 0x7fffffffLL;

int check_cache(const mlxq_kv_cache* c, int n_q_heads, const char* what, mlxq::KvCache* out) {
    if (!c) return fail(MLXQ_ERR_NULL, what, "NULL cache");
    if (c->dtype != MLXQ_BF16 && c->dtype != MLXQ_F16)
        return fail(MLXQ_ERR_DTYPE, what, "the cache's dtype must be bf16 or f16");
    if (c->head_dim != 64 && c->head_dim != 128)
        return fail(MLXQ_ERR_SHAPE, what, "head_dim must be 64 or 128");
    if (c->page_size != 8 && c->page_size != 16 && c->page_size != 32)
        return fail(MLXQ_ERR_SHAPE, what, "page_size must be 8, 16 or 32");
    if (c->bits != 16 && c->bits != 8 && c->bits != 4)
        return fail(MLXQ_ERR_UNSUPPORTED_BITS, what, "cache bits must be 16, 8 or 4");
    if (c->n_kv_heads <= 0 || c->n_kv_heads > 1024)
        return fail(MLXQ_ERR_SHAPE, what, "n_kv_heads must be in [1, 1024]");
    if (n_q_heads <= 0 || n_q_heads % c->n_kv_heads || n_q_heads / c->n_kv_heads > 8)
        return fail(MLXQ_ERR_SHAPE, what, "n_q_heads must be a multiple of n_kv_heads, at most 8 "
                                          "query heads per kv head");
    if (c->num_pages <= 0 || c->num_pages > kIntMax / c->page_size)
        return fail(MLXQ_ERR_SHAPE, what, "num_pages must be positive, with fewer than 2^31 rows");
    if (c->num_pages * c->page_size >= (1LL << 32) / c->n_kv_heads)
        return fail(MLXQ_ERR_SHAPE, what, "a pool holds fewer than 2^32 rows of one head");
    if (!c->k || !c->v) return fail(MLXQ_ERR_NULL, what, "NULL cache pool");
    if (!aligned(c->k, 16) || !aligned(c->v, 16))
        return fail(MLXQ_ERR_ALIGN, what, "cache pools must be 16-byte aligned");
    if (c->bits != 16) {
        if ((c->group_size != 32 && c->group_size != 64 && c->group_size != 128) ||
            c->group_size > c->head_dim)
            return fail(MLXQ_ERR_GROUP_SIZE, what,
                        "cache group_size must be 32, 64 or 128 and at most head_dim");
        if (!c->k_scales || !c->k_biases || !c->v_scales || !c->v_biases)
            return fail(MLXQ_ERR_NULL, what, "NULL cache scales or biases");
        if (!aligned(c->k_scales, 4) || !aligned(c->k_biases, 4) || !aligned(c->v_scales, 4) ||
            !aligned(c->v_biases, 4))
            return fail(MLXQ_ERR_ALIGN, what, "cache scales and biases must be 4-byte aligned");
    }
    out->k = c->k;
    out->v = c->v;
    out->ks = c->k_scales;
    out->kb = c->k_biases;
    out->vs = c->v_scales;
    out->vb = c->v_biases;
    out->pages = static_cast<int>(c->num_pages);
    out->page = c->page_size;
    out->Hkv = c->n_kv_heads;
    out->hd = c->head_dim;
    out->bits = c->bits;
    out->gs = c->bits == 16 ? c->head_dim : c->group_size;
    out->dtype = c->dtype;
    return MLXQ_OK;
}

}  // namespace

extern "C" {

int mlxq_norm_rope_kv_append(const mlxq_kv_cache* cache, const void* qkv, int64_t ld, void* q_out,
                             const void* q_norm, const void* k_norm, float eps,
                             const int32_t* positions, const int32_t* slots, int64_t tokens,
                             int n_q_heads, float rope_base, void* stream) {
    const char* what = "norm_rope_kv_append";
    mlxq::KvCache c;
    if (int rc = check_cache(cache, n_q_heads, what, &c)) return rc;
    if (tokens < 0 || tokens > kIntMax ||
        ld < (n_q_heads + 2 * static_cast<int64_t>(c.Hkv)) * c.hd || ld % 8 || ld > kIntMax)
        return fail(MLXQ_ERR_SHAPE, what, "ld must hold q, k and v (a multiple of 8)");
    if (!(rope_base > 1.0f) || !std::isfinite(rope_base))
        return fail(MLXQ_ERR_SHAPE, what, "rope_base must be > 1 and finite");
    if (!(eps >= 0.0f) || !std::isfinite(eps))
        return fail(MLXQ_ERR_SHAPE, what, "eps must be >= 0 and finite");
    if (tokens == 0) return MLXQ_OK;
    if (!qkv || !q_out || !positions || !slots) return fail(MLXQ_ERR_NULL, what, "NULL pointer");
    if (!aligned(qkv, 16) || !aligned(q_out, 16) || !aligned(q_norm, 16) || !aligned(k_norm, 16))
        return fail(MLXQ_ERR_ALIGN, what, "pointers must be 16-byte aligned");
    return done(mlxq::launch_norm_rope_append(c, qkv, ld, q_out, q_norm, k_norm, eps, positions,
                                              slots, static_cast<int>(tokens), n_q_heads, rope_base,
                                              mlxq::launch_overlap_enabled(),
                                              static_cast<cudaStream_t>(stream)),
                what);
}

int mlxq_kv_cache_read(const mlxq_kv_cache* cache, const int32_t* slots, int64_t n, void* k_out,
                       void* v_out, void* stream) {
    const char* what = "kv_cache_read";
    mlxq::KvCache c;
    if (int rc = check_cache(cache, cache ? cache->n_kv_heads : 1, what, &c)) return rc;
    if (n < 0 || n > kIntMax) return fail(MLXQ_ERR_SHAPE, what, "bad number of rows");
    if (n == 0) return MLXQ_OK;
    if (n * c.Hkv * (c.hd / 8) > (kIntMax - 256) * 256)
        return fail(MLXQ_ERR_SHAPE, what, "too many rows for one call");
    if (!slots || !k_out || !v_out) return fail(MLXQ_ERR_NULL, what, "NULL pointer");
    if (!aligned(k_out, 16) || !aligned(v_out, 16))
        return fail(MLXQ_ERR_ALIGN, what, "outputs must be 16-byte aligned");
    return done(mlxq::launch_cache_read(c, slots, static_cast<int>(n), k_out, v_out,
                                        mlxq::launch_overlap_enabled(),
                                        static_cast<cudaStream_t>(stream)),
                what);
}

size_t mlxq_paged_attention_rows_workspace_size(const mlxq_kv_cache* cache, int64_t batch,
                                                int64_t max_q_len, int64_t max_kv_len,
                                                int n_q_heads) {
    mlxq::KvCache c;
    if (check_cache(cache, n_q_heads, "paged_attention_rows", &c) || batch <= 0 || batch > 65535 ||
        max_q_len <= 0 || max_q_len > kIntMax / 64 || max_kv_len < 0 || max_kv_len > kIntMax / 2)
        return 0;
    mlxq::RowsArgs a = {};
    a.batch = static_cast<int>(batch);
    a.max_q = static_cast<int>(max_q_len);
    a.max_kv = static_cast<int>(max_kv_len);
    a.Hq = n_q_heads;
    return mlxq::attn_rows_workspace(c, a);
}

int mlxq_paged_attention_rows(const mlxq_kv_cache* cache, const void* q, const int32_t* cu_q,
                              int64_t total, int64_t max_q_len, const int32_t* block_table,
                              int64_t max_blocks, const int32_t* kv_lens, int64_t max_kv_len,
                              const int64_t* tree_mask, void* out, int64_t batch, int n_q_heads,
                              float scale, void* workspace, size_t workspace_bytes, void* stream) {
    const char* what = "paged_attention_rows";
    mlxq::KvCache c;
    if (int rc = check_cache(cache, n_q_heads, what, &c)) return rc;
    if (batch < 0 || batch > 65535 || total < 0 || total > kIntMax / 64 || max_q_len < 0 ||
        max_q_len > kIntMax / 64)
        return fail(MLXQ_ERR_SHAPE, what, "bad batch, total or query length");
    if (!cu_q && (total != batch || max_q_len != 1))
        return fail(MLXQ_ERR_SHAPE, what, "without cu_q there is one row per sequence");
    if (max_blocks <= 0 || max_blocks > kIntMax || max_kv_len < 0 || max_kv_len > kIntMax / 2 ||
        max_kv_len > max_blocks * c.page)
        return fail(MLXQ_ERR_SHAPE, what, "max_kv_len must be in [0, max_blocks * page_size]");
    if (tree_mask && max_q_len > 64)
        return fail(MLXQ_ERR_SHAPE, what, "a tree has at most 64 tokens");
    if (!std::isfinite(scale)) return fail(MLXQ_ERR_SHAPE, what, "scale must be finite");
    if (total == 0) return MLXQ_OK;
    if (!out) return fail(MLXQ_ERR_NULL, what, "NULL pointer");
    if (!aligned(q, 16) || !aligned(out, 16))
        return fail(MLXQ_ERR_ALIGN, what, "q and out must be 16-byte aligned");
    if (batch == 0 || max_q_len == 0)  // every row is behind the last sequence
        return done(cudaMemsetAsync(out, 0, static_cast<size_t>(total) * n_q_heads * c.hd * 2,
                                    static_cast<cudaStream_t>(stream)),
                    what);
    if (!q || !block_table || !kv_lens) return fail(MLXQ_ERR_NULL, what, "NULL pointer");
    mlxq::RowsArgs a;
    a.q = q;
    a.out = out;
    a.cu_q = cu_q;
    a.kv_lens = kv_lens;
    a.table = block_table;
    a.mask = reinterpret_cast<const long long*>(tree_mask);
    a.max_blocks = static_cast<int>(max_blocks);
    a.max_kv = static_cast<int>(max_kv_len);
    a.max_q = static_cast<int>(max_q_len);
    a.total = static_cast<int>(total);
    a.batch = static_cast<int>(batch);
    a.Hq = n_q_heads;
    a.scale = scale;
    a.tail = true;
    if (!mlxq::attn_rows_countable(c, a))
        return fail(MLXQ_ERR_SHAPE, what, "batch, query and key lengths are too large together");
    const size_t need = mlxq::attn_rows_workspace(c, a);
    if (need) {
        if (!workspace || workspace_bytes < need)
            return fail(MLXQ_ERR_WORKSPACE, what, "workspace missing or too small");
        if (!aligned(workspace, 256))
            return fail(MLXQ_ERR_ALIGN, what, "workspace must be 256-byte aligned");
    }
    return done(mlxq::launch_attn_rows(c, a, workspace, mlxq::launch_overlap_enabled(),
                                       static_cast<cudaStream_t>(stream)),
                what);
}

}  // extern "C"
