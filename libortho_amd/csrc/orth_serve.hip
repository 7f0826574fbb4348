// Host side of the serving entry points of include/orth_hip.h: argument
// validation, workspaces and launches of the page step, the cache append,
// the paged attention and the adapters.
#include "orth_checks.h"
#include "orth_serve.h"

using namespace orth;

namespace {

int check_cache(const orth_hip_cache_t *c) {
    if (!c) return invalid("cache is NULL");
    if (c->dtype != ORTH_DT_F16 && c->dtype != ORTH_DT_BF16)
        return host_fail(ORTH_ERR_UNSUPPORTED, "the cache's dtype must be F16 or BF16");
    if (c->page_size < 1) return invalid("page_size must be positive");
    if (c->kv_heads < 1) return invalid("kv_heads must be positive");
    if (c->head_dim < 8 || c->head_dim % 8 || c->head_dim > 256)
        return host_fail(ORTH_ERR_UNSUPPORTED, "head_dim must be a multiple of 8, at most 256");
    if (c->pages < 1 || c->pages > kMaxInt) return invalid("pages must be positive, at most 2^31 - 1");
    if (!c->k_cache || !c->v_cache) return invalid("k_cache or v_cache is NULL");
    if (!aligned(c->k_cache, 16) || !aligned(c->v_cache, 16)) return invalid("k_cache and v_cache must be 16-byte aligned");
    for (int i = 0; i < 3; i++)
        if (c->k_strides[i] % 8 || c->v_strides[i] % 8) return invalid("the cache's strides must be multiples of 8");
    const int64_t n[3] = {c->pages, c->page_size, c->kv_heads};
    if (!span_ok(c->k_strides, n, 3) || !span_ok(c->v_strides, n, 3))
        return invalid("a cache stride is negative or too large");
    return ORTH_OK;
}

}  // namespace

extern "C" {

int orth_page_step_hip(const orth_hip_step_t *s, void *stream) {
    return guarded([&]() -> int {
        if (!s) return invalid("step is NULL");
        if (s->requests < 0 || s->tokens < 0 || s->free_count < 0 || s->table_width < 0)
            return invalid("requests, tokens, free_count and table_width must not be negative");
        if (s->requests > ORTH_STEP_REQUESTS)
            return host_fail(ORTH_ERR_UNSUPPORTED, "a step holds at most 8192 requests");
        if (s->tokens > kMaxInt || s->free_count > kMaxInt || s->table_width > kMaxInt)
            return invalid("tokens, free_count and table_width are at most 2^31 - 1");
        if (s->page_size < 1) return invalid("page_size must be positive");
        if (s->table_stride < s->table_width || s->table_stride > kMaxSpan / ORTH_STEP_REQUESTS)
            return invalid("table_stride is smaller than table_width, or too large");
        if (!s->pool || !s->pool_out || !s->query_start) return invalid("pool, pool_out or query_start is NULL");
        if (s->requests > 0 && (!s->lengths || !s->new_tokens || !s->lengths_out))
            return invalid("lengths, new_tokens or lengths_out is NULL");
        if (s->requests > 0 && s->table_width > 0 && !s->block_table) return invalid("block_table is NULL");
        if (s->free_count > 0 && !s->free_pages) return invalid("free_pages is NULL");
        if (s->tokens > 0 && (!s->rows || !s->positions || !s->slots)) return invalid("rows, positions or slots is NULL");
        if (s->lengths_out && (s->lengths_out == s->lengths || s->lengths_out == s->new_tokens))
            return invalid("lengths_out must not be an input");
        if (s->pool_out == s->pool) return invalid("pool_out must not be pool");
        int dev = 0, cus = 0;
        int rc = host_device(&dev, &cus);
        if (rc != ORTH_OK) return rc;
        hipError_t e = launch_page_step(*s, static_cast<hipStream_t>(stream));
        return e == hipSuccess ? (int)ORTH_OK : host_fail_hip(e, "page step launch");
    });
}

int orth_cache_append_hip(const orth_hip_cache_t *c, const orth_hip_append_t *a, void *stream) {
    return guarded([&]() -> int {
        int rc = check_cache(c);
        if (rc == ORTH_OK) rc = check_append(a, c->kv_heads, c->head_dim);
        if (rc != ORTH_OK || a->tokens == 0) return rc;
        int dev = 0, cus = 0;
        rc = host_device(&dev, &cus);
        if (rc != ORTH_OK) return rc;
        hipError_t e = launch_cache_append(*c, *a, cus, static_cast<hipStream_t>(stream));
        return e == hipSuccess ? (int)ORTH_OK : host_fail_hip(e, "cache append launch");
    });
}

int orth_paged_attention_hip(const orth_hip_cache_t *c, const orth_hip_attend_t *a, void *stream) {
    return guarded([&]() -> int {
        int rc = check_cache(c);
        if (rc == ORTH_OK) rc = check_attend(a, c->page_size, c->kv_heads, c->head_dim);
        if (rc != ORTH_OK || a->tokens == 0) return rc;
        int dev = 0, cus = 0;
        rc = host_device(&dev, &cus);
        if (rc != ORTH_OK) return rc;
        void *work = nullptr;
        uint32_t *counters = nullptr;
        int64_t groups = 0;
        std::unique_lock<std::mutex> held;
        const int64_t bytes = attention_workspace_bytes(*c, *a, cus, &groups);
        if ((rc = host_workspace(dev, static_cast<hipStream_t>(stream), bytes, &work, &held)) != ORTH_OK) return rc;
        if ((rc = host_counters(dev, static_cast<hipStream_t>(stream), groups, &counters, &held)) != ORTH_OK) return rc;
        hipError_t e = launch_paged_attention(*c, *a, cus, work, counters, static_cast<hipStream_t>(stream));
        return e == hipSuccess ? (int)ORTH_OK : host_fail_hip(e, "paged attention launch");
    });
}

int orth_adapter_add_hip(const orth_hip_adapter_t *a, void *stream) {
    return guarded([&]() -> int {
        if (!a) return invalid("adapter is NULL");
        if (a->dtype != ORTH_DT_F16 && a->dtype != ORTH_DT_BF16)
            return host_fail(ORTH_ERR_UNSUPPORTED, "adapters take F16 or BF16");
        if (a->rank < 1 || a->rank > ORTH_ADAPTER_RANK)
            return host_fail(ORTH_ERR_UNSUPPORTED, "rank must lie in 1..256");
        if (a->in_features < 1 || a->out_features < 1) return invalid("in_features and out_features must be positive");
        if (a->in_features > kMaxInt || a->out_features > kMaxInt)
            return invalid("in_features and out_features are at most 2^31 - 1");
        if (a->tokens < 0 || a->tokens > kMaxInt) return invalid("tokens must not be negative, at most 2^31 - 1");
        if (a->count < 0 || a->count > kMaxInt) return invalid("count must not be negative, at most 2^31 - 1");
        if (a->count > 0 && (a->count > kMaxSpan / a->rank / a->in_features || a->count > kMaxSpan / a->rank / a->out_features))
            return invalid("the adapters are too large");
        if (a->tokens > 0) {
            if (!a->x || !a->y || !a->out || !a->adapters) return invalid("x, y, out or adapters is NULL");
            if (a->count > 0 && (!a->a || !a->b)) return invalid("a or b is NULL");
        }
        if (!aligned(a->x, 2) || !aligned(a->y, 2) || !aligned(a->out, 2) || !aligned(a->a, 2) || !aligned(a->b, 2))
            return invalid("x, y, out, a and b must be aligned to their elements");
        if (a->x_stride < 0 || a->y_stride < 0 || a->out_stride < 0 ||
            (a->tokens > 0 && (a->x_stride > kMaxSpan / a->tokens || a->y_stride > kMaxSpan / a->tokens ||
                               a->out_stride > kMaxSpan / a->tokens)))
            return invalid("a row stride is negative or too large");
        if (a->tokens > 1 && a->out_stride < a->out_features) return invalid("the rows of out overlap");
        if (a->out == a->y && a->tokens > 1 && a->out_stride != a->y_stride) return invalid("out is y with another stride");
        if (a->tokens == 0) return ORTH_OK;
        int dev = 0, cus = 0;
        int rc = host_device(&dev, &cus);
        if (rc != ORTH_OK) return rc;
        void *work = nullptr;
        std::unique_lock<std::mutex> held;
        const int64_t bytes = adapter_workspace_bytes(*a, cus);
        if (bytes > 0 && (rc = host_workspace(dev, static_cast<hipStream_t>(stream), bytes, &work, &held)) != ORTH_OK)
            return rc;
        hipError_t e = launch_adapter_add(*a, cus, work, static_cast<hipStream_t>(stream));
        return e == hipSuccess ? (int)ORTH_OK : host_fail_hip(e, "adapter launch");
    });
}

}  // extern "C"
