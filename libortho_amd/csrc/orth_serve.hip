// Host side of the serving entry points of include/orth_hip.h: argument
// validation, workspaces and launches of the page step, the cache append,
// the paged attention and the adapters.
#include <new>

#include "orth_host.h"
#include "orth_serve.h"

using namespace orth;

namespace {

int invalid(const char *message) { return host_fail(ORTH_ERR_INVALID_ARGUMENT, message); }

bool aligned(const void *p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// No C++ exception (an allocation of the host's maps) leaves a C entry.
template <class F>
int guarded(F &&body) noexcept {
    try {
        host_begin();
        return body();
    } catch (...) {
        try {
            return host_fail(ORTH_ERR_HIP, "out of host memory");
        } catch (...) {
            return ORTH_ERR_HIP;
        }
    }
}

constexpr int64_t kMaxInt = INT32_MAX;
constexpr int64_t kMaxSpan = (int64_t)1 << 46;  // elements an index may reach: products of strides stay within int64

// strides[0..n) times counts[0..n) stay within kMaxSpan; no stride negative
bool span_ok(const int64_t *strides, const int64_t *counts, int n) {
    for (int i = 0; i < n; i++)
        if (strides[i] < 0 || (counts[i] > 0 && strides[i] > kMaxSpan / counts[i])) return false;
    return true;
}

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

int check_heads(const int64_t *strides, int64_t tokens, int64_t heads, const char *message) {
    const int64_t n[2] = {tokens, heads};
    return span_ok(strides, n, 2) ? (int)ORTH_OK : invalid(message);
}

// Whether the vectors of an output [tokens, heads, dim] keep apart, tokens
// outside heads or heads outside tokens.
bool apart(const int64_t *strides, int64_t tokens, int64_t heads, int64_t dim) {
    const int64_t t = strides[0], h = strides[1];
    const int64_t token = (heads - 1) * h + dim, head = (tokens - 1) * t + dim;
    return (heads == 1 || h >= dim) && (tokens == 1 || t >= dim) &&
           (tokens == 1 || heads == 1 || t >= token || h >= head);
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
        if (rc != ORTH_OK) return rc;
        if (!a) return invalid("append is NULL");
        if (a->tokens < 0 || a->tokens > kMaxInt) return invalid("tokens must not be negative, at most 2^31 - 1");
        if (a->cos_sin) {
            if (a->rot < 0 || a->rot % 2 || a->rot > c->head_dim)
                return invalid("rot must be even and at most head_dim");
            if (a->cos_sin_rows < 0 || a->cos_sin_rows > kMaxInt) return invalid("cos_sin_rows must not be negative");
            if (!aligned(a->cos_sin, 4)) return invalid("cos_sin is not aligned to its elements");
            if (a->tokens > 0 && !a->positions) return invalid("positions is NULL");
        } else if (a->q) {
            return invalid("q is given without cos_sin");
        }
        if (a->q && a->q_heads < 1) return invalid("q_heads must be positive");
        if ((int64_t)(a->q ? a->q_heads : 0) + 2 * (int64_t)c->kv_heads > (1 << 30))
            return host_fail(ORTH_ERR_UNSUPPORTED, "q_heads + 2 * kv_heads passes 2^30");
        if (a->tokens > 0 && (!a->k || !a->v || !a->slots)) return invalid("k, v or slots is NULL");
        if (a->tokens > 0 && a->q && !a->q_out) return invalid("q_out is NULL");
        if (!aligned(a->q, 2) || !aligned(a->k, 2) || !aligned(a->v, 2) || !aligned(a->q_out, 2))
            return invalid("q, k, v and q_out must be aligned to their elements");
        if ((rc = check_heads(a->k_strides, a->tokens, c->kv_heads, "a stride of k is negative or too large")) != ORTH_OK ||
            (rc = check_heads(a->v_strides, a->tokens, c->kv_heads, "a stride of v is negative or too large")) != ORTH_OK)
            return rc;
        if (a->q && ((rc = check_heads(a->q_strides, a->tokens, a->q_heads, "a stride of q is negative or too large")) != ORTH_OK ||
                     (rc = check_heads(a->q_out_strides, a->tokens, a->q_heads, "a stride of q_out is negative or too large")) != ORTH_OK))
            return rc;
        if (a->q && a->q_out == a->q && (a->q_strides[0] != a->q_out_strides[0] || a->q_strides[1] != a->q_out_strides[1]))
            return invalid("q_out is q with other strides");
        if (a->tokens == 0) return ORTH_OK;
        if (a->q && !apart(a->q_out_strides, a->tokens, a->q_heads, c->head_dim)) return invalid("the vectors of q_out overlap");
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
        if (rc != ORTH_OK) return rc;
        if (!a) return invalid("attend is NULL");
        if (a->tokens < 0 || a->tokens > kMaxInt) return invalid("tokens must not be negative, at most 2^31 - 1");
        if (a->q_heads < 1 || a->q_heads % c->kv_heads) return invalid("q_heads must be a multiple of kv_heads");
        if (a->tokens > kMaxInt / a->q_heads) return host_fail(ORTH_ERR_UNSUPPORTED, "tokens * q_heads passes 2^31 - 1");
        if (a->window < 0) return invalid("window must not be negative");
        if (a->scale != a->scale) return invalid("scale is NaN");
        if (a->table_rows < 0 || a->table_width < 0 || a->table_rows > kMaxInt || a->table_width > kMaxInt)
            return invalid("table_rows and table_width must not be negative, at most 2^31 - 1");
        if (a->table_stride < a->table_width || (a->table_rows > 0 && a->table_stride > kMaxSpan / a->table_rows))
            return invalid("table_stride is smaller than table_width, or too large");
        if (a->table_width * c->page_size > kMostKeys)
            return host_fail(ORTH_ERR_UNSUPPORTED, "table_width * page_size passes 2^31 - 512");
        if (a->tokens > 0) {
            if (!a->q || !a->out || !a->positions) return invalid("q, out or positions is NULL");
            if (a->table_rows > 0 && a->table_width > 0 && !a->block_table) return invalid("block_table is NULL");
            if (!a->rows && a->tokens > a->table_rows) return invalid("more tokens than rows of block_table");
            if (!aligned(a->q, 2) || !aligned(a->out, 2)) return invalid("q and out must be aligned to their elements");
        }
        if ((rc = check_heads(a->q_strides, a->tokens, a->q_heads, "a stride of q is negative or too large")) != ORTH_OK ||
            (rc = check_heads(a->out_strides, a->tokens, a->q_heads, "a stride of out is negative or too large")) != ORTH_OK)
            return rc;
        if (a->tokens == 0) return ORTH_OK;
        if (!apart(a->out_strides, a->tokens, a->q_heads, c->head_dim)) return invalid("the vectors of out overlap");
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
