// Host side of the entry points over the cache in 4 bits: argument
// validation, workspaces and launches.
#include "orth_serve4.h"

#include "orth_checks.h"

using namespace orth;

namespace {

int check_int4_cache(const orth_hip_int4_cache_t *c) {
    if (!c) return invalid("cache is NULL");
    if (c->page_size < 1) return invalid("page_size must be positive");
    if (c->kv_heads < 1) return invalid("kv_heads must be positive");
    if (c->head_dim < 8 || c->head_dim % 8 || c->head_dim > 256)
        return host_fail(ORTH_ERR_UNSUPPORTED, "head_dim must be a multiple of 8, at most 256");
    const int32_t g = c->group_size;
    if (g != c->head_dim && ((g != 32 && g != 64 && g != 128) || c->head_dim % g))
        return host_fail(ORTH_ERR_UNSUPPORTED, "group_size must be head_dim, or 32, 64 or 128 where that divides it");
    if (c->pages < 1 || c->pages > kMaxInt) return invalid("pages must be positive, at most 2^31 - 1");
    if (!c->k_codes || !c->v_codes || !c->k_scales || !c->v_scales) return invalid("codes or scales is NULL");
    if (!aligned(c->k_codes, 16) || !aligned(c->v_codes, 16)) return invalid("codes must be 16-byte aligned");
    if (!aligned(c->k_scales, 4) || !aligned(c->v_scales, 4)) return invalid("scales must be 4-byte aligned");
    for (int i = 0; i < 3; i++) {
        if (c->k_code_strides[i] % 16 || c->v_code_strides[i] % 16) return invalid("strides of codes must be multiples of 16");
        if (c->k_scale_strides[i] % 2 || c->v_scale_strides[i] % 2) return invalid("strides of scales must be even");
    }
    const int64_t n[3] = {c->pages, c->page_size, c->kv_heads};
    if (!span_ok(c->k_code_strides, n, 3) || !span_ok(c->v_code_strides, n, 3) || !span_ok(c->k_scale_strides, n, 3) ||
        !span_ok(c->v_scale_strides, n, 3))
        return invalid("a cache stride is negative or too large");
    return ORTH_OK;
}

int check_dtype(int32_t dtype) {
    return dtype == ORTH_DT_F16 || dtype == ORTH_DT_BF16 ? (int)ORTH_OK
                                                         : host_fail(ORTH_ERR_UNSUPPORTED, "dtype must be F16 or BF16");
}

}  // namespace

extern "C" {

int orth_cache_append_int4_hip(const orth_hip_int4_cache_t *c, const orth_hip_append_t *a, int32_t dtype, void *stream) {
    return guarded([&]() -> int {
        int rc = check_int4_cache(c);
        if (rc == ORTH_OK) rc = check_dtype(dtype);
        if (rc == ORTH_OK) rc = check_append(a, c->kv_heads, c->head_dim);
        if (rc != ORTH_OK || a->tokens == 0) return rc;
        int dev = 0, cus = 0;
        if ((rc = host_device(&dev, &cus)) != ORTH_OK) return rc;
        hipError_t e = launch_cache_append4(*c, *a, dtype, cus, static_cast<hipStream_t>(stream));
        return e == hipSuccess ? (int)ORTH_OK : host_fail_hip(e, "cache append launch");
    });
}

int orth_cache_read_int4_hip(const orth_hip_int4_cache_t *c, const orth_hip_read_t *r, int32_t dtype, void *stream) {
    return guarded([&]() -> int {
        int rc = check_int4_cache(c);
        if (rc == ORTH_OK) rc = check_dtype(dtype);
        if (rc != ORTH_OK) return rc;
        if (!r) return invalid("read is NULL");
        if (r->count < 0 || r->count > kMaxInt) return invalid("count must not be negative, at most 2^31 - 1");
        if (r->count > 0 && (!r->k_out || !r->v_out || !r->slots)) return invalid("k_out, v_out or slots is NULL");
        if (!aligned(r->k_out, 2) || !aligned(r->v_out, 2)) return invalid("k_out and v_out must be aligned to their elements");
        if ((rc = check_heads(r->k_strides, r->count, c->kv_heads, "a stride of k_out is negative or too large")) != ORTH_OK ||
            (rc = check_heads(r->v_strides, r->count, c->kv_heads, "a stride of v_out is negative or too large")) != ORTH_OK)
            return rc;
        if (c->kv_heads > (1 << 24)) return host_fail(ORTH_ERR_UNSUPPORTED, "kv_heads passes 2^24");
        if (r->count == 0) return ORTH_OK;
        if (!apart(r->k_strides, r->count, c->kv_heads, c->head_dim) || !apart(r->v_strides, r->count, c->kv_heads, c->head_dim))
            return invalid("the vectors of k_out or v_out overlap");
        int dev = 0, cus = 0;
        if ((rc = host_device(&dev, &cus)) != ORTH_OK) return rc;
        hipError_t e = launch_cache_read4(*c, *r, dtype, cus, static_cast<hipStream_t>(stream));
        return e == hipSuccess ? (int)ORTH_OK : host_fail_hip(e, "cache read launch");
    });
}

int orth_paged_attention_int4_hip(const orth_hip_int4_cache_t *c, const orth_hip_attend_t *a, int32_t dtype, void *stream) {
    return guarded([&]() -> int {
        int rc = check_int4_cache(c);
        if (rc == ORTH_OK) rc = check_dtype(dtype);
        if (rc == ORTH_OK) rc = check_attend(a, c->page_size, c->kv_heads, c->head_dim);
        if (rc != ORTH_OK || a->tokens == 0) return rc;
        int dev = 0, cus = 0;
        if ((rc = host_device(&dev, &cus)) != ORTH_OK) return rc;
        void *work = nullptr;
        uint32_t *counters = nullptr;
        int64_t groups = 0;
        std::unique_lock<std::mutex> held;
        const int64_t bytes = attention4_workspace_bytes(*c, *a, cus, &groups);
        if (bytes > 0 && (rc = host_workspace(dev, static_cast<hipStream_t>(stream), bytes, &work, &held)) != ORTH_OK) return rc;
        if ((rc = host_counters(dev, static_cast<hipStream_t>(stream), groups, &counters, &held)) != ORTH_OK) return rc;
        hipError_t e = launch_paged_attention4(*c, *a, dtype, cus, work, counters, static_cast<hipStream_t>(stream));
        return e == hipSuccess ? (int)ORTH_OK : host_fail_hip(e, "paged attention launch");
    });
}

}  // extern "C"
