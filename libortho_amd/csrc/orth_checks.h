// Argument checks that the serving entry points share (orth_serve.hip,
// orth_serve4.hip).
#pragma once

#include <new>

#include "orth_hip.h"
#include "orth_host.h"
#include "orth_serve.h"

namespace orth {

inline int invalid(const char *message) { return host_fail(ORTH_ERR_INVALID_ARGUMENT, message); }

inline bool aligned(const void *p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

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
inline bool span_ok(const int64_t *strides, const int64_t *counts, int n) {
    for (int i = 0; i < n; i++)
        if (strides[i] < 0 || (counts[i] > 0 && strides[i] > kMaxSpan / counts[i])) return false;
    return true;
}

inline int check_heads(const int64_t *strides, int64_t tokens, int64_t heads, const char *message) {
    const int64_t n[2] = {tokens, heads};
    return span_ok(strides, n, 2) ? (int)ORTH_OK : invalid(message);
}

// Whether the vectors of an output [tokens, heads, dim] keep apart, tokens
// outside heads or heads outside tokens.
inline bool apart(const int64_t *strides, int64_t tokens, int64_t heads, int64_t dim) {
    const int64_t t = strides[0], h = strides[1];
    const int64_t token = (heads - 1) * h + dim, head = (tokens - 1) * t + dim;
    return (heads == 1 || h >= dim) && (tokens == 1 || t >= dim) &&
           (tokens == 1 || heads == 1 || t >= token || h >= head);
}

// The new tokens of a cache append, whatever the cache holds.
inline int check_append(const orth_hip_append_t *a, int32_t kv_heads, int32_t head_dim) {
    int rc = ORTH_OK;
    if (!a) return invalid("append is NULL");
    if (a->tokens < 0 || a->tokens > kMaxInt) return invalid("tokens must not be negative, at most 2^31 - 1");
    if (a->cos_sin) {
        if (a->rot < 0 || a->rot % 2 || a->rot > head_dim)
            return invalid("rot must be even and at most head_dim");
        if (a->cos_sin_rows < 0 || a->cos_sin_rows > kMaxInt) return invalid("cos_sin_rows must not be negative");
        if (!aligned(a->cos_sin, 4)) return invalid("cos_sin is not aligned to its elements");
        if (a->tokens > 0 && !a->positions) return invalid("positions is NULL");
    } else if (a->q) {
        return invalid("q is given without cos_sin");
    }
    if (a->q && a->q_heads < 1) return invalid("q_heads must be positive");
    if ((int64_t)(a->q ? a->q_heads : 0) + 2 * (int64_t)kv_heads > (1 << 30))
        return host_fail(ORTH_ERR_UNSUPPORTED, "q_heads + 2 * kv_heads passes 2^30");
    if (a->tokens > 0 && (!a->k || !a->v || !a->slots)) return invalid("k, v or slots is NULL");
    if (a->tokens > 0 && a->q && !a->q_out) return invalid("q_out is NULL");
    if (!aligned(a->q, 2) || !aligned(a->k, 2) || !aligned(a->v, 2) || !aligned(a->q_out, 2))
        return invalid("q, k, v and q_out must be aligned to their elements");
    if ((rc = check_heads(a->k_strides, a->tokens, kv_heads, "a stride of k is negative or too large")) != ORTH_OK ||
        (rc = check_heads(a->v_strides, a->tokens, kv_heads, "a stride of v is negative or too large")) != ORTH_OK)
        return rc;
    if (a->q && ((rc = check_heads(a->q_strides, a->tokens, a->q_heads, "a stride of q is negative or too large")) != ORTH_OK ||
                 (rc = check_heads(a->q_out_strides, a->tokens, a->q_heads, "a stride of q_out is negative or too large")) != ORTH_OK))
        return rc;
    if (a->q && a->q_out == a->q && (a->q_strides[0] != a->q_out_strides[0] || a->q_strides[1] != a->q_out_strides[1]))
        return invalid("q_out is q with other strides");
    if (a->tokens > 0 && a->q && !apart(a->q_out_strides, a->tokens, a->q_heads, head_dim)) return invalid("the vectors of q_out overlap");
    return ORTH_OK;
}

// The tokens and the block table of an attention over a paged cache.
inline int check_attend(const orth_hip_attend_t *a, int32_t page_size, int32_t kv_heads, int32_t head_dim) {
    int rc = ORTH_OK;
    if (!a) return invalid("attend is NULL");
    if (a->tokens < 0 || a->tokens > kMaxInt) return invalid("tokens must not be negative, at most 2^31 - 1");
    if (a->q_heads < 1 || a->q_heads % kv_heads) return invalid("q_heads must be a multiple of kv_heads");
    if (a->tokens > kMaxInt / a->q_heads) return host_fail(ORTH_ERR_UNSUPPORTED, "tokens * q_heads passes 2^31 - 1");
    if (a->window < 0) return invalid("window must not be negative");
    if (a->scale != a->scale) return invalid("scale is NaN");
    if (a->table_rows < 0 || a->table_width < 0 || a->table_rows > kMaxInt || a->table_width > kMaxInt)
        return invalid("table_rows and table_width must not be negative, at most 2^31 - 1");
    if (a->table_stride < a->table_width || (a->table_rows > 0 && a->table_stride > kMaxSpan / a->table_rows))
        return invalid("table_stride is smaller than table_width, or too large");
    if (a->table_width * page_size > kMostKeys)
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
    if (a->tokens > 0 && !apart(a->out_strides, a->tokens, a->q_heads, head_dim)) return invalid("the vectors of out overlap");
    return ORTH_OK;
}

}  // namespace orth
