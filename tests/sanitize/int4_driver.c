/* Drives the host checks of the entry points over a cache in 4 bits through
 * the edges of every field: nothing may read past a struct, overflow, or reach
 * a launch. */
#include <limits.h>
#include <math.h>
#include <stdio.h>
#include <string.h>

#include "orth_hip.h"

static int failures;

static void expect(const char *what, int got, int want) {
    if (got != want) {
        printf("%s: %d (%s)\n", what, got, orth_hip_last_error());
        failures++;
    }
}

#define P(n) ((void *)(uintptr_t)(n))

int main(void) {
    static const int64_t edges[] = {INT64_MIN, -1, 0, 1, 7, 8, 64, INT32_MAX, (int64_t)INT32_MAX + 1, (int64_t)1 << 46, INT64_MAX};
    static const int32_t small[] = {INT32_MIN, -1, 0, 1, 2, 7, 8, 32, 64, 128, 256, 257, 1 << 24, INT32_MAX};
    const int n = sizeof(edges) / sizeof(edges[0]), m = sizeof(small) / sizeof(small[0]);
    const orth_hip_int4_cache_t cache = {P(0x10000), P(0x20000), P(0x30000), P(0x40000), 16, 2, 64, 32, 8,
                                         {1024, 64, 32}, {1024, 64, 32}, {128, 8, 4}, {128, 8, 4}};
    const orth_hip_append_t append = {P(8), P(16), P(24), P(32), {256, 64}, {128, 64}, {128, 64}, {256, 64},
                                      P(40), P(48), P(56), 32, 5, 4, 64, 0, 0};
    const orth_hip_attend_t attend = {P(8), P(16), {256, 64}, {256, 64}, P(24), P(32), NULL, 8, 8, 8, 5, 4, 0, 0.125f, 0};
    const orth_hip_read_t read = {P(0x100), P(0x10000), {128, 64}, {128, 64}, P(40), 5};
    int i, k;

    expect("append", orth_cache_append_int4_hip(&cache, &append, ORTH_DT_F16, NULL), ORTH_ERR_NO_DEVICE);
    expect("read", orth_cache_read_int4_hip(&cache, &read, ORTH_DT_BF16, NULL), ORTH_ERR_NO_DEVICE);
    expect("attend", orth_paged_attention_int4_hip(&cache, &attend, ORTH_DT_F16, NULL), ORTH_ERR_NO_DEVICE);

    /* every 64-bit and 32-bit field at its edges: refused, or fit for a device */
#define TRY(T, base, field, values, count, call)                     \
    for (i = 0; i < (count); i++) {                                  \
        T x = base;                                                  \
        x.field = values[i];                                         \
        int rc = call;                                               \
        if (rc == ORTH_ERR_HIP) expect(#T "." #field, rc, ORTH_OK);  \
    }
#define EACH_CALL(field, values, count)                                                                                      \
    TRY(orth_hip_int4_cache_t, cache, field, values, count, orth_paged_attention_int4_hip(&x, &attend, ORTH_DT_F16, NULL)) \
    TRY(orth_hip_int4_cache_t, cache, field, values, count, orth_cache_append_int4_hip(&x, &append, ORTH_DT_BF16, NULL))   \
    TRY(orth_hip_int4_cache_t, cache, field, values, count, orth_cache_read_int4_hip(&x, &read, ORTH_DT_F16, NULL))
    EACH_CALL(pages, edges, n)
    for (k = 0; k < 3; k++) {
        EACH_CALL(k_code_strides[k], edges, n)
        EACH_CALL(v_code_strides[k], edges, n)
        EACH_CALL(k_scale_strides[k], edges, n)
        EACH_CALL(v_scale_strides[k], edges, n)
    }
    EACH_CALL(page_size, small, m)
    EACH_CALL(kv_heads, small, m)
    EACH_CALL(head_dim, small, m)
    EACH_CALL(group_size, small, m)
#define APPEND orth_cache_append_int4_hip(&cache, &x, ORTH_DT_F16, NULL)
    TRY(orth_hip_append_t, append, tokens, edges, n, APPEND)
    TRY(orth_hip_append_t, append, cos_sin_rows, edges, n, APPEND)
    TRY(orth_hip_append_t, append, q_strides[0], edges, n, APPEND)
    TRY(orth_hip_append_t, append, q_out_strides[1], edges, n, APPEND)
    TRY(orth_hip_append_t, append, k_strides[0], edges, n, APPEND)
    TRY(orth_hip_append_t, append, v_strides[1], edges, n, APPEND)
    TRY(orth_hip_append_t, append, q_heads, small, m, APPEND)
    TRY(orth_hip_append_t, append, rot, small, m, APPEND)
#define READ orth_cache_read_int4_hip(&cache, &x, ORTH_DT_F16, NULL)
    TRY(orth_hip_read_t, read, count, edges, n, READ)
    TRY(orth_hip_read_t, read, k_strides[0], edges, n, READ)
    TRY(orth_hip_read_t, read, v_strides[1], edges, n, READ)
#define ATTEND orth_paged_attention_int4_hip(&cache, &x, ORTH_DT_BF16, NULL)
    TRY(orth_hip_attend_t, attend, tokens, edges, n, ATTEND)
    TRY(orth_hip_attend_t, attend, table_rows, edges, n, ATTEND)
    TRY(orth_hip_attend_t, attend, table_width, edges, n, ATTEND)
    TRY(orth_hip_attend_t, attend, table_stride, edges, n, ATTEND)
    TRY(orth_hip_attend_t, attend, q_strides[0], edges, n, ATTEND)
    TRY(orth_hip_attend_t, attend, out_strides[1], edges, n, ATTEND)
    TRY(orth_hip_attend_t, attend, q_heads, small, m, ATTEND)
    TRY(orth_hip_attend_t, attend, window, small, m, ATTEND)
    for (k = 0; k < m; k++) {
        if (small[k] == ORTH_DT_F16 || small[k] == ORTH_DT_BF16) continue;
        expect("dtype", orth_cache_read_int4_hip(&cache, &read, small[k], NULL), ORTH_ERR_UNSUPPORTED);
    }
    {
        orth_hip_attend_t x = attend;
        x.scale = NAN;
        expect("scale", orth_paged_attention_int4_hip(&cache, &x, ORTH_DT_F16, NULL), ORTH_ERR_INVALID_ARGUMENT);
    }
    expect("null", orth_cache_append_int4_hip(NULL, &append, ORTH_DT_F16, NULL), ORTH_ERR_INVALID_ARGUMENT);
    expect("null", orth_cache_append_int4_hip(&cache, NULL, ORTH_DT_F16, NULL), ORTH_ERR_INVALID_ARGUMENT);
    expect("null", orth_cache_read_int4_hip(&cache, NULL, ORTH_DT_F16, NULL), ORTH_ERR_INVALID_ARGUMENT);
    expect("null", orth_paged_attention_int4_hip(NULL, &attend, ORTH_DT_F16, NULL), ORTH_ERR_INVALID_ARGUMENT);
    if (failures) return 1;
    printf("int4 ok\n");
    return 0;
}
