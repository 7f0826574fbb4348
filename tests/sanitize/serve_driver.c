/* Drives the serving entry points' host checks through the edges of every
 * field: nothing may read past a struct, overflow, or reach a launch. */
#include <limits.h>
#include <math.h>
#include <stdio.h>
#include <string.h>

#include "orth_hip.h"

static int failures;

static void expect(const char *what, int got, int a, int b) {
    if (got != a && got != b) {
        printf("%s: %d (%s)\n", what, got, orth_hip_last_error());
        failures++;
    }
}

#define P(n) ((void *)(uintptr_t)(n))

int main(void) {
    static const int64_t edges[] = {INT64_MIN, -1, 0, 1, 7, 8, 64, INT32_MAX, (int64_t)INT32_MAX + 1, (int64_t)1 << 46, INT64_MAX};
    static const int32_t small[] = {INT32_MIN, -1, 0, 1, 2, 7, 8, 64, 256, 257, INT32_MAX};
    const int n = sizeof(edges) / sizeof(edges[0]), m = sizeof(small) / sizeof(small[0]);
    const orth_hip_cache_t cache = {P(0x10000), P(0x20000), ORTH_DT_F16, 16, 2, 64, 8, {2048, 128, 64}, {2048, 128, 64}};
    const orth_hip_step_t step = {P(8), P(16), P(24), P(32), P(40), P(48), P(56), P(64), P(72), P(80), P(88), 4, 8, 8, 100, 6, 16, 0};
    const orth_hip_append_t append = {P(8), P(16), P(24), P(32), {256, 64}, {128, 64}, {128, 64}, {256, 64},
                                      P(40), P(48), P(56), 32, 5, 4, 64, 0, 0};
    const orth_hip_attend_t attend = {P(8), P(16), {256, 64}, {256, 64}, P(24), P(32), NULL, 8, 8, 8, 5, 4, 0, 0.125f, 0};
    const orth_hip_adapter_t adapter = {P(8), P(16), P(24), P(32), P(40), P(48), NULL, 64, 32, 32, 5, 64, 32, 3, 8, ORTH_DT_F16};
    int i, k;

    expect("step", orth_page_step_hip(&step, NULL), ORTH_ERR_NO_DEVICE, ORTH_ERR_NO_DEVICE);
    expect("append", orth_cache_append_hip(&cache, &append, NULL), ORTH_ERR_NO_DEVICE, ORTH_ERR_NO_DEVICE);
    expect("attend", orth_paged_attention_hip(&cache, &attend, NULL), ORTH_ERR_NO_DEVICE, ORTH_ERR_NO_DEVICE);
    expect("adapter", orth_adapter_add_hip(&adapter, NULL), ORTH_ERR_NO_DEVICE, ORTH_ERR_NO_DEVICE);

    /* every 64-bit and 32-bit field at its edges: refused, or fit for a device */
#define TRY64(T, base, field, call)                                              \
    for (i = 0; i < n; i++) {                                                    \
        T x = base;                                                              \
        x.field = edges[i];                                                      \
        int rc = call;                                                           \
        if (rc == ORTH_ERR_HIP) expect(#T "." #field, rc, ORTH_OK, ORTH_OK);     \
    }
#define TRY32(T, base, field, call)                                              \
    for (k = 0; k < m; k++) {                                                    \
        T x = base;                                                              \
        x.field = small[k];                                                      \
        int rc = call;                                                           \
        if (rc == ORTH_ERR_HIP) expect(#T "." #field, rc, ORTH_OK, ORTH_OK);     \
    }
#define STEP orth_page_step_hip(&x, NULL)
    TRY64(orth_hip_step_t, step, requests, STEP)
    TRY64(orth_hip_step_t, step, table_width, STEP)
    TRY64(orth_hip_step_t, step, table_stride, STEP)
    TRY64(orth_hip_step_t, step, free_count, STEP)
    TRY64(orth_hip_step_t, step, tokens, STEP)
    TRY32(orth_hip_step_t, step, page_size, STEP)
#define CACHE orth_paged_attention_hip(&x, &attend, NULL)
    TRY64(orth_hip_cache_t, cache, pages, CACHE)
    TRY64(orth_hip_cache_t, cache, k_strides[0], CACHE)
    TRY64(orth_hip_cache_t, cache, v_strides[2], CACHE)
    TRY32(orth_hip_cache_t, cache, dtype, CACHE)
    TRY32(orth_hip_cache_t, cache, page_size, CACHE)
    TRY32(orth_hip_cache_t, cache, kv_heads, CACHE)
    TRY32(orth_hip_cache_t, cache, head_dim, CACHE)
#define APPEND orth_cache_append_hip(&cache, &x, NULL)
    TRY64(orth_hip_append_t, append, tokens, APPEND)
    TRY64(orth_hip_append_t, append, cos_sin_rows, APPEND)
    TRY64(orth_hip_append_t, append, q_strides[0], APPEND)
    TRY64(orth_hip_append_t, append, q_out_strides[1], APPEND)
    TRY64(orth_hip_append_t, append, k_strides[0], APPEND)
    TRY32(orth_hip_append_t, append, q_heads, APPEND)
    TRY32(orth_hip_append_t, append, rot, APPEND)
#define ATTEND orth_paged_attention_hip(&cache, &x, NULL)
    TRY64(orth_hip_attend_t, attend, tokens, ATTEND)
    TRY64(orth_hip_attend_t, attend, table_rows, ATTEND)
    TRY64(orth_hip_attend_t, attend, table_width, ATTEND)
    TRY64(orth_hip_attend_t, attend, table_stride, ATTEND)
    TRY64(orth_hip_attend_t, attend, out_strides[0], ATTEND)
    TRY64(orth_hip_attend_t, attend, out_strides[1], ATTEND)
    TRY32(orth_hip_attend_t, attend, q_heads, ATTEND)
    TRY32(orth_hip_attend_t, attend, window, ATTEND)
#define ADAPTER orth_adapter_add_hip(&x, NULL)
    TRY64(orth_hip_adapter_t, adapter, tokens, ADAPTER)
    TRY64(orth_hip_adapter_t, adapter, in_features, ADAPTER)
    TRY64(orth_hip_adapter_t, adapter, out_features, ADAPTER)
    TRY64(orth_hip_adapter_t, adapter, count, ADAPTER)
    TRY64(orth_hip_adapter_t, adapter, x_stride, ADAPTER)
    TRY64(orth_hip_adapter_t, adapter, out_stride, ADAPTER)
    TRY32(orth_hip_adapter_t, adapter, rank, ADAPTER)
    TRY32(orth_hip_adapter_t, adapter, dtype, ADAPTER)
    {
        orth_hip_attend_t x = attend;
        x.scale = NAN;
        expect("scale", orth_paged_attention_hip(&cache, &x, NULL), ORTH_ERR_INVALID_ARGUMENT, ORTH_ERR_INVALID_ARGUMENT);
    }
    expect("null", orth_page_step_hip(NULL, NULL), ORTH_ERR_INVALID_ARGUMENT, ORTH_ERR_INVALID_ARGUMENT);
    expect("null", orth_paged_attention_hip(NULL, &attend, NULL), ORTH_ERR_INVALID_ARGUMENT, ORTH_ERR_INVALID_ARGUMENT);
    expect("null", orth_adapter_add_hip(NULL, NULL), ORTH_ERR_INVALID_ARGUMENT, ORTH_ERR_INVALID_ARGUMENT);
    if (failures) return 1;
    printf("serve ok\n");
    return 0;
}
