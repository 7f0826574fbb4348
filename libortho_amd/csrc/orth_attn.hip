// Attention of single tokens over the paged cache.
#include "orth_serve.h"

namespace orth {

namespace {

// A wave per query head: its lanes hold the head's elements, and the keys go
// by one at a time through a running maximum and sum.
template <bool BF>
__global__ __launch_bounds__(64) void paged_attention_kernel(orth_hip_cache_t c, orth_hip_attend_t a, FastDiv page) {
    const int64_t t = blockIdx.x;
    const int h = blockIdx.y, lane = threadIdx.x, D = c.head_dim;
    const int64_t kh = h / (a.q_heads / c.kv_heads);
    const uint16_t *q = (const uint16_t *)a.q + t * a.q_strides[0] + h * a.q_strides[1];
    uint16_t *out = (uint16_t *)a.out + t * a.out_strides[0] + h * a.out_strides[1];
    const int64_t row = a.rows ? a.rows[t] : t;
    int64_t end = (int64_t)a.positions[t] + 1;
    if (row < 0 || row >= a.table_rows) end = 0;
    int64_t begin = a.window > 0 && end > a.window ? end - a.window : 0;
    const int64_t held = a.table_width * c.page_size;
    end = end > held ? held : end;
    float qv[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -__builtin_inff(), l = 0.f;
    int64_t seen = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) qv[i] = lane + 64 * i < D ? load16<BF>(q[lane + 64 * i]) : 0.f;
    for (int64_t j = begin; j < end; j++) {
        const int64_t at = quotient((uint32_t)j, page), p = a.block_table[row * a.table_stride + at];
        if (p < 0 || p >= c.pages) continue;
        seen++;
        const int64_t in = j - at * c.page_size;
        const uint16_t *k = (const uint16_t *)c.k_cache + p * c.k_strides[0] + in * c.k_strides[1] + kh * c.k_strides[2];
        const uint16_t *v = (const uint16_t *)c.v_cache + p * c.v_strides[0] + in * c.v_strides[1] + kh * c.v_strides[2];
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (lane + 64 * i < D) s += qv[i] * load16<BF>(k[lane + 64 * i]);
        s = wave_sum(s) * a.scale;
        const float top = fmaxf(m, s), base = top == -__builtin_inff() ? 0.f : top;
        const float keep = __expf(m - base), w = __expf(s - base);
        l = l * keep + w;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            o[i] *= keep;
            if (lane + 64 * i < D) o[i] += w * load16<BF>(v[lane + 64 * i]);
        }
        m = top;
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (lane + 64 * i < D) out[lane + 64 * i] = store16<BF>(seen ? o[i] / l : 0.f);
}

}  // namespace

int64_t attention_workspace_bytes(const orth_hip_cache_t &, const orth_hip_attend_t &, int) { return 0; }

hipError_t launch_paged_attention(const orth_hip_cache_t &c, const orth_hip_attend_t &a, int, void *, hipStream_t stream) {
    const dim3 grid((unsigned)a.tokens, (unsigned)a.q_heads);
    const FastDiv page = fast_div((uint32_t)c.page_size);
    if (c.dtype == ORTH_DT_BF16) paged_attention_kernel<true><<<grid, 64, 0, stream>>>(c, a, page);
    else paged_attention_kernel<false><<<grid, 64, 0, stream>>>(c, a, page);
    return hipGetLastError();
}

}  // namespace orth
