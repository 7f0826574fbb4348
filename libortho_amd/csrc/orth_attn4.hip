// Attention of single tokens over the cache in 4 bits.
#include "orth_serve4.h"

namespace orth {

namespace {

struct Attend4Args {
    orth_hip_int4_cache_t c;
    orth_hip_attend_t a;
    int W, bf;
    float scale2;  // scale * log2(e)
};

// A wave per token and query head: 64 keys at a time, a lane a key's score,
// then a lane up to four elements of the output.
__global__ __launch_bounds__(64) void attend4_kernel(Attend4Args g) {
    __shared__ float q[256], weight[64];
    __shared__ int64_t place[64];  // page * page_size + slot of a chunk's keys, -1: not seen
    const int lane = threadIdx.x, D = g.c.head_dim;
    const int64_t t = blockIdx.x / (unsigned)g.a.q_heads, h = blockIdx.x - t * g.a.q_heads, kvh = h / (g.a.q_heads / g.c.kv_heads);
    const uint16_t *src = (const uint16_t *)g.a.q + t * g.a.q_strides[0] + h * g.a.q_strides[1];
    for (int d = lane; d < D; d += 64) q[d] = g.bf ? load16<true>(src[d]) : load16<false>(src[d]);
    const int64_t row = g.a.rows ? (int64_t)g.a.rows[t] : t;
    int64_t end = (int64_t)g.a.positions[t] + 1;
    const int64_t begin = g.a.window > 0 && end > g.a.window ? end - g.a.window : 0, held = g.a.table_width * g.c.page_size;
    end = row < 0 || row >= g.a.table_rows ? 0 : end < held ? end : held;
    const uint8_t *kc = (const uint8_t *)g.c.k_codes + kvh * g.c.k_code_strides[2], *vc = (const uint8_t *)g.c.v_codes + kvh * g.c.v_code_strides[2];
    const uint16_t *ks = (const uint16_t *)g.c.k_scales + kvh * g.c.k_scale_strides[2], *vs = (const uint16_t *)g.c.v_scales + kvh * g.c.v_scale_strides[2];
    float m = -__builtin_inff(), l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    __syncthreads();
    for (int64_t j0 = begin; j0 < end; j0 += 64) {
        const int64_t j = j0 + lane;
        int64_t pg = -1, in = 0;
        if (j < end) {
            pg = g.a.block_table[row * g.a.table_stride + j / g.c.page_size];
            in = j % g.c.page_size;
        }
        const bool seen = pg >= 0 && pg < g.c.pages;
        float x = -__builtin_inff();
        if (seen) {
            const uint8_t *c = kc + pg * g.c.k_code_strides[0] + in * g.c.k_code_strides[1];
            const uint16_t *s = ks + pg * g.c.k_scale_strides[0] + in * g.c.k_scale_strides[1];
            float sum = 0.f;
            for (int d = 0; d < D; d++) {
                const int b = c[d % 16 * g.W + d / 32], k = d / g.c.group_size;
                sum += q[d] * fmaf((float)(d & 16 ? b >> 4 : b & 15), load16<false>(s[2 * k]), load16<false>(s[2 * k + 1]));
            }
            x = sum * g.scale2;
        }
        float top = x;
        for (int d = 32; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
        if (!__any(seen)) continue;
        top = fmaxf(fmaxf(top, -3.0e38f), m);
        const float keep = exp2f(m - top), p = seen ? exp2f(x - top) : 0.f;
        m = top;
        l = l * keep + p;
        weight[lane] = p;
        place[lane] = seen ? pg * g.c.page_size + in : -1;
        __syncthreads();
        for (int e = 0; e < 4; e++) {
            const int d = lane + 64 * e;
            o[e] *= keep;
            if (d >= D) continue;
            const int at = d % 16 * g.W + d / 32, k = d / g.c.group_size;
            for (int i = 0; i < 64; i++) {
                if (place[i] < 0) continue;
                const int64_t p2 = place[i] / g.c.page_size, i2 = place[i] - p2 * g.c.page_size;
                const int b = vc[p2 * g.c.v_code_strides[0] + i2 * g.c.v_code_strides[1] + at];
                const uint16_t *s = vs + p2 * g.c.v_scale_strides[0] + i2 * g.c.v_scale_strides[1] + 2 * k;
                o[e] += weight[i] * fmaf((float)(d & 16 ? b >> 4 : b & 15), load16<false>(s[0]), load16<false>(s[1]));
            }
        }
        __syncthreads();
    }
    for (int d = 32; d > 0; d >>= 1) l += __shfl_xor(l, d, 64);
    uint16_t *out = (uint16_t *)g.a.out + t * g.a.out_strides[0] + h * g.a.out_strides[1];
    for (int e = 0; e < 4; e++) {
        const int d = lane + 64 * e;
        const float v = l == 0.f ? 0.f : o[e] / l;
        if (d < D) out[d] = g.bf ? store16<true>(v) : store16<false>(v);
    }
}

}  // namespace

int64_t attention4_workspace_bytes(const orth_hip_int4_cache_t &, const orth_hip_attend_t &, int, int64_t *groups) {
    *groups = 0;
    return 0;
}

hipError_t launch_paged_attention4(const orth_hip_int4_cache_t &c, const orth_hip_attend_t &a, int32_t dtype, int,
                                   void *, uint32_t *, hipStream_t stream) {
    Attend4Args g;
    g.c = c;
    g.a = a;
    g.W = ORTH_INT4_ROW_BYTES(c.head_dim) / 16;
    g.bf = dtype == ORTH_DT_BF16;
    g.scale2 = a.scale * 1.4426950408889634f;
    attend4_kernel<<<dim3((unsigned)(a.tokens * a.q_heads)), 64, 0, stream>>>(g);
    return hipGetLastError();
}

}  // namespace orth
