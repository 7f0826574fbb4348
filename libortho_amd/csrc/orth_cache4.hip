// The cache in 4 bits: quantising the new tokens' keys and values as they are
// written, and reading slots back in 16 bits.
#include "orth_serve4.h"

namespace orth {

namespace {

constexpr int64_t kLaunch = 1 << 23;  // workgroups of 256 along x (2^32 threads there run another number, without an error)

struct Append4Args {
    orth_hip_int4_cache_t c;
    orth_hip_append_t a;
    FastDiv page;
    int bf;
};

__device__ __forceinline__ float load_vec16(const uint16_t *p, int bf) {
    return bf ? load16<true>(*p) : load16<false>(*p);
}

// Through FP32, as torch and numpy round a 64-bit number to FP16.  (The empty
// asm keeps the two roundings apart: folded into one they differ in a tie, and
// the one is some thirty integer operations.)
__device__ __forceinline__ f16 half_of(double v) {
    float f = (float)v;
    asm("" : "+v"(f));
    return (f16)f;
}

// The least value of the 16 lanes that share a vector (rotations within a row of lanes).
__device__ __forceinline__ float row_min(float v) {
    v = fminf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x128, 0xf, 0xf, true)));
    v = fminf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x124, 0xf, 0xf, true)));
    v = fminf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x122, 0xf, 0xf, true)));
    return fminf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x121, 0xf, 0xf, true)));
}

// 16 lanes a vector: lane r holds elements 16 i + r, the nibbles of its unit.
template <int W, int GS>
__global__ __launch_bounds__(256) void cache_append4_kernel(Append4Args g) {
    constexpr int NE = 2 * W, NG = W / GS;
    const int64_t t = blockIdx.x;
    const int r = threadIdx.x & 15, D = g.c.head_dim, rot = g.a.rot, half = rot / 2;
    const int64_t slot = g.a.slots[t];
    bool write = slot >= 0 && slot < g.c.pages * g.c.page_size, placed = true;
    const float *cs = nullptr;
    if (g.a.cos_sin) {
        const int64_t pos = g.a.positions[t];
        placed = pos >= 0 && pos < g.a.cos_sin_rows;
        write = write && placed;
        if (placed) cs = g.a.cos_sin + pos * rot;
    }
    int64_t pg = 0, in = 0;
    if (write) {
        pg = slot <= INT32_MAX ? (int64_t)quotient((uint32_t)slot, g.page) : slot / g.c.page_size;
        in = slot - pg * g.c.page_size;
    }
    const int H = g.a.q ? g.a.q_heads : 0, G = g.c.kv_heads, all = H + 2 * G;
    // (every lane of a wave takes the same number of turns: lanes of a vector reduce together)
    for (int h0 = blockIdx.y * 16; h0 < all; h0 += gridDim.y * 16) {
        const int h = h0 + (int)(threadIdx.x >> 4);
        const bool is_q = h < H, is_k = !is_q && h < H + G, here = h < all;
        const uint16_t *src = nullptr;
        if (is_q) src = (const uint16_t *)g.a.q + t * g.a.q_strides[0] + h * g.a.q_strides[1];
        else if (is_k) src = (const uint16_t *)g.a.k + t * g.a.k_strides[0] + (h - H) * g.a.k_strides[1];
        else if (here) src = (const uint16_t *)g.a.v + t * g.a.v_strides[0] + (h - H - G) * g.a.v_strides[1];
        if (is_q) {
            uint16_t *dst = (uint16_t *)g.a.q_out + t * g.a.q_out_strides[0] + h * g.a.q_out_strides[1];
            float y[NE];
#pragma unroll
            for (int i = 0; i < NE; i++) {
                const int d = 16 * i + r;
                y[i] = 0.f;
                if (d >= D || !placed) continue;
                y[i] = load_vec16(src + d, g.bf);
                if (d >= rot) continue;
                const bool first = g.a.interleaved ? !(d & 1) : d < half;
                const int pd = g.a.interleaved ? d ^ 1 : first ? d + half : d - half, ci = g.a.interleaved ? d >> 1 : first ? d : d - half;
                const float w = load_vec16(src + pd, g.bf), c = cs[ci], s = cs[half + ci];
                y[i] = first ? y[i] * c - w * s : y[i] * c + w * s;
            }
            // (q_out may be q: every element of the vector is read before one is written)
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
            for (int i = 0; i < NE; i++)
                if (16 * i + r < D) dst[16 * i + r] = g.bf ? store16<true>(y[i]) : store16<false>(y[i]);
        }
        const bool kv = here && !is_q && write;
        float x[NE];
        float low[NG], high[NG];
        uint32_t odd = 0;  // groups with an element that is not finite
#pragma unroll
        for (int i = 0; i < NG; i++) low[i] = high[i] = __builtin_inff();
#pragma unroll
        for (int i = 0; i < NE; i++) {
            const int d = 16 * i + r;
            x[i] = 0.f;
            if (!kv || d >= D) continue;
            double v = load_vec16(src + d, g.bf);
            if (is_k && d < rot) {
                const bool first = g.a.interleaved ? !(d & 1) : d < half;
                const int pd = g.a.interleaved ? d ^ 1 : first ? d + half : d - half, ci = g.a.interleaved ? d >> 1 : first ? d : d - half;
                const double w = load_vec16(src + pd, g.bf), c = cs[ci], s = cs[half + ci];
                v = first ? v * c - w * s : v * c + w * s;
            }
            if (!(fabs(v) < __builtin_inf())) odd |= 1u << (i / (2 * GS));
            v = v > 65504.0 ? 65504.0 : v < -65504.0 ? -65504.0 : v;
            x[i] = (float)half_of(v);
            low[i / (2 * GS)] = fminf(low[i / (2 * GS)], x[i]);
            high[i / (2 * GS)] = fminf(high[i / (2 * GS)], -x[i]);
        }
        uint32_t code[W];
#pragma unroll
        for (int b = 0; b < W; b++) code[b] = 0;
        uint32_t pair[NG];
#pragma unroll
        for (int k = 0; k < NG; k++) {
            const float lo = row_min(low[k]), hi = -row_min(high[k]);
            f16 s = half_of(((double)hi - lo) / 15.0);
            if ((double)lo + 15.0 * (double)(float)s > 65504.0) s = __builtin_bit_cast(f16, (uint16_t)(__builtin_bit_cast(uint16_t, s) - 1));
            const double inv = 1.0 / (double)(float)s;
            const bool flat = !((float)s > 0.f), nan = ((__ballot(odd >> k & 1) >> (threadIdx.x & 48)) & 0xffff) != 0;
            pair[k] = nan ? 0x7e007e00u : (uint32_t)__builtin_bit_cast(uint16_t, s) | (uint32_t)__builtin_bit_cast(uint16_t, (f16)lo) << 16;
#pragma unroll
            for (int j = 0; j < 2 * GS; j++) {
                const int i = 2 * GS * k + j;
                // (x - low is exact, and so far from a half that a quotient is
                // not one: 2^-42 sends exact halves up and moves nothing else)
                int u = flat ? 0 : (int)floor(((double)x[i] - lo) * inv + (0.5 + 0x1p-42));
                u = u < 0 ? 0 : u > 15 ? 15 : u;
                if (nan || 16 * i + r >= D) u = 0;
                code[i / 2] |= (uint32_t)u << (i & 1 ? 4 : 0);
            }
        }
        if (kv) {
            const int64_t head = is_k ? h - H : h - H - G;
            const int64_t *st = is_k ? g.c.k_code_strides : g.c.v_code_strides, *ss = is_k ? g.c.k_scale_strides : g.c.v_scale_strides;
            uint8_t *row = (uint8_t *)(is_k ? g.c.k_codes : g.c.v_codes) + pg * st[0] + in * st[1] + head * st[2];
            uint16_t *sc = (uint16_t *)(is_k ? g.c.k_scales : g.c.v_scales) + pg * ss[0] + in * ss[1] + head * ss[2];
#pragma unroll
            for (int b = 0; b < W; b++) row[r * W + b] = (uint8_t)code[b];
            const int groups = D / g.c.group_size;
#pragma unroll
            for (int k = 0; k < NG; k++)
                if (r == k && k < groups) reinterpret_cast<uint32_t *>(sc)[k] = pair[k];
        }
    }
}

struct Read4Args {
    orth_hip_int4_cache_t c;
    orth_hip_read_t r;
    int W, bf;
};

// A thread eight elements of a vector.
__global__ __launch_bounds__(256) void cache_read4_kernel(Read4Args g) {
    const int chunks = g.c.head_dim / 8;
    const int64_t each = 2 * (int64_t)g.c.kv_heads * chunks;
    for (int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x; x < g.r.count * each; x += (int64_t)gridDim.x * 256) {
        const int64_t i = x / each;
        const int in_slot = (int)(x - i * each), vec = in_slot / chunks, d = (in_slot - vec * chunks) * 8;
        const bool is_v = vec >= g.c.kv_heads;
        const int64_t head = is_v ? vec - g.c.kv_heads : vec, slot = g.r.slots[i];
        const bool here = slot >= 0 && slot < g.c.pages * g.c.page_size;
        const int64_t pg = here ? slot / g.c.page_size : 0, in = here ? slot - pg * g.c.page_size : 0;
        const int64_t *st = is_v ? g.c.v_code_strides : g.c.k_code_strides, *ss = is_v ? g.c.v_scale_strides : g.c.k_scale_strides;
        const uint8_t *row = (const uint8_t *)(is_v ? g.c.v_codes : g.c.k_codes) + pg * st[0] + in * st[1] + head * st[2];
        const uint16_t *sc = (const uint16_t *)(is_v ? g.c.v_scales : g.c.k_scales) + pg * ss[0] + in * ss[1] + head * ss[2];
        const int64_t *so = is_v ? g.r.v_strides : g.r.k_strides;
        uint16_t *out = (uint16_t *)(is_v ? g.r.v_out : g.r.k_out) + i * so[0] + head * so[1] + d;
        const int k = d / g.c.group_size;
        const float scale = load16<false>(sc[2 * k]), low = load16<false>(sc[2 * k + 1]);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const uint8_t b = row[(d % 16 + e) * g.W + d / 32];
            const float v = here ? fmaf((float)(d & 16 ? b >> 4 : b & 15), scale, low) : 0.f;
            out[e] = g.bf ? store16<true>(v) : store16<false>(v);
        }
    }
}

}  // namespace

hipError_t launch_cache_append4(const orth_hip_int4_cache_t &c, const orth_hip_append_t &a, int32_t dtype, int cus,
                                hipStream_t stream) {
    Append4Args g;
    g.c = c;
    g.a = a;
    if (!a.cos_sin) g.a.rot = 0;
    g.page = fast_div((uint32_t)c.page_size);
    g.bf = dtype == ORTH_DT_BF16;
    const int64_t heads = (a.q ? (int64_t)a.q_heads : 0) + 2 * (int64_t)c.kv_heads, parts = (heads + 15) / 16;
    const int y = a.tokens >= 2 * cus ? 1 : (int)(parts < 65535 ? parts : 65535);
    for (int64_t t = 0; t < a.tokens; t += kLaunch) {
        const dim3 grid((unsigned)(a.tokens - t < kLaunch ? a.tokens - t : kLaunch), (unsigned)y);
        const hipError_t e = by_int4_layout(c, [&](auto unit, auto steps) -> hipError_t {
            cache_append4_kernel<unit.value, steps.value><<<grid, 256, 0, stream>>>(g);
            return hipGetLastError();
        });
        if (e != hipSuccess) return e;
        if (a.q) {
            g.a.q = (const uint16_t *)g.a.q + kLaunch * a.q_strides[0];
            g.a.q_out = (uint16_t *)g.a.q_out + kLaunch * a.q_out_strides[0];
        }
        g.a.k = (const uint16_t *)g.a.k + kLaunch * a.k_strides[0];
        g.a.v = (const uint16_t *)g.a.v + kLaunch * a.v_strides[0];
        g.a.slots += kLaunch;
        if (a.cos_sin) g.a.positions += kLaunch;
    }
    return hipSuccess;
}

hipError_t launch_cache_read4(const orth_hip_int4_cache_t &c, const orth_hip_read_t &r, int32_t dtype, int cus,
                              hipStream_t stream) {
    Read4Args g;
    g.c = c;
    g.r = r;
    g.W = ORTH_INT4_ROW_BYTES(c.head_dim) / 16;
    g.bf = dtype == ORTH_DT_BF16;
    const int64_t groups = (r.count * (2 * (int64_t)c.kv_heads * (c.head_dim / 8)) + 255) / 256;
    cache_read4_kernel<<<dim3((unsigned)(groups < 16 * cus ? groups : 16 * cus)), 256, 0, stream>>>(g);
    return hipGetLastError();
}

}  // namespace orth
