// The cache in 4 bits: quantising the new tokens' keys and values as they are
// written, and reading slots back in 16 bits.
#include "orth_serve4.h"

namespace orth {

namespace {

constexpr int64_t kLaunch = 1 << 23;  // workgroups of 256 along x (2^32 threads there run another number, without an error)

// ---------------------------------------------------------------- the append
//
// A vector lies across 16 lanes (32 where head_dim > 128), eight neighbouring
// elements a lane, so loads and the queries' stores are 16 bytes wide, the
// half layout's partners are a lane exchange away, and a group is 4, 8 or 16
// lanes (or all of them): its least and greatest value meet in as many steps.
// The codes' layout wants one byte of eight units from a lane, so eight lanes
// exchange nibbles in three steps and hold a unit each.
//
// What is quantised has to be the FP16 number nearest to the turned key, and a
// code the one nearest to the quotient: a last place of difference moves a
// code by a whole step.  FP32 decides all but the numbers next to a border,
// and 64 bits those (one key in some 800, one code in some 30,000).
//
// Memory-bound: an element is read once and, of keys and values, a quarter of
// it written.
struct Append4Args {
    orth_hip_int4_cache_t c;
    orth_hip_append_t a;
    FastDiv page;
    int W, bf;
    int group_lanes;  // lanes that share a group
    int vec;          // vectors are 16-byte aligned
};

// Through FP32, as torch and numpy round a 64-bit number to FP16.  (The empty
// asm keeps the two roundings apart: folded into one they differ in a tie, and
// the one is some thirty integer operations.)
__device__ __forceinline__ f16 half_of(double v) {
    float f = (float)v;
    asm("" : "+v"(f));
    return (f16)f;
}

// The value of lane ^ X.
template <int X>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v) {
    if constexpr (X == 1) return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xb1, 0xf, 0xf, true);
    else if constexpr (X == 2) return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4e, 0xf, 0xf, true);
    else if constexpr (X == 8) return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x128, 0xf, 0xf, true);
    else return (uint32_t)__builtin_amdgcn_ds_swizzle((int)v, X << 10 | 0x1f);
}
template <int X>
__device__ __forceinline__ float least_with(float v) {
    return fminf(v, __uint_as_float(lane_xor<X>(__float_as_uint(v))));
}

// One step of the exchange of nibbles: lanes that differ in X keep the half of
// each pair of 4 S bits that is theirs.
template <int X, int S>
__device__ __forceinline__ uint32_t exchange(uint32_t v, uint32_t keep) {
    const bool high = (threadIdx.x & X) != 0;
    const uint32_t o = lane_xor<X>(v);
    // (keep: the low one of each two fields of S nibbles)
    return high ? (v & ~keep) | ((o & ~keep) >> (4 * S)) : (v & keep) | ((o & keep) << (4 * S));
}

template <int LP>
__global__ __launch_bounds__(256) void cache_append4_kernel(Append4Args g) {
    constexpr int VECS = 256 / LP;
    const int64_t t = blockIdx.x;
    const int c = threadIdx.x % LP, d0 = 8 * c, D = g.c.head_dim, rot = g.a.rot, half = rot / 2;
    const int64_t slot = g.a.slots[t];
    bool write = slot >= 0 && slot < g.c.pages * g.c.page_size, placed = true;
    // this lane's cosines and sines, and whether its elements are turned, are
    // the first of their pairs, and find their partners in one other lane
    float cs[8], sn[8];
    const bool inter = g.a.interleaved != 0, aligned_half = inter || half % 8 == 0;
    int64_t pos = 0;
    if (g.a.cos_sin) {
        pos = g.a.positions[t];
        placed = pos >= 0 && pos < g.a.cos_sin_rows;
        write = write && placed;
    }
    const bool turns = d0 < rot && placed;
    const float *table = g.a.cos_sin + pos * rot;
    if (turns) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int d = d0 + e, ci = d >= rot ? 0 : inter ? d >> 1 : d < half ? d : d - half;
            cs[e] = d < rot ? table[ci] : 1.f;
            sn[e] = d < rot ? table[half + ci] : 0.f;
            if (d < rot && (inter ? !(d & 1) : d < half)) sn[e] = -sn[e];  // (a, b) -> a c - b s, b c + a s
        }
    }
    int64_t pg = 0, in = 0;
    if (write) {
        pg = slot <= INT32_MAX ? (int64_t)quotient((uint32_t)slot, g.page) : slot / g.c.page_size;
        in = slot - pg * g.c.page_size;
    }
    const int partner_lane = (int)(threadIdx.x & 63) + (d0 < half ? half / 8 : -(half / 8));
    const int H = g.a.q ? g.a.q_heads : 0, G = g.c.kv_heads, all = H + 2 * G;
    // (every lane of a wave takes the same number of turns: lanes of a vector work together)
    for (int h0 = blockIdx.y * VECS; h0 < all; h0 += gridDim.y * VECS) {
        const int h = h0 + (int)(threadIdx.x / LP);
        const bool is_q = h < H, is_k = !is_q && h < H + G, here = h < all && d0 < D;
        const uint16_t *src = nullptr;
        if (is_q) src = (const uint16_t *)g.a.q + t * g.a.q_strides[0] + h * g.a.q_strides[1];
        else if (is_k) src = (const uint16_t *)g.a.k + t * g.a.k_strides[0] + (h - H) * g.a.k_strides[1];
        else src = (const uint16_t *)g.a.v + t * g.a.v_strides[0] + (h - H - G) * g.a.v_strides[1];
        u32x4 raw = {0u, 0u, 0u, 0u};
        if (here && (is_q ? placed : write)) {
            if (g.vec) {
                raw = *reinterpret_cast<const u32x4 *>(src + d0);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) raw[e] = (uint32_t)src[d0 + 2 * e] | (uint32_t)src[d0 + 2 * e + 1] << 16;
            }
        }
        auto value = [&](const u32x4 &w, int e) -> float {
            const uint32_t b = w[e >> 1];
            return g.bf ? __uint_as_float(e & 1 ? b & 0xffff0000u : b << 16) : load16<false>((uint16_t)(e & 1 ? b >> 16 : b));
        };
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = value(raw, e);
        const bool turn = turns && (is_q || is_k);
        // partners: of the same place in another lane, or the neighbouring element
        float w[8];
        if (inter) {
#pragma unroll
            for (int e = 0; e < 8; e++) w[e] = x[e ^ 1];
        } else if (aligned_half) {
            u32x4 o;
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = (uint32_t)__builtin_amdgcn_ds_bpermute(partner_lane * 4, (int)raw[e]);
#pragma unroll
            for (int e = 0; e < 8; e++) w[e] = value(o, e);
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int d = d0 + e, pd = d < half ? d + half : d - half;
                w[e] = 0.f;
                if (turn && here && d < rot && (is_q || write)) w[e] = g.bf ? load16<true>(src[pd]) : load16<false>(src[pd]);
            }
        }
        if (is_q) {
            if (turn)
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (d0 + e < rot) x[e] = x[e] * cs[e] + w[e] * sn[e];
            // (q_out may be q: all lanes have read the vector before one writes it)
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            if (here) {
                uint16_t *dst = (uint16_t *)g.a.q_out + t * g.a.q_out_strides[0] + h * g.a.q_out_strides[1] + d0;
                uint16_t y[8];
#pragma unroll
                for (int e = 0; e < 8; e++) y[e] = g.bf ? store16<true>(x[e]) : store16<false>(x[e]);
                if (g.vec) {
                    u32x4 v;
#pragma unroll
                    for (int e = 0; e < 4; e++) v[e] = (uint32_t)y[2 * e] | (uint32_t)y[2 * e + 1] << 16;
                    *reinterpret_cast<u32x4 *>(dst) = v;
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++) dst[e] = y[e];
                }
            }
        }
        if (__all(is_q)) continue;
        const bool kv = h < all && !is_q && write;

        bool odd = false;  // an element is not finite
#pragma unroll
        for (int e = 0; e < 8; e++) {
            float v = x[e];
            if (is_k && turn && d0 + e < rot) {
                // x c + w s: the product's error comes back in a second fused
                // step, so f is within two last places of FP32
                const float p = w[e] * sn[e], f = fmaf(x[e], cs[e], p) + fmaf(w[e], sn[e], -p);
                const uint32_t b = __float_as_uint(f), a = b & 0x7fffffffu;
                v = f;
                // next to a border of FP16 numbers (a low part of 0x1000), or
                // below the normal ones, or too large
                if (((b + 4 - 0x1000) & 0x1fff) <= 8 || a < 0x38800000u || a > 0x47000000u) {
                    double y = (double)x[e] * cs[e] + (double)w[e] * sn[e];
                    y = y > 65504.0 ? 65504.0 : y < -65504.0 ? -65504.0 : y;
                    const bool finite = fabs((double)x[e]) < __builtin_inf() && fabs((double)w[e]) < __builtin_inf() &&
                                        fabsf(cs[e]) < __builtin_inff() && fabsf(sn[e]) < __builtin_inff();
                    v = finite ? (float)half_of(y) : __builtin_nanf("");
                }
            }
            odd |= !(fabsf(v) < __builtin_inff());
            v = v > 65504.f ? 65504.f : v < -65504.f ? -65504.f : v;
            x[e] = (float)(f16)v;
        }
        float lo = __builtin_inff(), hi = __builtin_inff();  // hi: of the negated elements
        if (here) {
#pragma unroll
            for (int e = 0; e < 8; e++) lo = fminf(lo, x[e]), hi = fminf(hi, -x[e]);
        }
        lo = least_with<2>(least_with<1>(lo)), hi = least_with<2>(least_with<1>(hi));
        if (g.group_lanes > 4) lo = least_with<4>(lo), hi = least_with<4>(hi);
        if (g.group_lanes > 8) lo = least_with<8>(lo), hi = least_with<8>(hi);
        if (LP == 32 && g.group_lanes > 16) lo = least_with<16>(lo), hi = least_with<16>(hi);
        hi = -hi;
        const uint64_t odd_lanes = __ballot(odd && here) >> (threadIdx.x & 63 & ~(g.group_lanes - 1));
        const bool nan = (odd_lanes & ((1ull << g.group_lanes) - 1)) != 0;
        // (hi - lo) / 15 in 64 bits: a product with the reciprocal, and its remainder's
        const double range = (double)hi - (double)lo, third = range * (1.0 / 15.0);
        f16 s = half_of(fma(fma(-15.0, third, range), 1.0 / 15.0, third));
        if ((double)lo + 15.0 * (double)(float)s > 65504.0) s = __builtin_bit_cast(f16, (uint16_t)(__builtin_bit_cast(uint16_t, s) - 1));
        const float scale = (float)s, inv = __builtin_amdgcn_rcpf(scale);
        const bool flat = !(scale > 0.f) || nan || !here;
        uint32_t nibbles = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            // (x - lo) / scale + 1/2, off by 2^-17 at the most
            float y = fmaf(x[e] - lo, inv, 0.5f);
            int u = (int)y;
            const float part = y - (float)u;
            if ((part < 0x1p-16f || part > 1.f - 0x1p-16f) && !flat) {
                // the difference is exact, and so far from a half that a quotient
                // is not one: 2^-42 sends exact halves up and moves nothing else
                u = (int)floor(((double)x[e] - (double)lo) / (double)scale + (0.5 + 0x1p-42));
            }
            u = u < 0 ? 0 : u > 15 ? 15 : u;
            nibbles |= (flat ? 0u : (uint32_t)u) << (4 * e);
        }
        // lanes c, c ^ 2, c ^ 4, c ^ 8 hold eight units' nibbles each: now a unit's eight
        nibbles = exchange<2, 1>(nibbles, 0x0f0f0f0fu);
        nibbles = exchange<4, 2>(nibbles, 0x00ff00ffu);
        nibbles = exchange<8, 4>(nibbles, 0x0000ffffu);
        if (kv) {
            const int64_t head = is_k ? h - H : h - H - G;
            const int64_t *st = is_k ? g.c.k_code_strides : g.c.v_code_strides, *ss = is_k ? g.c.k_scale_strides : g.c.v_scale_strides;
            const int unit = (c & 1) * 8 + (c >> 1 & 7);
            uint8_t *row = (uint8_t *)(is_k ? g.c.k_codes : g.c.v_codes) + pg * st[0] + in * st[1] + head * st[2] + unit * g.W;
            if (g.W == 4) *reinterpret_cast<uint32_t *>(row) = nibbles;
            else if (g.W == 2) *reinterpret_cast<uint16_t *>(row) = (uint16_t)nibbles;
            else if (g.W == 8) *reinterpret_cast<uint32_t *>(row + (c >> 4) * 4) = nibbles;
            else row[0] = (uint8_t)nibbles, row[1] = (uint8_t)(nibbles >> 8), row[2] = (uint8_t)(nibbles >> 16);
            if (here && (c & (g.group_lanes - 1)) == 0) {
                uint16_t *sc = (uint16_t *)(is_k ? g.c.k_scales : g.c.v_scales) + pg * ss[0] + in * ss[1] + head * ss[2];
                reinterpret_cast<uint32_t *>(sc)[c / g.group_lanes] =
                    nan ? 0x7e007e00u : (uint32_t)__builtin_bit_cast(uint16_t, s) | (uint32_t)__builtin_bit_cast(uint16_t, (f16)lo) << 16;
            }
        }
    }
}

// ------------------------------------------------------------------ the read
//
// A thread eight neighbouring elements: they are one nibble (h) of one byte
// (b) of eight units, whose 8 W bytes the threads of a vector share in the L1.
// Memory-bound: codes and scales read once, 16-byte stores.
struct Read4Args {
    orth_hip_int4_cache_t c;
    orth_hip_read_t r;
    FastDiv page, each, chunks;  // each: threads of a slot, chunks: of a vector
    int group_shift;             // of eight elements: 31 where the whole vector is one group
    int bf, vec;
};

template <int W>
__global__ __launch_bounds__(256) void cache_read4_kernel(Read4Args g) {
    const uint32_t x = blockIdx.x * 256u + threadIdx.x;
    const uint32_t i = quotient(x, g.each);
    if ((int64_t)i >= g.r.count) return;
    const uint32_t in_slot = x - i * g.each.d, vec = quotient(in_slot, g.chunks), c = in_slot - vec * g.chunks.d;
    const bool is_v = vec >= (uint32_t)g.c.kv_heads;
    const int64_t head = is_v ? vec - g.c.kv_heads : vec, slot = g.r.slots[i];
    const bool here = slot >= 0 && slot < g.c.pages * g.c.page_size;
    const int64_t pg = !here ? 0 : slot <= INT32_MAX ? (int64_t)quotient((uint32_t)slot, g.page) : slot / g.c.page_size;
    const int64_t in = here ? slot - pg * g.c.page_size : 0;
    const int64_t *st = is_v ? g.c.v_code_strides : g.c.k_code_strides, *ss = is_v ? g.c.v_scale_strides : g.c.k_scale_strides;
    const int b = c >> 2, shift = c & 2 ? 4 : 0;
    const uint8_t *row = (const uint8_t *)(is_v ? g.c.v_codes : g.c.k_codes) + pg * st[0] + in * st[1] + head * st[2] + (c & 1) * 8 * W;
    const uint32_t pair = reinterpret_cast<const uint32_t *>((const uint16_t *)(is_v ? g.c.v_scales : g.c.k_scales) + pg * ss[0] + in * ss[1] + head * ss[2])[c >> g.group_shift];
    uint32_t u[8];
    if constexpr (W == 4) {
        const u32x4 lo = reinterpret_cast<const u32x4 *>(row)[0], hi = reinterpret_cast<const u32x4 *>(row)[1];
#pragma unroll
        for (int e = 0; e < 8; e++) u[e] = (e < 4 ? lo[e & 3] : hi[e & 3]) >> (8 * b + shift);
    } else if constexpr (W == 2) {
        const u32x4 v = *reinterpret_cast<const u32x4 *>(row);
#pragma unroll
        for (int e = 0; e < 8; e++) u[e] = v[e >> 1] >> (16 * (e & 1) + 8 * b + shift);
    } else if constexpr (W == 8) {
#pragma unroll
        for (int e = 0; e < 8; e++) u[e] = reinterpret_cast<const uint32_t *>(row)[2 * e + (b >> 2)] >> (8 * (b & 3) + shift);
    } else {
        uint32_t v[7];
#pragma unroll
        for (int e = 0; e < 6; e++) v[e] = reinterpret_cast<const uint32_t *>(row)[e];
        v[6] = 0;
#pragma unroll
        for (int e = 0; e < 6; e++) v[e] = __builtin_amdgcn_alignbyte(v[e + 1], v[e], b);  // from byte b on
#pragma unroll
        for (int e = 0; e < 8; e++) u[e] = v[3 * e / 4] >> (8 * (3 * e % 4) + shift);
    }
    const float scale = load16<false>((uint16_t)pair), low = load16<false>((uint16_t)(pair >> 16));
    const int64_t *so = is_v ? g.r.v_strides : g.r.k_strides;
    uint16_t *out = (uint16_t *)(is_v ? g.r.v_out : g.r.k_out) + i * so[0] + head * so[1] + 8 * c;
    uint16_t y[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float v = here ? fmaf((float)(u[e] & 15), scale, low) : 0.f;
        y[e] = g.bf ? store16<true>(v) : store16<false>(v);
    }
    if (g.vec) {
        u32x4 v;
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = (uint32_t)y[2 * e] | (uint32_t)y[2 * e + 1] << 16;
        *reinterpret_cast<u32x4 *>(out) = v;
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) out[e] = y[e];
    }
}

// Whether vectors from p are 16-byte aligned.
bool wide(const void *p, const int64_t *s) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && s[0] % 8 == 0 && s[1] % 8 == 0;
}

}  // namespace

hipError_t launch_cache_append4(const orth_hip_int4_cache_t &c, const orth_hip_append_t &a, int32_t dtype, int cus,
                                hipStream_t stream) {
    Append4Args g;
    g.c = c;
    g.a = a;
    if (!a.cos_sin) g.a.rot = 0;
    g.page = fast_div((uint32_t)c.page_size);
    g.W = ORTH_INT4_ROW_BYTES(c.head_dim) / 16;
    g.bf = dtype == ORTH_DT_BF16;
    const int lanes = c.head_dim > 128 ? 32 : 16, vecs = 256 / lanes;
    g.group_lanes = c.group_size == c.head_dim ? lanes : c.group_size / 8;
    g.vec = wide(a.k, a.k_strides) && wide(a.v, a.v_strides) && (!a.q || (wide(a.q, a.q_strides) && wide(a.q_out, a.q_out_strides)));
    const int64_t heads = (a.q ? (int64_t)a.q_heads : 0) + 2 * (int64_t)c.kv_heads, parts = (heads + vecs - 1) / vecs;
    // a workgroup for every 16 (or 8) vectors where tokens alone leave CUs
    // idle, else one a token
    const int y = a.tokens >= 2 * cus ? 1 : (int)(parts < 65535 ? parts : 65535);
    for (int64_t t = 0; t < a.tokens; t += kLaunch) {
        const dim3 grid((unsigned)(a.tokens - t < kLaunch ? a.tokens - t : kLaunch), (unsigned)y);
        if (lanes == 32) cache_append4_kernel<32><<<grid, 256, 0, stream>>>(g);
        else cache_append4_kernel<16><<<grid, 256, 0, stream>>>(g);
        const hipError_t e = hipGetLastError();
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
    const uint32_t chunks = (uint32_t)c.head_dim / 8;
    const int64_t each = 2 * (int64_t)c.kv_heads * chunks;
    g.page = fast_div((uint32_t)c.page_size);
    g.each = fast_div((uint32_t)each);
    g.chunks = fast_div(chunks);
    g.group_shift = c.group_size == c.head_dim ? 31 : c.group_size == 128 ? 4 : c.group_size == 64 ? 3 : 2;
    g.bf = dtype == ORTH_DT_BF16;
    g.vec = wide(r.k_out, r.k_strides) && wide(r.v_out, r.v_strides);
    const int W = ORTH_INT4_ROW_BYTES(c.head_dim) / 16;
    // (thread numbers stay within 31 bits)
    const int64_t slots = ((int64_t)1 << 30) / each;
    for (int64_t i = 0; i < r.count; i += slots) {
        g.r.count = r.count - i < slots ? r.count - i : slots;
        const dim3 grid((unsigned)((g.r.count * each + 255) / 256));
        if (W == 2) cache_read4_kernel<2><<<grid, 256, 0, stream>>>(g);
        else if (W == 3) cache_read4_kernel<3><<<grid, 256, 0, stream>>>(g);
        else if (W == 4) cache_read4_kernel<4><<<grid, 256, 0, stream>>>(g);
        else cache_read4_kernel<8><<<grid, 256, 0, stream>>>(g);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        g.r.slots += slots;
        g.r.k_out = (uint16_t *)g.r.k_out + slots * r.k_strides[0];
        g.r.v_out = (uint16_t *)g.r.v_out + slots * r.v_strides[0];
    }
    return hipSuccess;
}

}  // namespace orth
