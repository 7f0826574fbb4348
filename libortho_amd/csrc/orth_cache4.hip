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
// What is quantised has to be the turned key in 64 bits rounded to FP32 and to
// FP16, and a code the one nearest to the quotient: a last place of difference
// moves a code by a whole step.  FP32 decides all but the numbers next to a border,
// and 64 bits those (one key in some 800, one code in some 30,000).
//
// An element is read once and, of keys and values, a quarter of it written;
// bound by memory where there are many tokens (32 + 8 heads of 128: 8,192
// tokens in 46 us, 3.9 TB/s; 2,048 in 14.5 to 15.3, 3 TB/s, and 5 more while
// what only numbers next to a border need was worked out beforehand, in 95
// registers instead of 63).
struct Append4Args {
    orth_hip_int4_cache_t c;
    orth_hip_append_t a;
    FastDiv page;
    int W;
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

// Two elements of 16 bits, rounded to nearest even.
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
template <bool BF>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    if constexpr (BF) return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, f16x2));
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

// LP: lanes of a vector.  PLAIN: vectors are 16-byte aligned, and a lane's
// elements are turned all or not at all, their partners being its own or
// another lane's.
template <int LP, bool BF, bool PLAIN>
__global__ __launch_bounds__(256) void cache_append4_kernel(Append4Args g) {
    constexpr int VECS = 256 / LP;
    const int64_t t = blockIdx.x;
    const int c = threadIdx.x % LP, d0 = 8 * c, D = g.c.head_dim, rot = g.a.rot, half = rot / 2;
    const int64_t slot = g.a.slots[t];
    bool write = slot >= 0 && slot < g.c.pages * g.c.page_size, placed = true;
    // this lane's cosines and sines, these negative for the first of a pair:
    // (a, b) -> a c - b s, b c + a s
    float cs[8], sn[8];
    const bool inter = g.a.interleaved != 0, aligned_half = PLAIN || half % 8 == 0;
    int64_t pos = 0;
    if (g.a.cos_sin) {
        pos = g.a.positions[t];
        placed = pos >= 0 && pos < g.a.cos_sin_rows;
        write = write && placed;
    }
    const bool turns = d0 < rot && placed;
    const float *table = g.a.cos_sin + pos * rot;
    if (turns) {
        if (PLAIN && !inter) {
            const float *p = table + (d0 < half ? d0 : d0 - half);
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                const f32x4_any vc = *reinterpret_cast<const f32x4_any *>(p + e), vs = *reinterpret_cast<const f32x4_any *>(p + half + e);
#pragma unroll
                for (int i = 0; i < 4; i++) cs[e + i] = vc[i], sn[e + i] = d0 < half ? -vs[i] : vs[i];
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int d = d0 + e, ci = d >= rot ? 0 : inter ? d >> 1 : d < half ? d : d - half;
                cs[e] = PLAIN || d < rot ? table[ci] : 1.f;
                sn[e] = PLAIN || d < rot ? table[half + ci] : 0.f;
                if (inter ? !(e & 1) : d < half) sn[e] = -sn[e];
            }
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
            if (PLAIN || g.vec) {
                raw = *reinterpret_cast<const u32x4 *>(src + d0);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) raw[e] = (uint32_t)src[d0 + 2 * e] | (uint32_t)src[d0 + 2 * e + 1] << 16;
            }
        }
        auto value = [&](const u32x4 &w, int e) -> float {
            const uint32_t b = w[e >> 1];
            if constexpr (BF) return __uint_as_float(e & 1 ? b & 0xffff0000u : b << 16);
            else return load16<false>((uint16_t)(e & 1 ? b >> 16 : b));
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
                if (turn && here && d < rot && (is_q || write)) w[e] = load16<BF>(src[pd]);
            }
        }
        if (is_q) {
            if (turn)
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (PLAIN || d0 + e < rot) x[e] = x[e] * cs[e] + w[e] * sn[e];
            // (q_out may be q: all lanes have read the vector before one writes it)
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            if (here) {
                uint16_t *dst = (uint16_t *)g.a.q_out + t * g.a.q_out_strides[0] + h * g.a.q_out_strides[1] + d0;
                u32x4 y;
#pragma unroll
                for (int e = 0; e < 4; e++) y[e] = pack16<BF>(x[2 * e], x[2 * e + 1]);
                if (PLAIN || g.vec) {
                    *reinterpret_cast<u32x4 *>(dst) = y;
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++) dst[e] = (uint16_t)(y[e / 2] >> 16 * (e % 2));
                }
            }
        }
        if (__all(is_q)) continue;
        const bool kv = h < all && !is_q && write;

        float odd = 0.f;  // NaN where an element is not finite
#pragma unroll
        for (int e = 0; e < 8; e++) {
            float v = x[e];
            if (is_k && turn && (PLAIN || d0 + e < rot)) {
                // x c + w s: the product's error comes back in a second fused
                // step, so f is within two last places of FP32
                const float p = w[e] * sn[e], f = fmaf(x[e], cs[e], p) + fmaf(w[e], sn[e], -p);
                const uint32_t b = __float_as_uint(f), a = b & 0x7fffffffu;
                v = f;
                // next to a border of FP16 numbers (a low part of 0x1000), or
                // below the normal ones, or too large
                if (((b + 4 - 0x1000) & 0x1fff) <= 8 || a < 0x38800000u || a > 0x47000000u) {
                    float ce = cs[e], se = sn[e];
                    asm volatile("" : "+v"(ce), "+v"(se));  // (what few elements need is not worked out beforehand)
                    double y = (double)x[e] * ce + (double)w[e] * se;
                    y = y > 65504.0 ? 65504.0 : y < -65504.0 ? -65504.0 : y;
                    const bool finite = fabs((double)x[e]) < __builtin_inf() && fabs((double)w[e]) < __builtin_inf() &&
                                        fabsf(ce) < __builtin_inff() && fabsf(se) < __builtin_inff();
                    v = finite ? (float)half_of(y) : __builtin_nanf("");
                }
            }
            odd = fmaf(v, 0.f, odd);
            x[e] = (float)(f16)__builtin_amdgcn_fmed3f(v, -65504.f, 65504.f);
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
        const uint64_t odd_lanes = __ballot(!(odd == 0.f) && here) >> (threadIdx.x & 63 & ~(g.group_lanes - 1));
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
// A thread sixteen elements of a key or a value: the low and the high nibbles
// of one byte (b) of eight units, so it loads 8 W bytes, which the threads of
// a vector share in the L1, and stores twice 16.  It keeps its place in the
// vectors for all the slots that its workgroup takes, so that a slot costs it
// little more than the elements; where the threads of a slot are whole waves
// (UNI), page and offsets are scalar.
// Memory-bound: codes and scales read once, the elements written (256 MB in
// 58 us, 4.4 TB/s; the call 65 us, with eight elements and one slot a thread 96).
struct Read4Args {
    orth_hip_int4_cache_t c;
    orth_hip_read_t r;
    FastDiv page, each, chunks;  // each: threads of a slot's keys, chunks: of a vector
    FastDiv parts;               // workgroups of 256 threads of those
    int at_once, per_group;      // slots of a workgroup: at once, and in all
    int group_shift;             // of 32 elements: 31 where the whole vector is one group
    int vec;
};

typedef const __attribute__((address_space(4))) int64_t *ConstLongs;  // (scalar loads: nothing writes there meanwhile)

template <int W, bool BF, bool UNI>
__global__ __launch_bounds__(256) void cache_read4_kernel(Read4Args g) {
    const bool is_v = blockIdx.y != 0;
    const int64_t *st = is_v ? g.c.v_code_strides : g.c.k_code_strides, *ss = is_v ? g.c.v_scale_strides : g.c.k_scale_strides;
    const int64_t *so = is_v ? g.r.v_strides : g.r.k_strides;
    const int64_t page_stride = st[0], slot_stride = st[1], spage_stride = ss[0], sslot_stride = ss[1], out_stride = so[0];
    const int tid = threadIdx.x;
    int own = (int)quotient(tid, g.each);  // (0 where a slot takes the whole workgroup, or several)
    if constexpr (UNI) own = __builtin_amdgcn_readfirstlane(own);
    const uint32_t group = quotient(blockIdx.x, g.parts), x = (blockIdx.x - group * g.parts.d) * 256u + tid - own * g.each.d;
    if (own >= g.at_once || x >= g.each.d) return;
    const uint32_t head = quotient(x, g.chunks), c = x - head * g.chunks.d;
    const int b = c >> 1, d = 32 * b + 8 * (c & 1), D = g.c.head_dim;
    const uint8_t *codes = (const uint8_t *)(is_v ? g.c.v_codes : g.c.k_codes) + head * st[2] + (c & 1) * 8 * W + (W == 8 ? b >> 2 << 2 : 0);
    const uint16_t *scales = (const uint16_t *)(is_v ? g.c.v_scales : g.c.k_scales) + head * ss[2] + 2 * (b >> g.group_shift);
    uint16_t *out = (uint16_t *)(is_v ? g.r.v_out : g.r.k_out) + head * so[1] + d;
    // bytes b of two units as the low bytes of 16 bits each
    const uint32_t of_words = 0x0c000c00u | (b & 3) * 0x10001u | 0x40000u, of_halves = 0x0c000c00u | b | (2 + b) << 16;
    const int64_t first = (int64_t)group * g.per_group, stop = first + g.per_group < g.r.count ? first + g.per_group : g.r.count;
    for (int64_t i = first + own; i < stop; i += g.at_once) {
        const int64_t slot = UNI ? ((ConstLongs)g.r.slots)[i] : g.r.slots[i];
        const bool here = slot >= 0 && slot < g.c.pages * g.c.page_size;
        const int64_t pg = !here ? 0 : slot <= INT32_MAX ? (int64_t)quotient((uint32_t)slot, g.page) : slot / g.c.page_size;
        const int64_t in = here ? slot - pg * g.c.page_size : 0;
        const uint32_t *row = reinterpret_cast<const uint32_t *>(codes + (pg * page_stride + in * slot_stride));
        uint32_t pair = *reinterpret_cast<const uint32_t *>(scales + (pg * spage_stride + in * sslot_stride));
        uint32_t u[4];  // byte b of the units 2 e and 2 e + 1
        if constexpr (W == 4) {
            const u32x4 lo = reinterpret_cast<const u32x4 *>(row)[0], hi = reinterpret_cast<const u32x4 *>(row)[1];
#pragma unroll
            for (int e = 0; e < 4; e++)
                u[e] = __builtin_amdgcn_perm(e < 2 ? lo[2 * e + 1] : hi[2 * (e & 1) + 1], e < 2 ? lo[2 * e] : hi[2 * (e & 1)], of_words);
        } else if constexpr (W == 2) {
            const u32x4 v = *reinterpret_cast<const u32x4 *>(row);
#pragma unroll
            for (int e = 0; e < 4; e++) u[e] = __builtin_amdgcn_perm(0u, v[e], of_halves);
        } else if constexpr (W == 8) {
#pragma unroll
            for (int e = 0; e < 4; e++) u[e] = __builtin_amdgcn_perm(row[4 * e + 2], row[4 * e], of_words);
        } else {
            uint32_t v[7];
#pragma unroll
            for (int e = 0; e < 6; e++) v[e] = row[e];
            v[6] = 0;
#pragma unroll
            for (int e = 0; e < 6; e++) v[e] = __builtin_amdgcn_alignbyte(v[e + 1], v[e], b);  // from byte b on
#pragma unroll
            for (int e = 0; e < 4; e++) {  // bytes 6 e and 6 e + 3
                constexpr uint32_t none = 0x0c000c00u;
                const int at = 6 * e % 4;
                u[e] = __builtin_amdgcn_perm(v[6 * e / 4 + 1 > 5 ? 5 : 6 * e / 4 + 1], v[6 * e / 4], none | at | (at + 3) << 16);
            }
        }
        pair = here ? pair : 0u;  // zeros
        u32x4 y[2];
        if constexpr (BF) {
            const float scale = load16<false>((uint16_t)pair), low = load16<false>((uint16_t)(pair >> 16));
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    y[h][e] = pack16<true>(fmaf((float)(u[e] >> 4 * h & 15), scale, low), fmaf((float)(u[e] >> (16 + 4 * h) & 15), scale, low));
        } else {
            // 0x6400 | code is 1024 + code; the fused product and sum round once
            const f16x2 p = __builtin_bit_cast(f16x2, pair), scale = {p[0], p[0]}, low = {p[1], p[1]}, k1024 = {(f16)1024.f, (f16)1024.f};
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const f16x2 code = __builtin_bit_cast(f16x2, (u[e] >> 4 * h & 0x000f000fu) | 0x64006400u) - k1024;
                    y[h][e] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(code, scale, low));
                }
        }
        uint16_t *dst = out + i * out_stride;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            if (d + 16 * h >= D) break;
            if (g.vec) {
                *reinterpret_cast<u32x4 *>(dst + 16 * h) = y[h];
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) dst[16 * h + 2 * e] = (uint16_t)y[h][e], dst[16 * h + 2 * e + 1] = (uint16_t)(y[h][e] >> 16);
            }
        }
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
    const int lanes = c.head_dim > 128 ? 32 : 16, vecs = 256 / lanes;
    g.group_lanes = c.group_size == c.head_dim ? lanes : c.group_size / 8;
    g.vec = wide(a.k, a.k_strides) && wide(a.v, a.v_strides) && (!a.q || (wide(a.q, a.q_strides) && wide(a.q_out, a.q_out_strides)));
    const bool plain = g.vec && (a.interleaved ? g.a.rot % 8 == 0 : g.a.rot % 16 == 0);
    const int64_t heads = (a.q ? (int64_t)a.q_heads : 0) + 2 * (int64_t)c.kv_heads, parts = (heads + vecs - 1) / vecs;
    // a workgroup for every 16 (or 8) vectors where tokens alone leave CUs
    // idle, else one a token (32 + 8 heads of 128, three a token and one: 64
    // tokens 5.5 and 6.3 us, 512 6.7 and 6.9, 700 8.6 and 7.9, 8,192 64 and 46)
    const int y = a.tokens >= 2 * cus ? 1 : (int)(parts < 65535 ? parts : 65535);
    for (int64_t t = 0; t < a.tokens; t += kLaunch) {
        const dim3 grid((unsigned)(a.tokens - t < kLaunch ? a.tokens - t : kLaunch), (unsigned)y);
        auto go = [&](auto bf, auto plain) {
            constexpr bool BF = decltype(bf)::value != 0, PLAIN = decltype(plain)::value != 0;
            if (lanes == 32) cache_append4_kernel<32, BF, PLAIN><<<grid, 256, 0, stream>>>(g);
            else cache_append4_kernel<16, BF, PLAIN><<<grid, 256, 0, stream>>>(g);
        };
        auto by = [&](auto plain) { dtype == ORTH_DT_BF16 ? go(Int<1>(), plain) : go(Int<0>(), plain); };
        if (plain) by(Int<1>());
        else by(Int<0>());
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
    const uint32_t chunks = 2 * (((uint32_t)c.head_dim + 31) / 32), each = (uint32_t)c.kv_heads * chunks;
    g.page = fast_div((uint32_t)c.page_size);
    g.each = fast_div(each);
    g.chunks = fast_div(chunks);
    g.at_once = each < 256 ? (int)(256 / each) : 1;
    g.group_shift = c.group_size == c.head_dim ? 31 : c.group_size == 128 ? 2 : c.group_size == 64 ? 1 : 0;
    g.vec = wide(r.k_out, r.k_strides) && wide(r.v_out, r.v_strides);
    const int W = ORTH_INT4_ROW_BYTES(c.head_dim) / 16;
    const uint32_t parts = (each + 255) / 256;
    g.parts = fast_div(parts);
    // eight rounds of full CUs where the slots are enough, and a workgroup then
    // takes several (six requests' keys and values, 260 MB: 69 us with one
    // round, 61 with four, 57 with eight and with a slot a turn)
    const int64_t rounds = (r.count + g.at_once - 1) / g.at_once, fill = (int64_t)cus * 8 * 8 / (2 * parts) + 1;
    const int64_t turns = (rounds + fill - 1) / fill, groups = (rounds + turns - 1) / turns;
    g.per_group = (int)(g.at_once * turns);          // (fill is 1 only where at_once is: no more than the slots)
    const dim3 grid((unsigned)(groups * parts), 2);  // (one launch: no more than 2^20 parts)
    auto go = [&](auto unit, auto uni) {
        constexpr int U = decltype(unit)::value;
        constexpr bool S = decltype(uni)::value != 0;
        if (dtype == ORTH_DT_BF16) cache_read4_kernel<U, true, S><<<grid, 256, 0, stream>>>(g);
        else cache_read4_kernel<U, false, S><<<grid, 256, 0, stream>>>(g);
    };
    auto by = [&](auto unit) { each % 64 == 0 ? go(unit, Int<1>()) : go(unit, Int<0>()); };
    if (W == 2) by(Int<2>());
    else if (W == 3) by(Int<3>());
    else if (W == 4) by(Int<4>());
    else by(Int<8>());
    return hipGetLastError();
}

}  // namespace orth
