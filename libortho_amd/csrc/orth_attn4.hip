// Attention of single tokens over the cache in 4 bits.
//
// One pass over the keys with a running maximum and sum of the softmax, as
// over the cache in 16 bits (orth_attn.hip): a wave takes 32 keys from
// registers alone, as two matrix products over v_mfma_f32_16x16x32_f16 whose
// 16 columns are the query heads that share a key head, or, where several
// tokens of one request come together, those of up to 16 / heads neighbouring
// tokens, each with its own range of keys.
//
// Keys and values are low + u * scale.  The codes u enter the products, exact
// in FP16; scales and lows stay outside, in FP32:
//
//   scores  S[key] = scale2 (sum_g scale_g (q . u)_g + low_g sum_g q).  A lane
//           loads units 4 lg .. 4 lg + 3 of its key; byte b of them is step b
//           of the product: one v_perm_b32 pairs the bytes of two units, two
//           masks make their nibbles subnormal numbers u 2^-24 and 16 u 2^-24
//           (the matrix units take them exactly; the query's elements beside
//           the latter are divided by 16).  A step is 32 elements, so a group
//           is a whole number of steps and has its own accumulator.
//   values  O[d] = sum_j (p_j scale_j) (u_j - 8) + sum_j p_j (low_j + 8
//           scale_j).  A lane loads its unit of eight keys; v_perm_b32 pairs
//           the bytes of two keys, a mask and an or make 1024 + u and 1024 +
//           16 u, one packed subtraction u - 8 and 16 (u - 8): codes about
//           zero, so that the sums are no larger than what they are to give.
//           The weights p scale enter as two FP16 parts, 2^-24 of the weight
//           or 2^-39 of the largest of their column: the running maximum is
//           that of score + exponent of the key's largest scale, so that
//           weights are at most 1 whatever the values' size is.
//
// Queries are multiplied by the power of two that brings their largest element
// to 2^14 and beyond, so that BF16 ones fit FP16.  Scale and low of the tile's
// keys and values are held by one lane each (16 lanes of a group: eight keys,
// eight values) and broadcast within the row of 16 lanes by DPP.
#include "orth_attend.h"
#include "orth_serve4.h"

namespace orth {

namespace {

__device__ __forceinline__ int64_t uniform64(int64_t v) {
    return (int64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)v) | (int64_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32;
}

struct Attend4Args : AttendArgs<orth_hip_int4_cache_t> {
    static constexpr bool blocks = true;
    int block;   // tokens that may share a head tile, a power of two
    int groups;  // of a vector
    int bf;
    __device__ __forceinline__ uint16_t round(float v) const { return bf ? store16<true>(v) : store16<false>(v); }
};

template <int N, class F, int... I>
__device__ __forceinline__ void each_of(F &&f, std::integer_sequence<int, I...>) {
    (f(Int<I>()), ...);
}
template <int N, class F>
__device__ __forceinline__ void each(F &&f) {
    each_of<N>(f, std::make_integer_sequence<int, N>());
}

// Lane I's value of each row of 16 lanes.
template <int I>
__device__ __forceinline__ float from_lane(float v) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x150 + I, 0xf, 0xf, true));
}

// acc += lane I's v * x.  (The compiler folds the broadcast into a product or a
// sum, not into a fused one.  The wait covers a v, or an x by an
// exponential, written just before.)
template <int I>
__device__ __forceinline__ void add_from_lane(float &acc, float v, float x) {
    asm("s_nop 1\n\tv_fmac_f32_dpp %0, %1, %2 row_newbcast:%3 row_mask:0xf bank_mask:0xf" : "+v"(acc) : "v"(v), "v"(x), "n"(I));
}
// The same over x[0 .. 8) with lanes 8 .. 15.
__device__ __forceinline__ void add_from_lanes(float &acc, float v, const float *x) {
    asm("s_nop 1\n\t"
        "v_fmac_f32_dpp %0, %1, %2 row_newbcast:8 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %0, %1, %3 row_newbcast:9 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %0, %1, %4 row_newbcast:10 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %0, %1, %5 row_newbcast:11 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %0, %1, %6 row_newbcast:12 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %0, %1, %7 row_newbcast:13 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %0, %1, %8 row_newbcast:14 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %0, %1, %9 row_newbcast:15 row_mask:0xf bank_mask:0xf"
        : "+v"(acc)
        : "v"(v), "v"(x[0]), "v"(x[1]), "v"(x[2]), "v"(x[3]), "v"(x[4]), "v"(x[5]), "v"(x[6]), "v"(x[7]));
}
// lane I's v * x + y, as a product and a sum (see add_from_lane; x may be a
// matrix product's result, whose wait only the compiler knows).
template <int I>
__device__ __forceinline__ float sum_from_lane(float v, float x, float y) {
#pragma clang fp contract(off)
    const float z = from_lane<I>(v) * x;
    return z + y;
}

__device__ __forceinline__ f32x4 mfma16(const u32x4 &a, const u32x4 &b, const f32x4 &c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Bytes A and B of the words that `w` holds, as 16-bit halves.
template <int A, int B>
__device__ __forceinline__ uint32_t two_bytes(const uint32_t *w) {
    return __builtin_amdgcn_perm(w[B / 4], w[A / 4], 0x0c000c00u | (A % 4) | (4 + B % 4) << 16);
}

typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(4)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(4)));

// N words from p.
template <int N>
__device__ __forceinline__ void load_words(uint32_t *w, const void *p) {
    const uint32_t *s = static_cast<const uint32_t *>(p);
    int i = 0;
#pragma unroll
    for (; i + 4 <= N; i += 4) {
        const u32x4_any v = *reinterpret_cast<const u32x4_any *>(s + i);
#pragma unroll
        for (int c = 0; c < 4; c++) w[i + c] = v[c];
    }
    if constexpr (N % 4 >= 2) {
        const u32x2_any v = *reinterpret_cast<const u32x2_any *>(s + N / 4 * 4);
        w[N / 4 * 4] = v[0];
        w[N / 4 * 4 + 1] = v[1];
    }
    if constexpr (N % 2) w[N - 1] = s[N - 1];
}

// Workgroups that a CU holds at once (by registers).
template <int W>
constexpr int kResident = W > 4 ? 1 : 2;

// W: bytes of a unit; GS: steps of 32 elements of a group; PG8: page_size is a
// multiple of 8, so eight keys from a multiple of 8 lie in one page and one
// table entry serves them.
template <int W, int GS, bool PG8>
__global__ __launch_bounds__(256, kResident<W>) void attend4_kernel(Attend4Args g) {
    constexpr int NG = W / GS, VD = (W + 3) / 4;
    constexpr int row_floats = 32 * W + 4;
    // o [waves][gt][32 W + 4], then (m, l) [waves][16]; both start at 16 bytes, and so does each row of o
    extern __shared__ __align__(16) float lds[];
    float2 *lds_stat = reinterpret_cast<float2 *>(lds + kWaves * g.gt * row_floats);
    const int D = g.c.head_dim;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int lane = threadIdx.x & 63;
    const int items = g.c.kv_heads * g.gtiles / g.nh;  // items of a token
    const int hw = wave / g.nsub, sub = wave - hw * g.nsub;

    Share w;
    if (!share_of(g, lane, items, &w)) return;
    const uint64_t first = uniform64(w.cur), stop = uniform64(w.stop), per = uniform64(w.per);
    uint64_t cur = w.cur;
    int64_t t = w.t;
    Keys k = w.k;
    int item = __builtin_amdgcn_readfirstlane(w.item), tokens = 1;
    uint32_t unit = (uint32_t)__builtin_amdgcn_readfirstlane((int)w.unit);
    if (g.block > 1) k = keys_at(g, t, lane, &tokens);
    cur = uniform64(cur), t = uniform64(t);

    while (cur < stop) {
        // (the empty asm: nothing that follows from the lane is kept in registers
        // from one item to the next)
        asm volatile("" : "+v"(lane));
        const int col = lane & 15, lg = lane >> 4;
        const int64_t k_slot = g.c.k_code_strides[1], v_slot = g.c.v_code_strides[1];
        const bool q8 = ((reinterpret_cast<uintptr_t>(g.a.q) | (uintptr_t)(g.a.q_strides[0] * 2) | (uintptr_t)(g.a.q_strides[1] * 2)) & 7) == 0;
        const bool o16 = ((reinterpret_cast<uintptr_t>(g.a.out) | (uintptr_t)(g.a.out_strides[0] * 2) | (uintptr_t)(g.a.out_strides[1] * 2)) & 15) == 0;
        // this lane's pairs: the keys' (col < 8) or the values'
        const bool of_value = col >= 8;
        const int64_t s_page = of_value ? g.c.v_scale_strides[0] : g.c.k_scale_strides[0];
        const int64_t s_slot = of_value ? g.c.v_scale_strides[1] : g.c.k_scale_strides[1];
        // held with the codes' 2^-24 of the scores (keys), or the weights' 2^14 (values, whose codes are 8 less)
        const float s_held = of_value ? 0x1p14f : 0x1p24f, s_middle = of_value ? 8.f : 0.f;
        // (W == 3: the last unit is read from a byte earlier, so that its word ends with the row)
        const int v_at = W == 3 && col == 15 ? 44 : W * col, v_shift = W == 3 && col == 15 ? 8 : 0;
        const uint64_t left = stop - cur;
        const uint32_t n = k.units - unit < left ? k.units - unit : (uint32_t)left;
        const int ht = item * g.nh + hw, kvh = g.gtiles == 1 ? ht : ht / g.gtiles, gt0 = (ht - kvh * g.gtiles) * 16;  // first query head of the tile
        const int cols = tokens > 1 ? tokens * g.group : g.group - gt0 < 16 ? g.group - gt0 : 16;
        const int64_t row = g.a.rows ? (int64_t)__builtin_amdgcn_readfirstlane(g.a.rows[t]) : t;

        // this column's query, and the keys its token sees
        u32x4 q[W];
        float qs[NG], unscale;  // scale2 times the sums of the groups' elements; scale2 / the query's power of two
        int begin = k.begin, end = k.end, most_begin = k.begin, least_end = k.end;
        {
            const int j = tokens > 1 && col < cols ? col / g.group : 0;
            const uint16_t *p = (const uint16_t *)g.a.q + (t + j) * g.a.q_strides[0] + ((int64_t)kvh * g.group + gt0 + (col - j * g.group)) * g.a.q_strides[1];
            float x[W][8], top = 0.f, odd = 0.f;
#pragma unroll
            for (int s = 0; s < W; s++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int d = 32 * s + 16 * h + 4 * lg;
                    uint16_t e[4] = {0, 0, 0, 0};
                    if (col < cols && d < D) {
                        if (q8) {
                            const uint2 v = *reinterpret_cast<const uint2 *>(p + d);
                            e[0] = (uint16_t)v.x, e[1] = (uint16_t)(v.x >> 16), e[2] = (uint16_t)v.y, e[3] = (uint16_t)(v.y >> 16);
                        } else {
#pragma unroll
                            for (int c = 0; c < 4; c++) e[c] = p[d + c];
                        }
                    }
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        const float v = g.bf ? load16<true>(e[c]) : load16<false>(e[c]);
                        x[s][4 * h + c] = v;
                        top = fmaxf(top, fabsf(v));
                        odd += v * 0.f;  // NaN from what is not finite
                    }
                }
            const int up = 15 - __builtin_amdgcn_frexp_expf(column_max(top));
            unscale = ldexpf(g.scale2, -up) + column_sum(odd);
#pragma unroll
            for (int s = 0; s < W; s++) {
                float y[8];
#pragma unroll
                for (int c = 0; c < 8; c++) y[c] = ldexpf(x[s][c], c < 4 ? up : up - 4);
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    // elements 4 lg + 0, 1; 16 on; 4 lg + 2, 3; 16 on
                    const f16x2 h = {(f16)y[c == 0 ? 0 : c == 1 ? 4 : c == 2 ? 2 : 6], (f16)y[c == 0 ? 1 : c == 1 ? 5 : c == 2 ? 3 : 7]};
                    q[s][c] = __builtin_bit_cast(uint32_t, h);
                }
            }
#pragma unroll
            for (int i = 0; i < NG; i++) {
                float sum = 0.f;
#pragma unroll
                for (int s = i * GS; s < (i + 1) * GS; s++)
#pragma unroll
                    for (int c = 0; c < 8; c++) sum += x[s][c];
                qs[i] = column_sum(sum) * g.scale2;
            }
            if (tokens > 1) {
                int64_t b, e;
                range_of(g, t + j, &b, &e);
                begin = most_begin = (int)b;
                end = least_end = (int)e;
#pragma unroll
                for (int d = 1; d < 16; d *= 2) {
                    const int ob = __shfl_xor(most_begin, d, 64), oe = __shfl_xor(least_end, d, 64);
                    most_begin = most_begin > ob ? most_begin : ob;
                    least_end = least_end < oe ? least_end : oe;
                }
                most_begin = __builtin_amdgcn_readfirstlane(most_begin);
                least_end = __builtin_amdgcn_readfirstlane(least_end);
            }
        }

        const int32_t *table = g.a.block_table + row * g.a.table_stride;
        const uint8_t *kbase = (const uint8_t *)g.c.k_codes + kvh * g.c.k_code_strides[2];
        const uint8_t *vbase = (const uint8_t *)g.c.v_codes + kvh * g.c.v_code_strides[2];
        const uint16_t *sbase = of_value ? (const uint16_t *)g.c.v_scales + kvh * g.c.v_scale_strides[2]
                                         : (const uint16_t *)g.c.k_scales + kvh * g.c.k_scale_strides[2];
        const int last = k.end - 1;
        const uint64_t upto = (uint64_t)(unit + n) * (kPair * g.nsub);
        const int step = g.nsub, tile_end = k.tile0 + (int)(upto < (uint64_t)k.tiles ? upto : (uint64_t)k.tiles);
        int tile = k.tile0 + (int)unit * (kPair * g.nsub) + sub;

        f32x4 o[2 * W];
        float m = -__builtin_inff(), l = 0.f, lows[NG];  // lows: sum p (low + 8 scale)
#pragma unroll
        for (int e = 0; e < 2 * W; e++) o[e] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NG; i++) lows[i] = 0.f;

        // a key's page (-1: outside the cache) and its place; keys past the last
        // are taken as the last (with PG8 the first key of a group of eight
        // stands for all: the group lies in its page also where the last key
        // ends inside it)
        const int limit = PG8 ? last & ~7 : last;
        auto entry = [&](int key) -> int32_t { return table[quotient((uint32_t)(key < limit ? key : limit), g.page)]; };
        auto place = [&](int key, int32_t page, int64_t s0, int64_t s1) -> int64_t {
            key = key < limit ? key : limit;
            const uint32_t in = (uint32_t)key - quotient((uint32_t)key, g.page) * g.page.d;
            return ((uint32_t)page < (uint64_t)g.c.pages ? (int64_t)page : 0) * s0 + (int64_t)in * s1;
        };

        // what a wave holds of a tile until it is taken
        uint32_t kc[2][W];        // units 4 lg .. of keys 8 (col / 4) + col % 4 and + 4
        uint32_t vc[8][VD];       // unit col of keys 8 lg ..
        uint32_t pair[NG];        // (scale, low) of key (col < 8) or value 8 lg + col % 8
        int32_t page = 0;         // of keys 8 lg ..
        uint32_t seen8 = 0xff;    // (without PG8: which of them lie in a page of the cache)
        int32_t ke = 0, ve = 0;   // with PG8: the pages of the next tile to load

        auto load_entries = [&](int tl) {
            if constexpr (PG8) {
                ke = entry(tl * kTile + (col >> 2) * 8);
                ve = entry(tl * kTile + lg * 8);
            }
        };
        auto load_k = [&](int tl) {
            const int key = tl * kTile + (col >> 2) * 8;
            const uint8_t *p[2];
            if constexpr (PG8) {
                p[0] = kbase + place(key, ke, g.c.k_code_strides[0], k_slot) + (col & 3) * k_slot;
                p[1] = p[0] + 4 * k_slot;
            } else {
#pragma unroll
                for (int tau = 0; tau < 2; tau++) {
                    const int x = key + 4 * tau + (col & 3);
                    p[tau] = kbase + place(x, entry(x), g.c.k_code_strides[0], k_slot);
                }
            }
#pragma unroll
            for (int tau = 0; tau < 2; tau++) load_words<W>(kc[tau], p[tau] + lg * 4 * W);
        };
        auto load_v = [&](int tl) {
            const int key = tl * kTile + lg * 8;
            const uint8_t *p = vbase;
            const uint16_t *sp = sbase;
            if constexpr (PG8) {
                page = ve;
                p += place(key, ve, g.c.v_code_strides[0], v_slot);
                sp += place(key, ve, s_page, s_slot) + (col & 7) * s_slot;
            } else {
                seen8 = 0;
                const int x = key + (col & 7);
                sp += place(x, entry(x), s_page, s_slot);
            }
            if constexpr (W == 8) {  // (only vectors past 128 elements may have fewer groups than steps)
#pragma unroll
                for (int i = 0; i < NG; i++) pair[i] = reinterpret_cast<const uint32_t *>(sp)[i < g.groups ? i : g.groups - 1];
            } else {
                load_words<NG>(pair, sp);
            }
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const uint8_t *x = p;
                if constexpr (PG8) {
                    x += i * v_slot;
                } else {
                    const int32_t pg = entry(key + i);
                    x += place(key + i, pg, g.c.v_code_strides[0], v_slot);
                    seen8 |= (uint32_t)((uint32_t)pg < (uint64_t)g.c.pages) << i;
                }
                x += v_at;
                if constexpr (W == 2) vc[i][0] = *reinterpret_cast<const uint16_t *>(x);
                else if constexpr (W == 3) __builtin_memcpy(&vc[i][0], x, 4);
                else load_words<VD>(vc[i], x);
            }
        };

        if (tile < tile_end) {
            load_entries(tile);
            load_k(tile);
            load_v(tile);
            load_entries(tile + step);
        }
        for (; tile < tile_end; tile += step) {
            // scores
            float sc[NG], lo[NG], size = 0.f;
#pragma unroll
            for (int i = 0; i < NG; i++) {
                const f16x2 v = __builtin_bit_cast(f16x2, pair[i]);
                const float scale = (float)v[0];
                size = fmaxf(size, fabsf(scale));
                sc[i] = scale * s_held;
                lo[i] = fmaf(scale, s_middle, (float)v[1]);
            }
            const float expo = (float)__builtin_amdgcn_frexp_expf(size);
            float x[8], offset[8];
            each<NG>([&](auto group) {
                constexpr int C = group.value;
                f32x4 acc[2];
#pragma unroll
                for (int tau = 0; tau < 2; tau++) acc[tau] = f32x4{0.f, 0.f, 0.f, 0.f};
                each<GS>([&](auto b) {
                    constexpr int B = C * GS + b.value;
#pragma unroll
                    for (int tau = 0; tau < 2; tau++) {
                        const uint32_t y = two_bytes<B, W + B>(kc[tau]), z = two_bytes<2 * W + B, 3 * W + B>(kc[tau]);
                        acc[tau] = mfma16(u32x4{y & 0x000f000fu, y & 0x00f000f0u, z & 0x000f000fu, z & 0x00f000f0u}, q[B], acc[tau]);
                    }
                });
                each<8>([&](auto i) {
                    constexpr int I = i.value;
                    if constexpr (C == 0) {
                        x[I] = from_lane<I>(sc[0]) * acc[I >> 2][I & 3];
                        offset[I] = from_lane<I>(lo[0]) * qs[0];
                    } else {
                        x[I] = sum_from_lane<I>(sc[C], acc[I >> 2][I & 3], x[I]);
                        add_from_lane<I>(offset[I], lo[C], qs[C]);
                    }
                });
            });
            __builtin_amdgcn_sched_barrier(0);
            load_k(tile + step);  // (past the end: the last keys again)
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = fmaf(unscale, x[i], offset[i]);

            const int key0 = tile * kTile;
            const bool paged = PG8 ? (uint32_t)page < (uint64_t)g.c.pages : seen8 == 0xff;
            const bool masked = key0 < most_begin || key0 + kTile > least_end || !__all(paged);
            uint32_t in8 = 0xff;  // which of the lane's keys its column sees
            if (masked) {
                asm volatile("");  // (a branch: tiles at the ends of a range are few)
                in8 = 0;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int key = key0 + 8 * lg + i;
                    const bool in = key >= begin && key < end && (PG8 ? paged : (seen8 >> i & 1) != 0);
                    in8 |= (uint32_t)in << i;
                    if (!in) x[i] = -__builtin_inff();
                }
            }
            float top = -__builtin_inff();
            each<8>([&](auto i) { top = fmaxf(top, x[i.value] + from_lane<8 + i.value>(expo)); });
            top = fmaxf(fmaxf(column_max(top), kLeast), m);
            if (__any(top > m)) {
                const float keep = __builtin_amdgcn_exp2f(m - top);
                l *= keep;
#pragma unroll
                for (int i = 0; i < NG; i++) lows[i] *= keep;
#pragma unroll
                for (int e = 0; e < 2 * W; e++)
#pragma unroll
                    for (int i = 0; i < 4; i++) o[e][i] *= keep;
                m = top;
            }
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[i] = __builtin_amdgcn_exp2f(x[i] - m);
                l += x[i];
            }
            each<NG>([&](auto group) {
                constexpr int C = group.value;
                float weight[8];
                float sum = 0.f;
                add_from_lanes(sum, lo[C], x);
                each<8>([&](auto i) { weight[i.value] = from_lane<8 + i.value>(sc[C]) * x[i.value]; });
                if (masked) {  // once more without the hidden keys, whose numbers may be anything
                    asm volatile("");
                    sum = 0.f;
                    each<8>([&](auto i) {
                        const bool in = in8 >> i.value & 1;
                        const float scale = from_lane<8 + i.value>(sc[C]), low = from_lane<8 + i.value>(lo[C]);
                        weight[i.value] = in ? scale * x[i.value] : 0.f;
                        sum += in ? low * x[i.value] : 0.f;
                    });
                }
                lows[C] += sum;
                u32x4 part[2];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const f16x2 big = {(f16)weight[2 * i], (f16)weight[2 * i + 1]};
                    const f16x2 small = {(f16)(weight[2 * i] - (float)big[0]), (f16)(weight[2 * i + 1] - (float)big[1])};
                    part[0][i] = __builtin_bit_cast(uint32_t, big);
                    part[1][i] = __builtin_bit_cast(uint32_t, small);
                }
                each<GS>([&](auto b) {
                    constexpr int B = C * GS + b.value;
                    u32x4 even, odd;  // elements 32 B + col and 16 on of the lane's eight keys
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint32_t w2[2] = {W == 3 ? vc[2 * i][B / 4] >> v_shift : vc[2 * i][B / 4],
                                                W == 3 ? vc[2 * i + 1][B / 4] >> v_shift : vc[2 * i + 1][B / 4]};
                        const uint32_t y = two_bytes<B % 4, 4 + B % 4>(w2);
                        const f16x2 e = __builtin_bit_cast(f16x2, (y & 0x000f000fu) | 0x64006400u) - f16x2{(f16)1032.f, (f16)1032.f};
                        const f16x2 h = __builtin_bit_cast(f16x2, (y & 0x00f000f0u) | 0x64006400u) - f16x2{(f16)1152.f, (f16)1152.f};
                        even[i] = __builtin_bit_cast(uint32_t, e);
                        odd[i] = __builtin_bit_cast(uint32_t, h);
                    }
#pragma unroll
                    for (int z = 0; z < 2; z++) {
                        o[2 * B] = mfma16(even, part[z], o[2 * B]);
                        o[2 * B + 1] = mfma16(odd, part[z], o[2 * B + 1]);
                    }
                });
            });
            __builtin_amdgcn_sched_barrier(0);
            load_v(tile + step);
            load_entries(tile + 2 * step);
            __builtin_amdgcn_sched_barrier(0);
        }

        // join the waves of each head tile
        l = column_sum(l);
#pragma unroll
        for (int i = 0; i < NG; i++) lows[i] = column_sum(lows[i]);
        if (col < cols) {
            float *dst = lds + (wave * g.gt + col) * row_floats + 4 * lg;
#pragma unroll
            for (int e = 0; e < 2 * W; e++) {
                const float f = e % 2 ? 0x1p-18f : 0x1p-14f, b = lows[e / (2 * GS)];
                *reinterpret_cast<f32x4 *>(dst + 16 * e) = f32x4{fmaf(o[e][0], f, b), fmaf(o[e][1], f, b), fmaf(o[e][2], f, b), fmaf(o[e][3], f, b)};
            }
            if (lg == 0) lds_stat[wave * 16 + col] = float2{m, l};
        }
        __syncthreads();
        finish_item(g, wave * 64 + lane, lds, lds_stat, row_floats, o16, first, cur, per, t, tokens, k, item, unit, n);
        __syncthreads();
        cur += n;
        unit = 0;
        if (++item == items) {
            item = 0;
            t = uniform64(t + tokens);
            if (cur < stop) k = keys_at(g, t, lane, &tokens);
        }
    }
}

// What both the workspace and the launch go by.
Attend4Args attend4_args(const orth_hip_int4_cache_t &c, const orth_hip_attend_t &a, int cus, int64_t *groups) {
    Attend4Args g;
    g.c = c;
    g.a = a;
    g.page = fast_div((uint32_t)c.page_size);
    g.scale2 = a.scale * 1.4426950408889634f;
    g.group = a.q_heads / c.kv_heads;
    g.gtiles = (g.group + 15) / 16;
    g.groups = c.head_dim / c.group_size;
    g.block = 1;
    if (a.rows && a.tokens > 1)
        while (2 * g.block * g.group <= 16) g.block *= 2;
    g.gt = g.block * g.group < 16 ? g.block * g.group : 16;
    attend_tiles(g, cus, a.tokens);
    *groups = attend_groups(g, (int64_t)cus * (c.head_dim > 128 ? kResident<8> : kResident<4>), g.block);
    return g;
}

}  // namespace

int64_t attention4_workspace_bytes(const orth_hip_int4_cache_t &c, const orth_hip_attend_t &a, int cus, int64_t *groups) {
    int64_t n = 0;
    const Attend4Args g = attend4_args(c, a, cus, &n);
    *groups = attend_units(g, g.block) > 1 ? n : 0;  // (items of one unit are not split)
    return attend_bytes(g, n);
}

hipError_t launch_paged_attention4(const orth_hip_int4_cache_t &c, const orth_hip_attend_t &a, int32_t dtype, int cus,
                                   void *work, uint32_t *counters, hipStream_t stream) {
    int64_t groups = 0;
    Attend4Args g = attend4_args(c, a, cus, &groups);
    attend_workspace(g, groups, work, counters);
    g.bf = dtype == ORTH_DT_BF16;
    const hipError_t e = by_int4_layout(c, [&](auto unit, auto steps) -> hipError_t {
        constexpr int W = decltype(unit)::value, GS = decltype(steps)::value;
        const size_t lds = (size_t)kWaves * g.gt * (32 * W + 4) * 4 + kWaves * 16 * sizeof(float2);
        auto go = [&](auto kernel) -> hipError_t {
            if (lds > 48 * 1024) {
                hipError_t s = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                                   hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
                if (s != hipSuccess) return s;
            }
            kernel<<<dim3((unsigned)groups), 256, lds, stream>>>(g);
            return hipGetLastError();
        };
        return c.page_size % 8 == 0 ? go(attend4_kernel<W, GS, true>) : go(attend4_kernel<W, GS, false>);
    });
    if (e != hipSuccess) return e;
    return attend_joins(g, groups, g.block) ? launch_join(g, groups, stream) : hipSuccess;
}

}  // namespace orth
