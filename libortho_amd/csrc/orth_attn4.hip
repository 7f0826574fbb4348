// Attention over the cache in 4 bits: single tokens, and several tokens of a
// request (a prompt, a draft) together.
//
// One pass over the keys with a running maximum and sum of the softmax, as
// over the cache in 16 bits (orth_attn.hip): a wave takes 32 keys from
// registers alone, as two matrix products over v_mfma_f32_16x16x32_f16 whose
// 16 columns are the query heads that share a key head, or, where several
// tokens of one request come together, those of up to 16 / heads neighbouring
// tokens, each with its own range of keys.
//
// Keys and values are low + u * scale = mid + c * scale with c = u - 8 and mid
// = low + 8 scale: sums about the middle are no larger than what they give.
// The c enter the products, exact in FP16; scales and mids stay outside, in
// FP32:
//
//   scores  S[key] = scale2 (sum_g scale_g (q . c)_g + mid_g sum_g q).  A lane
//           loads units 4 lg .. 4 lg + 3 of its key; byte b of them is step b
//           of the product: one v_perm_b32 pairs the bytes of two units, two
//           masks and two packed subtractions make their c of them.  A step is
//           32 elements, so a group is a whole number of steps and has its own
//           accumulator.
//   values  O[d] = sum_j (p_j scale_j) c_j + sum_j p_j mid_j.  A lane loads
//           its unit of eight keys; v_perm_b32 pairs the bytes of two keys,
//           and their c are taken as above.
//           The weights p scale enter as two FP16 parts, off by 2^-24 of the
//           weight or 2^-39 of the largest of their column: the running
//           maximum is that of score + exponent of the key's largest scale, so
//           that the largest weight is between 1/2 and 1, held as 2^14 to 2^15,
//           whatever the values' size is.  (One maximum for all groups: one
//           each would take 8 products and a maximum over keys and lanes a
//           group more, for groups whose scales are below 2^-28 of another's
//           of the same head.)
//
// Queries are multiplied by the power of two that brings their largest element
// to 2^14 and beyond, so that BF16 ones fit FP16: elements below 2^-28 of it are
// subnormal there, multiples of 2^-24.  Scale and low of the tile's keys and
// values are held by four lanes of a score's column each, two keys and two
// values a lane, and broadcast within quads of lanes by DPP.
//
// Bound by memory and instructions about equally where there are many keys
// (128 requests of 2,048 to 16,384 keys, 8 of 64 heads, 943 MB: 239 us, 3.9
// TB/s).  A head's row of a slot is half a line of 128 bytes, so the waves of
// neighbouring heads keep step (a barrier a tile) and find each other's lines
// in the L1 (without it some 11% slower, 1,258 MB read; 1,088 with it, the rest
// (scale, low) pairs whose lines hold the heads of two workgroups).  Few keys:
// a chain of latencies (190 keys, 32 heads: 13 us).  A prompt of 2,048 tokens, 8
// of 32 heads: 288 us.
// Two tiles of keys in one product where no more than eight columns are used,
// and one softmax for both, was 2% faster at the largest call and up to 15%
// slower at the others; four workgroups a CU 3% slower than three.
#include "orth_attend.h"
#include "orth_serve4.h"

namespace orth {

namespace {

struct Attend4Args : AttendArgs<orth_hip_int4_cache_t> {
    static constexpr bool blocks = true;
    int block;   // tokens that may share a head tile, a power of two
    int groups;  // of a vector
    int bf;
    int wave_floats;  // of a wave's part of the LDS
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

// Lane I's value of each quad of lanes.
template <int I>
__device__ __forceinline__ float from_quad(float v) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), I * 0x55, 0xf, 0xf, true));
}
// acc[0 .. 4) += lanes 0 .. 3's v * x, acc[4 .. 8) += theirs of w * x.  (The
// compiler folds the broadcast into a product or a sum, not into a fused one.
// The wait covers a v or w written just before.)
__device__ __forceinline__ void add_each_from_quads(float *acc, float v, float w, float x) {
    asm("s_nop 1\n\t"
        "v_fmac_f32_dpp %0, %8, %10 quad_perm:[0,0,0,0] row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %1, %8, %10 quad_perm:[1,1,1,1] row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %2, %8, %10 quad_perm:[2,2,2,2] row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %3, %8, %10 quad_perm:[3,3,3,3] row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %4, %9, %10 quad_perm:[0,0,0,0] row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %5, %9, %10 quad_perm:[1,1,1,1] row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %6, %9, %10 quad_perm:[2,2,2,2] row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %7, %9, %10 quad_perm:[3,3,3,3] row_mask:0xf bank_mask:0xf"
        : "+v"(acc[0]), "+v"(acc[1]), "+v"(acc[2]), "+v"(acc[3]), "+v"(acc[4]), "+v"(acc[5]), "+v"(acc[6]), "+v"(acc[7])
        : "v"(v), "v"(w), "v"(x));
}
// acc += the sum of lanes 0 .. 3's v * x[0 .. 4) and theirs of w * x[4 .. 8).
// (The wait also covers an x by an exponential.)
__device__ __forceinline__ void add_from_quads(float &acc, float v, float w, const float *x) {
    asm("s_nop 1\n\t"
        "v_fmac_f32_dpp %0, %1, %3 quad_perm:[0,0,0,0] row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %0, %1, %4 quad_perm:[1,1,1,1] row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %0, %1, %5 quad_perm:[2,2,2,2] row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %0, %1, %6 quad_perm:[3,3,3,3] row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %0, %2, %7 quad_perm:[0,0,0,0] row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %0, %2, %8 quad_perm:[1,1,1,1] row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %0, %2, %9 quad_perm:[2,2,2,2] row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %0, %2, %10 quad_perm:[3,3,3,3] row_mask:0xf bank_mask:0xf"
        : "+v"(acc)
        : "v"(v), "v"(w), "v"(x[0]), "v"(x[1]), "v"(x[2]), "v"(x[3]), "v"(x[4]), "v"(x[5]), "v"(x[6]), "v"(x[7]));
}
// lane I's v * x + y, as a product and a sum (x may be a
// matrix product's result, whose wait only the compiler knows).
template <int I>
__device__ __forceinline__ float sum_from_quad(float v, float x, float y) {
#pragma clang fp contract(off)
    const float z = from_quad<I>(v) * x;
    return z + y;
}
// w - part[H].
template <int H>
__device__ __forceinline__ float rest(float w, f16x2 part) {
    float r;
    if constexpr (H == 0) asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(part), "v"(w));
    else asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(part), "v"(w));
    return r;
}

__device__ __forceinline__ f32x4 mfma16(const u32x4 &a, const u32x4 &b, const f32x4 &c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Bytes A and B of the words that `w` holds, below bits that are set.
template <int A, int B>
__device__ __forceinline__ uint32_t two_bytes(const uint32_t *w) {
    return __builtin_amdgcn_perm(w[B / 4], w[A / 4], 0x0d000d00u | (A % 4) | (4 + B % 4) << 16);
}
// Their low and their high nibbles, less 8, as FP16 numbers: 1024 + u and
// 64 + u with exponents left from the bits above, then less 1032 and 72, exactly.
// (The nibbles alone are subnormal numbers, which the matrix units take as well
// and which save the subtraction: 128 requests 231 us for 239, 128 tokens of
// four prompts 95 for 103.  But a matrix product aligns what it sums by
// exponents, a subnormal number's is that of 2^-14 whatever it is, and what
// falls off below 24 bits of the largest is lost: sums came out 2^-17 of their
// magnitude short.  Of 128 requests' 1,048,576 elements 8,493 were not the
// rounded 64-bit ones, with u as normal numbers 1,010, with u - 8 108, and 113
// where everything is FP32.)
__device__ __forceinline__ uint32_t low_codes(uint32_t y) {
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, y & 0x640f640fu) - f16x2{(f16)1032.f, (f16)1032.f});
}
__device__ __forceinline__ uint32_t high_codes(uint32_t y) {
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, y & 0x54f054f0u) - f16x2{(f16)72.f, (f16)72.f});
}

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef const __attribute__((address_space(4))) int32_t *ConstInts;  // (scalar loads: nothing writes there meanwhile)
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

// N words, or the 16 bits of half a word, at base + at + more.
template <int N>
__device__ __forceinline__ void load_from(uint32_t *w, const uint8_t *base, uint32_t at, uint32_t more) {
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(base), 0, -1, 0x00020000);
    int i = 0;
#pragma unroll
    for (; i + 4 <= N; i += 4) {
        const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(r, (int)(at + 4 * i), (int)more, 0);
#pragma unroll
        for (int c = 0; c < 4; c++) w[i + c] = v[c];
    }
    if constexpr (N % 4 == 3) {
        typedef uint32_t u32x3 __attribute__((ext_vector_type(3)));
        const u32x3 v = __builtin_amdgcn_raw_buffer_load_b96(r, (int)at, (int)more, 0);
        w[0] = v[0], w[1] = v[1], w[2] = v[2];
    } else if constexpr (N % 4 == 2) {
        const auto v = __builtin_amdgcn_raw_buffer_load_b64(r, (int)at, (int)more, 0);
        w[0] = v[0], w[1] = v[1];
    } else if constexpr (N == 1) {
        w[0] = __builtin_amdgcn_raw_buffer_load_b32(r, (int)at, (int)more, 0);
    }
}
__device__ __forceinline__ uint32_t load_half_from(const uint8_t *base, uint32_t at, uint32_t more) {
    return __builtin_amdgcn_raw_buffer_load_b16(__builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(base), 0, -1, 0x00020000),
                                                (int)at, (int)more, 0);
}

// Workgroups that a CU holds at once (by registers).
template <int W, bool PG16>
constexpr int kResident = W > 4 ? (PG16 ? 2 : 1) : 3;

// W: bytes of a unit; GS: steps of 32 elements of a group.
// PG16: page_size is a multiple of 16, so 16 keys from a multiple of 16 lie in
// one page: a scalar table entry and scalar addresses serve them, and lanes
// add offsets that stay the same for the whole item.  (Without it every key has
// an entry and an address of its own: 128 requests 411 us in pages of 28, 239
// in pages of 32; 190 keys 16 and 13.)
template <int W, int GS, bool PG16>
__global__ __launch_bounds__(256, (kResident<W, PG16>)) void attend4_kernel(Attend4Args g) {
    constexpr int NG = W / GS, VD = (W + 3) / 4;
    constexpr int row_floats = 32 * W + 4;
    // o [waves][gt][32 W + 4], in its place before, for each wave, its queries as
    // the products take them, and (m, l) [waves][16]; all start at 16 bytes, and
    // so does each row of o
    extern __shared__ __align__(16) float lds[];
    float2 *lds_stat = reinterpret_cast<float2 *>(lds + kWaves * g.wave_floats);
    const int D = g.c.head_dim;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int lane = threadIdx.x & 63;
    const int items = g.c.kv_heads * g.gtiles / g.nh;  // items of a token
    const int hw = wave / g.nsub, sub = wave - hw * g.nsub;

    Share w;
    if (!share_of(g, lane, items, &w)) return;
    w = uniform(w);
    const uint64_t first = w.cur, stop = w.stop, per = w.per;
    uint64_t cur = w.cur;
    int64_t t = w.t;
    Keys k = w.k;
    int item = w.item, tokens = 1;
    uint32_t unit = w.unit;
    if (g.block > 1) k = keys_at(g, t, lane, &tokens);

    // A SIMD prefers its oldest wave, which then ends long before the others
    // and leaves them alone with their latencies (shares of one length ended
    // between 116 and 274 us): a wave that is through a quarter of its share
    // gives way to those that are not (128 requests: 251 us without, 239 with;
    // 128 tokens of four prompts 110 and 104, 32 ragged requests 42.5 and 41.5).
    const uint32_t quarter = (uint32_t)(stop - first) * kPair / 4 + 1;
    uint32_t taken = 0;
    __builtin_amdgcn_s_setprio(3);
    while (cur < stop) {
        // (the empty asm: nothing that follows from the lane is kept in registers
        // from one item to the next)
        asm volatile("" : "+v"(lane));
        const int col = lane & 15, lg = lane >> 4;  // columns: queries
        const bool q8 = ((reinterpret_cast<uintptr_t>(g.a.q) | (uintptr_t)(g.a.q_strides[0] * 2) | (uintptr_t)(g.a.q_strides[1] * 2)) & 7) == 0;
        const bool o16 = ((reinterpret_cast<uintptr_t>(g.a.out) | (uintptr_t)(g.a.out_strides[0] * 2) | (uintptr_t)(g.a.out_strides[1] * 2)) & 15) == 0;
        // (W == 3: the last unit is read from a byte earlier, so that its word ends with the row)
        const int v_at = W == 3 && col == 15 ? 44 : W * col, v_shift = W == 3 && col == 15 ? 8 : 0;

        const uint64_t left = stop - cur;
        const uint32_t n = k.units - unit < left ? k.units - unit : (uint32_t)left;
        const int ht = item * g.nh + hw, kvh = g.gtiles == 1 ? ht : ht / g.gtiles, gt0 = (ht - kvh * g.gtiles) * 16;  // first query head of the tile
        const int cols = tokens > 1 ? tokens * g.group : g.group - gt0 < 16 ? g.group - gt0 : 16;
        const int64_t row = g.a.rows ? (int64_t)__builtin_amdgcn_readfirstlane(g.a.rows[t]) : t;

        // this column's query, and the keys its token sees
        u32x4 *const q = reinterpret_cast<u32x4 *>(lds + wave * g.wave_floats);  // [W][lanes]
        const int j = tokens > 1 && col < cols ? col / g.group : 0;
        uint2 raw[W][2];  // elements 32 s + 16 h + 4 lg .. + 3
        {
            // (columns and elements that there are not: the first one's again, cleared below)
            const int head = col < cols ? col - j * g.group : 0;
            const uint16_t *p = (const uint16_t *)g.a.q + (t + j) * g.a.q_strides[0] + ((int64_t)kvh * g.group + gt0 + head) * g.a.q_strides[1];
            if (q8) {
#pragma unroll
                for (int x = 0; x < 2 * W; x++) {
                    const int d = 16 * x + 4 * lg;
                    raw[x / 2][x % 2] = *reinterpret_cast<const uint2 *>(p + (d < D ? d : 0));
                }
            } else {
#pragma unroll
                for (int x = 0; x < 2 * W; x++) {
                    const int d = 16 * x + 4 * lg;
                    const uint16_t *e = p + (d < D ? d : 0);
                    raw[x / 2][x % 2] = uint2{(uint32_t)e[0] | (uint32_t)e[1] << 16, (uint32_t)e[2] | (uint32_t)e[3] << 16};
                }
            }
        }
        float qs[NG], unscale;  // sums of the groups' elements, multiplied; scale2 / the query's power of two
        int begin = k.begin, end = k.end, most_begin = k.begin, least_end = k.end;

        const ConstInts table = (ConstInts)(g.a.block_table + row * g.a.table_stride);
        const uint8_t *kbase = (const uint8_t *)g.c.k_codes + kvh * g.c.k_code_strides[2];
        const uint8_t *vbase = (const uint8_t *)g.c.v_codes + kvh * g.c.v_code_strides[2];
        const uint8_t *ksbase = (const uint8_t *)((const uint16_t *)g.c.k_scales + kvh * g.c.k_scale_strides[2]);
        const uint8_t *vsbase = (const uint8_t *)((const uint16_t *)g.c.v_scales + kvh * g.c.v_scale_strides[2]);
        const int last = k.end - 1;
        const uint64_t upto = (uint64_t)(unit + n) * (kPair * g.nsub);
        const int tiles = (int)(upto < (uint64_t)k.tiles ? upto : (uint64_t)k.tiles);
        const int step = g.nsub;
        int pass = (int)unit * (kPair * g.nsub) + sub;
        const uint32_t key_first = (uint32_t)k.tile0 * kTile;

        f32x4 o[2 * W];
        float m = -__builtin_inff(), l = 0.f, mids[NG];  // mids: sum p mid
#pragma unroll
        for (int e = 0; e < 2 * W; e++) o[e] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NG; i++) mids[i] = 0.f;

        // what a wave holds of a pass until it is taken
        uint32_t kc[2][W];   // units 4 lg .. of keys 16 tau + col
        uint32_t vc[8][VD];  // unit col of keys 16 tau + 4 lg + i, as 4 tau + i
        uint32_t kp[2][NG], vp[2][NG];  // (scale, low) of key and value 16 tau + 4 lg + lane % 4
        uint32_t seen8 = 0xff;     // which of this column's eight keys lie in a page of the cache
        int32_t page[2];           // with PG16: the pages of the next pass to load

        // keys past the last are taken as the last (with PG16 the first key of
        // sixteen stands for all: they lie in its page also where the last key
        // ends inside it)
        const uint32_t limit = (uint32_t)(PG16 ? last & ~15 : last);
        auto entry = [&](uint32_t key) -> int32_t { return table[quotient(key < limit ? key : limit, g.page)]; };
        auto inside = [&](uint32_t key) -> uint32_t {  // a key's slot in its page
            key = key < limit ? key : limit;
            return key - quotient(key, g.page) * g.page.d;
        };
        auto known = [&](int32_t pg) -> int64_t { return (uint32_t)pg < (uint64_t)g.c.pages ? (int64_t)pg : 0; };
        auto key_of = [&](int ps, int tau) -> uint32_t { return key_first + (uint32_t)ps * kTile + 16 * tau; };
        auto load_entries = [&](int ps) {
            if constexpr (PG16) {
#pragma unroll
                for (int tau = 0; tau < 2; tau++) page[tau] = entry(key_of(ps, tau));
            }
        };
        // (with PG16 strides are those of the keys and the values, and 32-bit)
        const uint32_t slot = (uint32_t)g.c.k_code_strides[1], scale_slot = (uint32_t)g.c.k_scale_strides[1] * 2;
        const uint32_t k_at = (uint32_t)col * slot + lg * 4 * W, v_first = 4 * lg * slot + v_at;
        const uint32_t s_at = (4 * lg + (lane & 3)) * scale_slot;
        auto code_place = [&](uint32_t key, int32_t pg) -> uint64_t {
            return (uint64_t)(uint32_t)known(pg) * (uint32_t)g.c.k_code_strides[0] + inside(key) * slot;
        };
        auto scale_place = [&](uint32_t key, int32_t pg) -> uint64_t {
            return (uint64_t)(uint32_t)known(pg) * (uint32_t)(g.c.k_scale_strides[0] * 2) + inside(key) * scale_slot;
        };
        auto load_k = [&](int ps) {
#pragma unroll
            for (int tau = 0; tau < 2; tau++) {
                const uint32_t key = key_of(ps, tau);
                if constexpr (PG16) {
                    load_from<W>(kc[tau], kbase + code_place(key, page[tau]), k_at, 0);
                } else {
                    const uint32_t x = key + col;
                    load_words<W>(kc[tau], kbase + known(entry(x)) * g.c.k_code_strides[0] + (int64_t)inside(x) * g.c.k_code_strides[1] + lg * 4 * W);
                }
            }
        };
        auto load_pairs = [&](uint32_t *pair, const uint8_t *p) {
            if constexpr (W == 8) {  // (only vectors past 128 elements may have fewer groups than steps)
#pragma unroll
                for (int i = 0; i < NG; i++) pair[i] = reinterpret_cast<const uint32_t *>(p)[i < g.groups ? i : g.groups - 1];
            } else {
                load_words<NG>(pair, p);
            }
        };
        auto load_v = [&](int ps) {
#pragma unroll
            for (int tau = 0; tau < 2; tau++) {
                if constexpr (PG16) {
                    const uint64_t at = scale_place(key_of(ps, tau), page[tau]) + s_at;
                    load_pairs(kp[tau], ksbase + at);
                    load_pairs(vp[tau], vsbase + at);
                } else {
                    const uint32_t x = key_of(ps, tau) + 4 * lg + (lane & 3);
                    const int64_t pg = known(entry(x)), in = inside(x);
                    load_pairs(kp[tau], ksbase + 2 * (pg * g.c.k_scale_strides[0] + in * g.c.k_scale_strides[1]));
                    load_pairs(vp[tau], vsbase + 2 * (pg * g.c.v_scale_strides[0] + in * g.c.v_scale_strides[1]));
                }
            }
            seen8 = 0;
#pragma unroll
            for (int tau = 0; tau < 2; tau++) {
                const uint32_t key = key_of(ps, tau);
                const uint8_t *p = vbase;
                if constexpr (PG16) {
                    p += code_place(key, page[tau]);
                    if ((uint32_t)page[tau] < (uint64_t)g.c.pages) seen8 |= 0xfu << 4 * tau;
                }
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    uint32_t *dst = vc[4 * tau + i];
                    if constexpr (PG16 && W != 3) {
                        if constexpr (W == 2) dst[0] = load_half_from(p, v_first, i * slot);
                        else load_from<VD>(dst, p, v_first, i * slot);
                    } else {
                        const uint8_t *x = p + (v_first + i * slot);
                        if constexpr (!PG16) {
                            const uint32_t y = key + 4 * lg + i;
                            const int32_t pg = entry(y);
                            x = p + known(pg) * g.c.v_code_strides[0] + (int64_t)inside(y) * g.c.v_code_strides[1] + v_at;
                            seen8 |= (uint32_t)((uint32_t)pg < (uint64_t)g.c.pages) << (4 * tau + i);
                        }
                        if constexpr (W == 2) dst[0] = *reinterpret_cast<const uint16_t *>(x);
                        else if constexpr (W == 3) __builtin_memcpy(dst, x, 4);
                        else load_words<VD>(dst, x);
                    }
                }
            }
        };

        if (pass < tiles) {
            load_entries(pass);
            load_k(pass);
            load_v(pass);
            load_entries(pass + step);
        }
        {
            float x[W][8];
            uint32_t most = 0;  // the largest of the elements' bits but for their signs, in each half
#pragma unroll
            for (int y = 0; y < 2 * W; y++) {
                uint2 &w2 = raw[y / 2][y % 2];
                if (col >= cols || 16 * y + 4 * lg >= D) w2 = uint2{0u, 0u};
                typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
                auto more = [&](uint32_t v) {
                    most = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, most), __builtin_bit_cast(u16x2, v & 0x7fff7fffu)));
                };
                more(w2.x);
                more(w2.y);
            }
            most = most >> 16 > (most & 0xffff) ? most >> 16 : most & 0xffff;
            float top;
            if (g.bf) {
#pragma unroll
                for (int y = 0; y < 2 * W; y++) {
                    const uint2 v = raw[y / 2][y % 2];
                    float *dst = &x[y / 2][4 * (y % 2)];
                    dst[0] = __uint_as_float(v.x << 16), dst[1] = __uint_as_float(v.x & 0xffff0000u);
                    dst[2] = __uint_as_float(v.y << 16), dst[3] = __uint_as_float(v.y & 0xffff0000u);
                }
                top = __uint_as_float(most << 16);
            } else {
#pragma unroll
                for (int y = 0; y < 2 * W; y++) {
                    const f16x2 v0 = __builtin_bit_cast(f16x2, raw[y / 2][y % 2].x), v1 = __builtin_bit_cast(f16x2, raw[y / 2][y % 2].y);
                    float *dst = &x[y / 2][4 * (y % 2)];
                    dst[0] = (float)v0[0], dst[1] = (float)v0[1], dst[2] = (float)v1[0], dst[3] = (float)v1[1];
                }
                top = load16<false>((uint16_t)most);
            }
            const float odd = column_sum(top * 0.f);  // NaN where an element is not finite
            const int up = 15 - __builtin_amdgcn_frexp_expf(column_max(top));
            unscale = ldexpf(g.scale2, -up) + odd;
            float sums[NG] = {};  // (of the elements as multiplied: no sum of finite ones overflows)
#pragma unroll
            for (int s = 0; s < W; s++) {
                float y[8];
#pragma unroll
                for (int c = 0; c < 8; c++) {
                    y[c] = ldexpf(x[s][c], up);
                    sums[s / GS] += y[c];
                }
                u32x4 v;
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    // elements 4 lg + 0, 1; 16 on; 4 lg + 2, 3; 16 on
                    const int e = c == 0 ? 0 : c == 1 ? 4 : c == 2 ? 2 : 6;
                    v[c] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{y[e], y[e + 1]}, f16x2));
                }
                q[64 * s + lane] = v;
            }
            __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
#pragma unroll
            for (int i = 0; i < NG; i++) qs[i] = column_sum(sums[i]);
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
        for (; pass < tiles; pass += step) {
            if (g.nsub == 1) __builtin_amdgcn_s_barrier();  // (each wave has a head, and all the same tiles)
            taken++;
            if (taken == quarter) __builtin_amdgcn_s_setprio(2);
            else if (taken == 2 * quarter) __builtin_amdgcn_s_setprio(1);
            else if (taken == 3 * quarter) __builtin_amdgcn_s_setprio(0);
            // scores: lane (col, lg) gets those of its eight keys
            float x[8];
            each<NG>([&](auto group) {
                constexpr int C = group.value;
                f32x4 acc[2];
#pragma unroll
                for (int tau = 0; tau < 2; tau++) acc[tau] = f32x4{0.f, 0.f, 0.f, 0.f};
                each<GS>([&](auto b) {
                    constexpr int B = C * GS + b.value;
                    const u32x4 qb = q[64 * B + lane];
#pragma unroll
                    for (int tau = 0; tau < 2; tau++) {
                        const uint32_t y = two_bytes<B, W + B>(kc[tau]), z = two_bytes<2 * W + B, 3 * W + B>(kc[tau]);
                        acc[tau] = mfma16(u32x4{low_codes(y), high_codes(y), low_codes(z), high_codes(z)}, qb, acc[tau]);
                    }
                });
                float sc[2], mid[2];
#pragma unroll
                for (int tau = 0; tau < 2; tau++) {
                    const f16x2 v = __builtin_bit_cast(f16x2, kp[tau][C]);
                    sc[tau] = (float)v[0];
                    mid[tau] = fmaf((float)v[0], 8.f, (float)v[1]);
                }
                each<8>([&](auto i) {
                    constexpr int I = i.value, T = I >> 2;
                    if constexpr (C == 0) x[I] = from_quad<(I & 3)>(sc[T]) * acc[T][I & 3];
                    else x[I] = sum_from_quad<(I & 3)>(sc[T], acc[T][I & 3], x[I]);
                });
                add_each_from_quads(x, mid[0], mid[1], qs[C]);
            });
            __builtin_amdgcn_sched_barrier(0);
            load_k(pass + step);  // (past the end: the last keys again)
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] *= unscale;

            const int key0 = (int)key_of(pass, 0);
            const bool masked = (key0 < most_begin) | (key0 > least_end - kTile) | !__all(seen8 == 0xffu);
            uint32_t in8 = 0xff;  // which of the lane's keys its column sees
            if (masked) {
                asm volatile("");  // (a branch: passes at the ends of a range are few)
                in8 = 0;
                const int mine = key0 + 4 * lg;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int key = mine + 16 * (i >> 2) + (i & 3);
                    const bool in = key >= begin && key < end && (seen8 >> i & 1) != 0;
                    in8 |= (uint32_t)in << i;
                    if (!in) x[i] = -__builtin_inff();
                }
                asm volatile("" : "+v"(in8));  // (kept as bits)
            }
            float expo[2];
#pragma unroll
            for (int tau = 0; tau < 2; tau++) {
                float size = 0.f;
#pragma unroll
                for (int i = 0; i < NG; i++) size = fmaxf(size, fabsf((float)__builtin_bit_cast(f16x2, vp[tau][i])[0]));
                expo[tau] = (float)__builtin_amdgcn_frexp_expf(size);
            }
            float top = -__builtin_inff();
            each<8>([&](auto i) { top = fmaxf(top, x[i.value] + from_quad<(i.value & 3)>(expo[i.value >> 2])); });
            top = fmaxf(fmaxf(column_max(top), kLeast), m);
            if (__any(top > m)) {
                const float keep = __builtin_amdgcn_exp2f(m - top);
                l *= keep;
#pragma unroll
                for (int i = 0; i < NG; i++) mids[i] *= keep;
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
                float sc[2], mid[2];
#pragma unroll
                for (int tau = 0; tau < 2; tau++) {
                    const f16x2 v = __builtin_bit_cast(f16x2, vp[tau][C]);
                    sc[tau] = (float)v[0] * 0x1p15f;  // (held so, as FP16)
                    mid[tau] = fmaf((float)v[0], 8.f, (float)v[1]);
                }
                float weight[8], sum = 0.f;
                add_from_quads(sum, mid[0], mid[1], x);
                each<8>([&](auto i) { weight[i.value] = from_quad<(i.value & 3)>(sc[i.value >> 2]) * x[i.value]; });
                // (taken here, not once for each side of the branch, where they lose the broadcast that a product takes in)
                asm volatile("" : "+v"(weight[0]), "+v"(weight[1]), "+v"(weight[2]), "+v"(weight[3]), "+v"(weight[4]),
                             "+v"(weight[5]), "+v"(weight[6]), "+v"(weight[7]));
                if (masked) {  // once more without the hidden keys, whose numbers may be anything
                    asm volatile("");
                    sum = 0.f;
                    each<8>([&](auto i) {
                        const bool in = in8 >> i.value & 1;
                        const float scale = from_quad<(i.value & 3)>(sc[i.value >> 2]), middle = from_quad<(i.value & 3)>(mid[i.value >> 2]);
                        weight[i.value] = in ? scale * x[i.value] : 0.f;
                        sum += in ? middle * x[i.value] : 0.f;
                    });
                }
                mids[C] += sum;
                u32x4 part[2];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const f16x2 big = __builtin_convertvector(f32x2{weight[2 * i], weight[2 * i + 1]}, f16x2);
                    const f16x2 small = __builtin_convertvector(f32x2{rest<0>(weight[2 * i], big), rest<1>(weight[2 * i + 1], big)}, f16x2);
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
                        even[i] = low_codes(y);
                        odd[i] = high_codes(y);
                    }
#pragma unroll
                    for (int z = 0; z < 2; z++) {
                        o[2 * B] = mfma16(even, part[z], o[2 * B]);
                        o[2 * B + 1] = mfma16(odd, part[z], o[2 * B + 1]);
                    }
                });
            });
            __builtin_amdgcn_sched_barrier(0);
            load_v(pass + step);
            load_entries(pass + 2 * step);
            __builtin_amdgcn_sched_barrier(0);
        }

        // join the waves of each head tile
        l = column_sum(l);
#pragma unroll
        for (int i = 0; i < NG; i++) mids[i] = column_sum(mids[i]);
        if (col < cols) {
            float *dst = lds + wave * g.wave_floats + col * row_floats + 4 * lg;
#pragma unroll
            for (int e = 0; e < 2 * W; e++) {
                constexpr float f = 0x1p-15f;  // (the weights' 2^15)
                const float b = mids[e / (2 * GS)];
                *reinterpret_cast<f32x4 *>(dst + 16 * e) = f32x4{fmaf(o[e][0], f, b), fmaf(o[e][1], f, b), fmaf(o[e][2], f, b), fmaf(o[e][3], f, b)};
            }
            if (lg == 0) lds_stat[wave * 16 + col] = float2{m, l};
        }
        __syncthreads();
        finish_item(g, wave * 64 + lane, lds, lds_stat, row_floats, g.wave_floats, o16, first, cur, per, t, tokens, k, item, unit, n);
        __syncthreads();
        cur = uniform64(cur + n);
        unit = 0;
        if (++item == items) {
            item = 0;
            t = uniform64(t + tokens);
            if (cur < stop) k = keys_at(g, t, lane, &tokens);
        }
    }
}

// Whether sixteen keys lie in one page, keys and values lie alike, and a
// page's offsets are 32-bit.
bool by_sixteen(const orth_hip_int4_cache_t &c) {
    constexpr int64_t most = (int64_t)1 << 31;
    for (int i = 0; i < 2; i++)
        if (c.k_code_strides[i] != c.v_code_strides[i] || c.k_scale_strides[i] != c.v_scale_strides[i]) return false;
    return c.page_size % 16 == 0 && c.k_code_strides[0] < most && c.k_scale_strides[0] < most / 2 &&
           c.k_code_strides[1] < most / c.page_size && c.k_scale_strides[1] < most / 2 / c.page_size;
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
    // Neighbouring tokens share a product where some request must have several:
    // more tokens than requests.  (A table of more rows than tokens may have
    // several of one request too, which the host cannot see: 128 tokens of four
    // prompts 103 us with up to 511 rows, 249 with 512.)
    g.block = 1;
    if (a.rows && a.tokens > a.table_rows)
        while (2 * g.block * g.group <= 16) g.block *= 2;
    g.gt = g.block * g.group < 16 ? g.block * g.group : 16;
    // The pieces of a full tile are twice as long, so there neighbouring heads
    // go together from two items a CU on, else from one for four CUs (8 key
    // heads with 16 columns each; one, two and four heads a workgroup: 1,024
    // items of a head, 128 tokens of four prompts 108, 110 and 136 us, 8 tokens
    // of 64 prompts 130, 106 and 116; 128 requests of 2,048 to 16,384 keys, the
    // call that would rather have four, 395, 283 and 266; 4,096 items, 512
    // tokens of four prompts: 336, 309 and 309).
    attend_tiles(g, g.gt > 8 ? 2 * cus : cus / 4, (a.tokens + g.block - 1) / g.block);
    const int resident = by_sixteen(c) ? c.head_dim > 128 ? kResident<8, true> : kResident<4, true>
                                       : c.head_dim > 128 ? kResident<8, false> : kResident<4, false>;
    *groups = attend_groups(g, (int64_t)cus * resident, g.block);
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
        const int rows = g.gt * (32 * W + 4), queries = 256 * W;
        g.wave_floats = rows > queries ? rows : queries;
        const size_t lds = (size_t)kWaves * g.wave_floats * 4 + kWaves * 16 * sizeof(float2);
        auto go = [&](auto kernel) -> hipError_t {
            if (lds > 48 * 1024) {
                hipError_t s = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                                   hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
                if (s != hipSuccess) return s;
            }
            kernel<<<dim3((unsigned)groups), 256, lds, stream>>>(g);
            return hipGetLastError();
        };
        return by_sixteen(c) ? go(attend4_kernel<W, GS, true>) : go(attend4_kernel<W, GS, false>);
    });
    if (e != hipSuccess) return e;
    return attend_joins(g, groups, g.block) ? launch_join(g, groups, stream) : hipSuccess;
}

}  // namespace orth
