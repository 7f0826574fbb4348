// Attention of single tokens over the paged cache.
//
// One pass over the keys with a running maximum m and sum l of the softmax:
// a tile of 32 keys gives scores s (scaled to base 2), m' = max(m, s), p =
// 2^(s - m'), and the sums l and o = sum p v are scaled by 2^(m - m') where
// m rises; the result is o / l.
//
// A wave takes a tile from registers alone, as two matrix products over
// v_mfma_f32_16x16x32 (the query heads that share a key head are the 16
// columns, zeros where there are fewer):
//
//   scores  S^T = K Q^T.  The A operand's row and eight elements are a lane's
//           16-byte load of one key, so keys go from the cache to the
//           operand.  Row 4 g + i of product tau is key 8 g + 4 tau + i of the
//           tile: then the scores a lane gets (rows 4 g + i of its lane group
//           g, both products) are those of keys 8 g .. 8 g + 7.
//   values  O^T = V^T P^T.  These eight are the B operand's elements of that
//           lane, so the weights never leave their lane.  The A operand wants
//           eight keys of one element per lane: a lane loads 8 keys x EL
//           elements (a key's vector lies across 16 lanes) and transposes
//           them in registers, one v_perm_b32 per two values.
//
// The weights enter the second product as FP32 values do: as 16-bit parts,
// three in BF16 and two in FP16 (split_pair), whose products with the values
// are exact and add up in FP32.  FP16 ones are held 2^14 times larger, which
// keeps the parts of small weights normal numbers, BF16 ones 2^16 times
// smaller: sums of 2^16 of the type's largest numbers do not overflow before
// they are divided by l, and products with its smallest are numbers of FP32.
//
// Bound by reading the cache once, cut evenly over the resident workgroups
// (orth_attend.h).
//
// Measured (one MI355X, a call among others, inputs from HBM): 128 requests
// of 2,048 to 16,384 keys, 8 of 64 heads of 128, BF16: 585 us, 5.7 TB/s (what
// a kernel that only reads reaches); 32 ragged requests up to 4,096 keys, 32
// heads, FP16: 73.2 us, 4.6 TB/s; one of 32,768 keys, 8 of 32 heads: 37.0 us
// (32 the keys, 5 the join of 64 pieces a key head), 3.6 TB/s; one of 190
// keys, 32 heads: 8.7 us, a chain of latencies (position 1.2, share 0.7, table
// 1.6, keys 2, join 1).  HBM reads by counter: 3.37 GB, 344 MB and 135 MB for
// the first three, as their keys and values.  Several tokens of one request
// read its keys each for itself (2,048 tokens of one prompt: 836 us).
// A wave per query head on the vector unit (no matrix products, no split)
// took 35,500, 7,900, 57,500 and 164 us.
#include "orth_attend.h"

namespace orth {

namespace {

template <bool BF>
struct Attend16 : AttendArgs<orth_hip_cache_t> {
    static constexpr bool blocks = false;
    static __device__ __forceinline__ uint16_t round(float v) { return store16<BF>(v); }
};

template <bool BF>
__device__ __forceinline__ f32x4 mfma(const u32x4 &a, const u32x4 &b, const f32x4 &c) {
    if constexpr (BF)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Two weights as pairs of 16-bit parts, part[0] the largest.  BF16: three
// parts of eight bits each, cut off, whose sum is the FP32 weight exactly.
// FP16: two parts of eleven bits, rounded to nearest (the second one's sign is
// a bit more): 2^-24 of the weight, as an FP32 operation's rounding, or 2^-39
// of the largest weight where that is more.
template <bool BF>
constexpr int kParts = BF ? 3 : 2;
template <bool BF>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t part[kParts<BF>]) {
    if constexpr (BF) {
#pragma unroll
        for (int k = 0; k < 3; k++) {
            const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
            part[k] = __builtin_amdgcn_perm(b, a, 0x07060302u);
            x -= __uint_as_float(a & 0xffff0000u);
            y -= __uint_as_float(b & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 2; k++) {
            typedef f16 f16x2 __attribute__((ext_vector_type(2)));
            f16x2 h = {(f16)x, (f16)y};
            // (a first part is not zero, so that a weight times an infinite
            // value is infinite; the second part takes it back)
            if (k == 0) h = __builtin_elementwise_max(h, f16x2{(f16)0x1p-24f, (f16)0x1p-24f});
            part[k] = __builtin_bit_cast(uint32_t, h);
            x -= (float)h[0];
            y -= (float)h[1];
        }
    }
}

// 16-bit elements with infinities (and NaN) as the type's largest numbers: what
// the parts behind the first of a split factor are multiplied with.  A zero
// part times an infinity would be a NaN, and one of the other sign would turn
// the first part's infinity into one.  (As whole numbers, values without a
// sign bit lie below 2^15 in order, those with one above.)
template <bool BF>
__device__ __forceinline__ u32x4 finite16(u32x4 v) {
    typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
    typedef int16_t i16x8 __attribute__((ext_vector_type(8)));
    constexpr int16_t most = BF ? 0x7f7f : 0x7bff;
    const u16x8 u = __builtin_elementwise_min(__builtin_bit_cast(u16x8, v), (u16x8)(uint16_t)(most | 0x8000));
    return __builtin_bit_cast(u32x4, __builtin_elementwise_min(__builtin_bit_cast(i16x8, u), (i16x8)most));
}

// KS: steps of 32 elements over head_dim; PG8: page_size is a multiple of 8,
// so eight keys from a multiple of 8 lie in one page and one table entry
// serves them; TAIL: head_dim is not KS * 32.
template <int KS, bool BF, bool PG8, bool TAIL>
__global__ __launch_bounds__(256, KS > 4 ? 1 : KS > 2 ? 2 : 3) void attend_kernel(Attend16<BF> g) {
    constexpr int EL = KS <= 2 ? 4 : KS <= 4 ? 8 : 16;  // elements of a value vector per lane
    constexpr int VW = EL / 2;                          // words of them
    constexpr bool VTAIL = TAIL || 16 * EL != 32 * KS;
    constexpr float kHeld = BF ? 0x1p-16f : 0x1p14f;  // (multiplied, not added to the exponent, which would lose its low bits)
    // o [waves][gt][16 EL + 4], then (m, l) [waves][16]; both start at 16 bytes, and so does each row of o
    extern __shared__ __align__(16) float lds[];
    static_assert((16 * EL + 4) % 4 == 0, "rows of o");
    const int D = g.c.head_dim, row_floats = 16 * EL + 4;
    float2 *lds_stat = reinterpret_cast<float2 *>(lds + kWaves * g.gt * row_floats);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, lg = lane >> 4;
    const int items = g.c.kv_heads * g.gtiles / g.nh;  // items of a token
    const int hw = wave / g.nsub, sub = wave - hw * g.nsub;

    Share w;
    if (!share_of(g, lane, items, &w)) return;
    // (in scalar registers some 20 vector registers fewer are used.  Without
    // PG8, whose loop needs them for its addresses, that is faster: a prompt of
    // 2,048 tokens, 8 of 32 heads, FP16, pages of 7, 1,251 us and 1,008, 32
    // requests of 16 to 2,000 keys, 16 heads of 64, 21.5 and 20.3.  With it the
    // items' starts and ends get slower: the prompt, BF16, pages of 16, 836 and
    // 867, the 32 requests 16.6 and 17.0.)
    if constexpr (!PG8) w = uniform(w);
    const uint64_t first = w.cur, stop = w.stop, per = w.per;
    uint64_t cur = w.cur;
    int64_t t = w.t;
    Keys k = w.k;
    int item = w.item;
    uint32_t unit = w.unit;

    const int64_t k_slot = g.c.k_strides[1], v_slot = g.c.v_strides[1];
    const bool q16 = ((reinterpret_cast<uintptr_t>(g.a.q) | (uintptr_t)(g.a.q_strides[0] * 2) | (uintptr_t)(g.a.q_strides[1] * 2)) & 15) == 0;
    const bool o16 = ((reinterpret_cast<uintptr_t>(g.a.out) | (uintptr_t)(g.a.out_strides[0] * 2) | (uintptr_t)(g.a.out_strides[1] * 2)) & 15) == 0;

    while (cur < stop) {
        const uint64_t left = stop - cur;
        const uint32_t n = k.units - unit < left ? k.units - unit : (uint32_t)left;
        const int ht = item * g.nh + hw, kvh = g.gtiles == 1 ? ht : ht / g.gtiles, gt0 = (ht - kvh * g.gtiles) * 16;  // first query head of the tile
        const int cols = g.group - gt0 < 16 ? g.group - gt0 : 16;
        const int64_t q_head = (int64_t)kvh * g.group + gt0;

        // the queries: column col, elements 32 j + 8 lg .. + 7
        u32x4 q[KS];
#pragma unroll
        for (int j = 0; j < KS; j++) {
            const int d = 32 * j + 8 * lg;
            q[j] = u32x4{0u, 0u, 0u, 0u};
            if (col < cols && (!TAIL || d < D)) {
                const uint16_t *p = (const uint16_t *)g.a.q + t * g.a.q_strides[0] + (q_head + col) * g.a.q_strides[1] + d;
                if (q16) {
                    q[j] = *reinterpret_cast<const u32x4 *>(p);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) q[j][e] = (uint32_t)p[2 * e] | (uint32_t)p[2 * e + 1] << 16;
                }
            }
        }

        const int64_t row = g.a.rows ? (int64_t)g.a.rows[t] : t;
        const int32_t *table = g.a.block_table + row * g.a.table_stride;
        const uint16_t *kbase = (const uint16_t *)g.c.k_cache + kvh * g.c.k_strides[2];
        const uint16_t *vbase = (const uint16_t *)g.c.v_cache + kvh * g.c.v_strides[2];
        const int last = k.end - 1;
        const uint64_t upto = (uint64_t)(unit + n) * (kPair * g.nsub);
        const int step = g.nsub, tile_end = k.tile0 + (int)(upto < (uint64_t)k.tiles ? upto : (uint64_t)k.tiles);
        int tile = k.tile0 + (int)unit * (kPair * g.nsub) + sub;

        f32x4 o[EL];
        float m = -__builtin_inff(), l = 0.f;
#pragma unroll
        for (int e = 0; e < EL; e++) o[e] = f32x4{0.f, 0.f, 0.f, 0.f};

        // a key's page (-1: outside the cache) and its address, in elements
        // from the head's base; keys past the last are taken as the last
        auto entry = [&](int key) -> int32_t { return table[quotient((uint32_t)(key < last ? key : last), g.page)]; };
        auto place = [&](int key, int32_t page, const int64_t *strides) -> int64_t {
            key = key < last ? key : last;
            const uint32_t in = (uint32_t)key - quotient((uint32_t)key, g.page) * g.page.d;
            return ((uint32_t)page < (uint64_t)g.c.pages ? (int64_t)page : 0) * strides[0] + (int64_t)in * strides[1];
        };
        // (with PG8 the first key of a group of eight stands for all: the
        // group lies in its page also where the last key ends inside it)
        const int last8 = last & ~7;
        auto entry8 = [&](int key) -> int32_t { return table[quotient((uint32_t)(key < last8 ? key : last8), g.page)]; };
        auto place8 = [&](int key, int32_t page, const int64_t *strides) -> int64_t {
            key = key < last8 ? key : last8;
            const uint32_t in = (uint32_t)key - quotient((uint32_t)key, g.page) * g.page.d;
            return ((uint32_t)page < (uint64_t)g.c.pages ? (int64_t)page : 0) * strides[0] + (int64_t)in * strides[1];
        };

        u32x4 kf[2][KS];
        uint32_t vf[8][VW];
        uint32_t seen8 = 0xff;  // (without PG8: which of the lane's eight keys lie in a page of the cache)
        int32_t ke = 0, ve = 0, ve_now = 0;

        auto load_k = [&](int tl, int32_t e) {
            const int key = tl * kTile + (col >> 2) * 8;
            const uint16_t *p[2];
            if constexpr (PG8) {
                p[0] = kbase + place8(key, e, g.c.k_strides) + (col & 3) * k_slot;
                p[1] = p[0] + 4 * k_slot;
            } else {
#pragma unroll
                for (int tau = 0; tau < 2; tau++) {
                    const int x = key + 4 * tau + (col & 3);
                    p[tau] = kbase + place(x, entry(x), g.c.k_strides);
                }
            }
#pragma unroll
            for (int tau = 0; tau < 2; tau++)
#pragma unroll
                for (int j = 0; j < KS; j++) {
                    const int d = 32 * j + 8 * lg;
                    kf[tau][j] = *reinterpret_cast<const u32x4 *>(p[tau] + (!TAIL || d < D ? d : 0));
                }
        };
        auto load_v = [&](int tl, int32_t e) {
            const int key = tl * kTile + lg * 8;
            const int d0 = !VTAIL || col * EL < D ? col * EL : 0, d1 = !VTAIL || col * EL + 8 < D ? col * EL + 8 : 0;
            const uint16_t *p = vbase;
            if constexpr (PG8) p += place8(key, e, g.c.v_strides);
            else seen8 = 0;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const uint16_t *x = p;
                if constexpr (PG8) {
                    x += i * v_slot;
                } else {
                    const int32_t pg = entry(key + i);
                    x += place(key + i, pg, g.c.v_strides);
                    seen8 |= (uint32_t)((uint32_t)pg < (uint64_t)g.c.pages) << i;
                }
                if constexpr (EL == 4) {
                    const uint2 w = *reinterpret_cast<const uint2 *>(x + d0);
                    vf[i][0] = w.x;
                    vf[i][1] = w.y;
                } else {
                    const u32x4 w = *reinterpret_cast<const u32x4 *>(x + d0);
#pragma unroll
                    for (int c = 0; c < 4; c++) vf[i][c] = w[c];
                    if constexpr (EL == 16) {
                        const u32x4 z = *reinterpret_cast<const u32x4 *>(x + d1);
#pragma unroll
                        for (int c = 0; c < 4; c++) vf[i][4 + c] = z[c];
                    }
                }
            }
        };

        if (tile < tile_end) {
            if constexpr (PG8) {
                ke = entry8(tile * kTile + (col >> 2) * 8);
                ve = entry8(tile * kTile + lg * 8);
            }
            load_k(tile, ke);
            load_v(tile, ve);
            ve_now = ve;
            if constexpr (PG8) {
                ke = entry8((tile + step) * kTile + (col >> 2) * 8);
                ve = entry8((tile + step) * kTile + lg * 8);
            }
        }
        for (; tile < tile_end; tile += step) {
            const bool more = tile + step < tile_end;
            f32x4 s[2];
#pragma unroll
            for (int tau = 0; tau < 2; tau++) {
                s[tau] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < KS; j++) {
                    u32x4 a = kf[tau][j];
                    if constexpr (TAIL)
                        if (32 * j + 8 * lg >= D) a = u32x4{0u, 0u, 0u, 0u};
                    s[tau] = mfma<BF>(a, q[j], s[tau]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            int32_t ve_next = ve;
            if (more) {
                load_k(tile + step, ke);
                if constexpr (PG8) {
                    ke = entry8((tile + 2 * step) * kTile + (col >> 2) * 8);
                    ve = entry8((tile + 2 * step) * kTile + lg * 8);
                }
            }
            __builtin_amdgcn_sched_barrier(0);

            float x[8];
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = s[i >> 2][i & 3] * g.scale2;
            const int key0 = tile * kTile;
            const bool paged = PG8 ? (uint32_t)ve_now < (uint64_t)g.c.pages : seen8 == 0xff;
            bool any = true;
            if (key0 < k.begin || key0 + kTile > k.end || !__all(paged)) {
                // the keys outside the token's range or the cache: no score,
                // and zero values (0 times an infinity would be a NaN)
                bool here = false;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int key = key0 + 8 * lg + i;
                    const bool in = key >= k.begin && key < k.end && (PG8 ? paged : (seen8 >> i & 1) != 0);
                    here |= in;
                    if (!in) {
                        x[i] = -__builtin_inff();
#pragma unroll
                        for (int c = 0; c < VW; c++) vf[i][c] = 0u;
                    }
                }
                any = __any(here);
            }
            if (any) {
                float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
                top = fmaxf(fmaxf(column_max(top), kLeast), m);
                if (__any(top > m)) {
                    const float keep = __builtin_amdgcn_exp2f(m - top);
                    l *= keep;
#pragma unroll
                    for (int e = 0; e < EL; e++)
#pragma unroll
                        for (int i = 0; i < 4; i++) o[e][i] *= keep;
                    m = top;
                }
                u32x4 p[kParts<BF>];
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const float p0 = kHeld * __builtin_amdgcn_exp2f(x[i] - m), p1 = kHeld * __builtin_amdgcn_exp2f(x[i + 1] - m);
                    l += p0 + p1;
                    uint32_t part[kParts<BF>];
                    split_pair<BF>(p0, p1, part);
#pragma unroll
                    for (int k = 0; k < kParts<BF>; k++) p[k][i >> 1] = part[k];
                }
#pragma unroll
                for (int c = 0; c < VW; c++) {
                    u32x4 a, b;  // elements 2 c and 2 c + 1 of the lane's eight keys
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        a[i] = __builtin_amdgcn_perm(vf[2 * i + 1][c], vf[2 * i][c], 0x05040100u);
                        b[i] = __builtin_amdgcn_perm(vf[2 * i + 1][c], vf[2 * i][c], 0x07060302u);
                    }
#pragma unroll
                    for (int k = 0; k < kParts<BF>; k++) {
                        o[2 * c] = mfma<BF>(a, p[k], o[2 * c]);
                        o[2 * c + 1] = mfma<BF>(b, p[k], o[2 * c + 1]);
                        if (k == 0) {
                            a = finite16<BF>(a);
                            b = finite16<BF>(b);
                        }
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            if (more) load_v(tile + step, ve_next);
            ve_now = ve_next;
            __builtin_amdgcn_sched_barrier(0);
        }
        l = column_sum(l);

        // join the waves of each head tile
        if (col < cols) {
            float *dst = lds + (wave * g.gt + col) * row_floats;
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int e = 0; e < EL; e += 4)
                    *reinterpret_cast<f32x4 *>(dst + (4 * lg + i) * EL + e) = f32x4{o[e][i], o[e + 1][i], o[e + 2][i], o[e + 3][i]};
            if (lg == 0) lds_stat[wave * 16 + col] = float2{m, l};
        }
        __syncthreads();
        finish_item(g, threadIdx.x, lds, lds_stat, row_floats, g.gt * row_floats, o16, first, cur, per, t, 1, k, item, unit, n);
        __syncthreads();
        cur += n;
        unit = 0;
        if (++item == items) {
            item = 0;
            t++;
            if (cur < stop) k = keys_of(g, t);
        }
    }
}

// What both the workspace and the launch go by.
template <bool BF>
Attend16<BF> attend_args(const orth_hip_cache_t &c, const orth_hip_attend_t &a, int cus, int64_t *groups) {
    Attend16<BF> g;
    g.c = c;
    g.a = a;
    g.page = fast_div((uint32_t)c.page_size);
    g.scale2 = a.scale * 1.4426950408889634f;
    g.group = a.q_heads / c.kv_heads;
    g.gtiles = (g.group + 15) / 16;
    g.gt = g.group < 16 ? g.group : 16;
    attend_tiles(g, cus / 4, a.tokens);
    *groups = attend_groups(g, (int64_t)cus * (c.head_dim > 128 ? 1 : c.head_dim > 64 ? 2 : 3));
    return g;
}

template <int KS, bool BF>
hipError_t attend_launch(const Attend16<BF> &g, int64_t groups, size_t lds, hipStream_t stream) {
    const bool pg8 = g.c.page_size % 8 == 0, tail = g.c.head_dim != 32 * KS;
    auto go = [&](auto kernel) -> hipError_t {
        if (lds > 48 * 1024) {
            hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
            if (e != hipSuccess) return e;
        }
        kernel<<<dim3((unsigned)groups), 256, lds, stream>>>(g);
        return hipGetLastError();
    };
    if (!pg8) return go(attend_kernel<KS, BF, false, true>);
    return tail ? go(attend_kernel<KS, BF, true, true>) : go(attend_kernel<KS, BF, true, false>);
}

template <bool BF>
hipError_t attend_by_width(const Attend16<BF> &g, int64_t groups, hipStream_t stream) {
    const int D = g.c.head_dim, el = D <= 64 ? 4 : D <= 128 ? 8 : 16;
    const size_t lds = (size_t)kWaves * g.gt * (16 * el + 4) * 4 + kWaves * 16 * sizeof(float2);
    hipError_t e = D <= 64 ? attend_launch<2, BF>(g, groups, lds, stream)
                 : D <= 96 ? attend_launch<3, BF>(g, groups, lds, stream)
                 : D <= 128 ? attend_launch<4, BF>(g, groups, lds, stream)
                            : attend_launch<8, BF>(g, groups, lds, stream);
    if (e != hipSuccess) return e;
    return attend_joins(g, groups) ? launch_join(g, groups, stream) : hipSuccess;
}

template <bool BF>
hipError_t attend(const orth_hip_cache_t &c, const orth_hip_attend_t &a, int cus, void *work, uint32_t *counters, hipStream_t stream) {
    int64_t groups = 0;
    Attend16<BF> g = attend_args<BF>(c, a, cus, &groups);
    attend_workspace(g, groups, work, counters);
    return attend_by_width<BF>(g, groups, stream);
}

}  // namespace

int64_t attention_workspace_bytes(const orth_hip_cache_t &c, const orth_hip_attend_t &a, int cus, int64_t *groups) {
    int64_t n = 0;
    const Attend16<false> g = attend_args<false>(c, a, cus, &n);
    *groups = attend_units(g) > 1 ? n : 0;  // (items of one unit are not split)
    return attend_bytes(g, n);
}

hipError_t launch_paged_attention(const orth_hip_cache_t &c, const orth_hip_attend_t &a, int cus, void *work, uint32_t *counters,
                                  hipStream_t stream) {
    return c.dtype == ORTH_DT_BF16 ? attend<true>(c, a, cus, work, counters, stream) : attend<false>(c, a, cus, work, counters, stream);
}

}  // namespace orth
