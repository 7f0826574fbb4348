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
// Bound by reading the cache once.  The work is cut evenly over the resident
// workgroups by the keys the tokens really see, which only the device knows:
// every wave sums up the tokens' units (two tiles for each wave that shares a
// head tile: 64, 128 or 256 keys) and finds its workgroup's share (of 128
// tokens in one load and one scan).  A share that ends
// inside a (token, key head) leaves a piece (m, l, o); the workgroup that
// writes an item's last piece joins them, or a second launch where an item
// has many.  Whole items are written at once.
//
// Measured (one MI355X, a call among others, inputs from HBM): 128 requests
// of 2,048 to 16,384 keys, 8 of 64 heads of 128, BF16: 594 us, 5.6 TB/s (a
// kernel that only reads reaches 5.7); 32 ragged requests up to 4,096 keys, 32
// heads, FP16: 73.8 us, 4.6 TB/s; one of 32,768 keys, 8 of 32 heads: 37.3 us
// (32 the keys, 5 the join of 64 pieces a key head), 3.6 TB/s; one of 190
// keys, 32 heads: 8.9 us, a chain of latencies (position 1.2, share 0.7, table
// 1.6, keys 2, join 1).  HBM reads by counter: 3.37 GB, 344 MB and 135 MB for
// the first three, as their keys and values.  Several tokens of one request
// read its keys each for itself (2,048 tokens of one prompt: 853 us).
// A wave per query head on the vector unit (no matrix products, no split)
// took 35,500, 7,900, 57,500 and 164 us.
#include "orth_serve.h"

namespace orth {

namespace {

constexpr int kWaves = 4;
constexpr int kTile = 32;                // keys a wave takes at a time
constexpr int kPair = 2;                 // tiles a wave takes in a unit, the least share of a workgroup
constexpr int kPieces = 16;              // pieces of an item (and one for its ends) that a workgroup joins
constexpr float kLeast = -3.0e38f;       // the maximum of a token that has seen keys, at the least

// Loads run up to two steps of kWaves tiles ahead of the last key: their key
// numbers stay within an int.
static_assert(kMostKeys + (2 * kWaves + 1) * kTile <= INT32_MAX, "a table's keys");

struct AttendArgs {
    orth_hip_cache_t c;
    orth_hip_attend_t a;
    FastDiv page;
    float scale2;        // scale * log2(e)
    int group, gtiles;   // query heads of a key head, and their tiles of 16
    int gt;              // query heads of a tile: min(group, 16)
    int nh, nsub;        // head tiles a workgroup takes at once, and the waves of each: nh * nsub = 4
    float *part;         // pieces [workgroups * 2][nh][gt][head_dim]
    float2 *stat;        // (m, l) [workgroups * 2][nh][16]
    uint32_t *arrived;   // [workgroups], zeros: the pieces written so far of the split item that starts there
    int4 *many;          // [workgroups / kPieces, up]: (token, item, first piece's slot, last workgroup) of an item
                         // of more than kPieces + 1 pieces, or a token of -1: joined by a second launch
};

struct Keys {
    int begin, end;  // the keys a token sees
    int tile0, tiles;
    uint32_t units;
};

// a / b, in 32 bits where both fit (a 64-bit division takes a quarter of a
// microsecond, and a short call is a chain of such latencies).
__device__ __forceinline__ uint64_t div64(uint64_t a, uint64_t b) {
    if ((a | b) >> 32) return a / b;
    return (uint32_t)a / (uint32_t)b;
}

// Memory of all XCDs: written through and read past the L2 of this one.
__device__ __forceinline__ void store_shared(float *p, float a, float b) {
    __hip_atomic_store(reinterpret_cast<uint64_t *>(p), (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a),
                       __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 load_shared(const float *p) {
    const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t *>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return float2{__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32))};
}

__device__ __forceinline__ Keys keys_of(const AttendArgs &g, int64_t t) {
    const int64_t row = g.a.rows ? (int64_t)g.a.rows[t] : t;
    int64_t end = (int64_t)g.a.positions[t] + 1;
    int64_t begin = g.a.window > 0 && end > g.a.window ? end - g.a.window : 0;
    const int64_t held = g.a.table_width * g.c.page_size;
    end = end < held ? end : held;
    if (row < 0 || row >= g.a.table_rows || end <= begin) begin = end = 0;
    Keys k;
    k.begin = (int)begin;
    k.end = (int)end;
    k.tile0 = k.begin / kTile;
    k.tiles = (int)(((int64_t)k.end + kTile - 1) / kTile) - k.tile0;
    const int unit = kPair * g.nsub;
    k.units = k.tiles > unit ? (uint32_t)(k.tiles + unit - 1) / unit : 1;  // (one that sees nothing is written too)
    return k;
}

// Inclusive sums of the units of tokens t0 + 2 lane, + 1, whose keys are in k[2].  (32 bits
// hold them: a token has at most 2^23 units of 256 keys, or 2^22 of 64 where
// the launch has seen that its table holds no more than 2^28 keys, and a scan
// takes 128 tokens.)
constexpr int kScan = 128;
__device__ __forceinline__ uint32_t block_units(const AttendArgs &g, int64_t t0, int lane, Keys k[2]) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int64_t t = t0 + 2 * lane + i;
        k[i] = Keys{0, 0, 0, 0, 0};
        if (t < g.a.tokens) k[i] = keys_of(g, t);
    }
    return wave_scan(k[0].units + k[1].units);
}

// The maximum over the four lanes that hold one column.
__device__ __forceinline__ float column_max(float v) {
    const uint32_t u = __float_as_uint(v);
    const auto h = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t w = __float_as_uint(fmaxf(__uint_as_float(h[0]), __uint_as_float(h[1])));
    const auto q = __builtin_amdgcn_permlane16_swap(w, w, false, false);
    return fmaxf(__uint_as_float(q[0]), __uint_as_float(q[1]));
}
__device__ __forceinline__ float column_sum(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

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
__global__ __launch_bounds__(256, KS > 4 ? 1 : KS > 2 ? 2 : 3) void attend_kernel(AttendArgs g) {
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

    // ------------------------------------------------ this workgroup's share
    Keys mine[2];
    uint32_t incl = 0;
    uint64_t run = 0;
    for (int64_t t0 = 0; t0 < g.a.tokens; t0 += kScan) {
        incl = block_units(g, t0, lane, mine);
        run += (uint32_t)__builtin_amdgcn_readlane((int)incl, 63);
    }
    const uint64_t total = run * items;
    uint64_t per = div64(total + gridDim.x - 1, gridDim.x);
    uint64_t cur = blockIdx.x * per;
    const uint64_t first = cur, stop = cur + per < total ? cur + per : total;
    const bool marks = blockIdx.x % kPieces == 0 && threadIdx.x == 0;
    if (cur >= total) {
        if (marks) g.many[blockIdx.x / kPieces] = int4{-1, 0, 0, 0};
        return;
    }
    const uint64_t want = div64(cur, items);  // the unit, were a token one item
    int64_t t = 0;
    Keys k;
    uint64_t before = 0;  // units of the tokens in front of t
    for (int64_t t0 = 0;; t0 += kScan) {
        if (g.a.tokens > kScan) incl = block_units(g, t0, lane, mine);
        const uint32_t all = (uint32_t)__builtin_amdgcn_readlane((int)incl, 63);
        if (before + all > want) {
            const uint32_t at = (uint32_t)(want - before);
            const int l = __ffsll((unsigned long long)__ballot(incl > at)) - 1;
            const uint32_t end = (uint32_t)__builtin_amdgcn_readlane((int)incl, l);
            const uint32_t u1 = (uint32_t)__builtin_amdgcn_readlane((int)mine[1].units, l);
            const bool second = end - u1 <= at;
            t = t0 + 2 * l + (second ? 1 : 0);
            const Keys &x = second ? mine[1] : mine[0];
            k.begin = __builtin_amdgcn_readlane(x.begin, l);
            k.end = __builtin_amdgcn_readlane(x.end, l);
            k.tile0 = __builtin_amdgcn_readlane(x.tile0, l);
            k.tiles = __builtin_amdgcn_readlane(x.tiles, l);
            k.units = (uint32_t)__builtin_amdgcn_readlane((int)x.units, l);
            before += second ? end - u1 : end - u1 - k.units;
            break;
        }
        before += all;
    }
    const uint64_t inside = cur - before * items;
    int item = (int)div64(inside, k.units);
    uint32_t unit = (uint32_t)(inside - (uint64_t)item * k.units);

    if (marks) {
        // an item of more than kPieces + 1 pieces has a workgroup of these
        // behind its first one, and only one within kPieces of it, at whose
        // start no other item lies: it names the item to the second launch
        const uint64_t u0 = cur - unit;
        const int from = (int)div64(u0, per), to = (int)div64(u0 + k.units - 1, per);
        const bool big = to - from > kPieces && from < (int)blockIdx.x && (int)blockIdx.x - from <= kPieces;
        g.many[blockIdx.x / kPieces] = big ? int4{(int)t, item, from * 2 + (u0 == from * per ? 0 : 1), to} : int4{-1, 0, 0, 0};
    }

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
        const bool whole = n == k.units;
        const int slot = (int)blockIdx.x * 2 + (cur == first ? 0 : 1);
        const int chunks = D / 8;  // eight elements of one query head a thread
        for (int x = threadIdx.x; x < g.nh * g.gt * chunks; x += 256) {
            const int hx = x / chunks, d = (x - hx * chunks) * 8, hh = hx / g.gt, h = hx - hh * g.gt;
            const int tile_x = item * g.nh + hh, kv = g.gtiles == 1 ? tile_x : tile_x / g.gtiles, head0 = (tile_x - kv * g.gtiles) * 16;
            if (head0 + h >= g.group) continue;
            float top = -__builtin_inff(), sum = 0.f;
            float r[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            for (int v = hh * g.nsub; v < (hh + 1) * g.nsub; v++) top = fmaxf(top, lds_stat[v * 16 + h].x);
            const float base = top == -__builtin_inff() ? 0.f : top;
            for (int v = hh * g.nsub; v < (hh + 1) * g.nsub; v++) {
                const float2 st = lds_stat[v * 16 + h];
                const float w = __builtin_amdgcn_exp2f(st.x - base);
                sum += w * st.y;
                const float *src = lds + (v * g.gt + h) * row_floats + d;
#pragma unroll
                for (int i = 0; i < 8; i++) r[i] += w * src[i];
            }
            if (whole) {
                const bool nothing = top == -__builtin_inff();
                uint16_t *out = (uint16_t *)g.a.out + t * g.a.out_strides[0] + ((int64_t)kv * g.group + head0 + h) * g.a.out_strides[1] + d;
                uint16_t y[8];
#pragma unroll
                for (int i = 0; i < 8; i++) y[i] = store16<BF>(nothing ? 0.f : r[i] / sum);
                if (o16) {
                    u32x4 v;
#pragma unroll
                    for (int i = 0; i < 4; i++) v[i] = (uint32_t)y[2 * i] | (uint32_t)y[2 * i + 1] << 16;
                    *reinterpret_cast<u32x4 *>(out) = v;
                } else {
#pragma unroll
                    for (int i = 0; i < 8; i++) out[i] = y[i];
                }
            } else {
                const int64_t piece = (int64_t)slot * g.nh + hh;
                float *dst = g.part + (piece * g.gt + h) * D + d;
#pragma unroll
                for (int i = 0; i < 8; i += 2) store_shared(dst + i, r[i], r[i + 1]);
                if (d == 0) store_shared(&g.stat[piece * 16 + h].x, top, sum);
            }
        }
        if (!whole) {
            const uint64_t u0 = cur - unit;
            const int from = (int)div64(u0, per), to = (int)div64(u0 + k.units - 1, per);  // the item's workgroups
            const int slot0 = from * 2 + (u0 == from * per ? 0 : 1);
            if (to - from <= kPieces) {
                // The last of the item's workgroups to arrive joins its
                // pieces.  No fence: the pieces are written through to memory
                // (store_shared), every wave waits for its own to be there,
                // the barrier collects the waves, then one lane counts the
                // workgroup in; the last one reads past its L2.  No workgroup
                // waits for another, and the count is left at zero.
                __shared__ int last_one;
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                __syncthreads();
                if (threadIdx.x == 0) {
                    const uint32_t there = __hip_atomic_fetch_add(g.arrived + from, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    last_one = there == (uint32_t)(to - from);
                    if (last_one) __hip_atomic_store(g.arrived + from, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
                __syncthreads();
                if (last_one) {
                    const int quads = D / 4;
                    for (int x = threadIdx.x; x < g.nh * g.gt * quads; x += 256) {
                        const int hx = x / quads, e4 = (x - hx * quads) * 4, hh = hx / g.gt, h = hx - hh * g.gt;
                        const int ht = item * g.nh + hh, kv = g.gtiles == 1 ? ht : ht / g.gtiles, head0 = (ht - kv * g.gtiles) * 16;
                        if (head0 + h >= g.group) continue;
                        float top = -__builtin_inff(), sum = 0.f, r[4] = {0.f, 0.f, 0.f, 0.f};
                        for (int i0 = from; i0 <= to; i0 += 4) {
                            float2 st[4], v[4][2];
#pragma unroll
                            for (int u = 0; u < 4; u++) {
                                const int i = i0 + u < to ? i0 + u : to;
                                const int64_t piece = (int64_t)(i == from ? slot0 : 2 * i) * g.nh + hh;
                                const float *src = g.part + (piece * g.gt + h) * D + e4;
                                st[u] = load_shared(&g.stat[piece * 16 + h].x);
                                v[u][0] = load_shared(src);
                                v[u][1] = load_shared(src + 2);
                            }
                            float most = top;
#pragma unroll
                            for (int u = 0; u < 4; u++) most = fmaxf(most, st[u].x);  // (the last one again where there are fewer)
                            const float base = most == -__builtin_inff() ? 0.f : most, keep = __builtin_amdgcn_exp2f(top - base);
                            sum *= keep;
#pragma unroll
                            for (int e = 0; e < 4; e++) r[e] *= keep;
#pragma unroll
                            for (int u = 0; u < 4; u++) {
                                if (i0 + u > to) continue;
                                const float w = __builtin_amdgcn_exp2f(st[u].x - base);
                                sum += w * st[u].y;
                                r[0] += w * v[u][0].x;
                                r[1] += w * v[u][0].y;
                                r[2] += w * v[u][1].x;
                                r[3] += w * v[u][1].y;
                            }
                            top = most;
                        }
                        uint16_t *out = (uint16_t *)g.a.out + t * g.a.out_strides[0] + ((int64_t)kv * g.group + head0 + h) * g.a.out_strides[1] + e4;
#pragma unroll
                        for (int e = 0; e < 4; e++) out[e] = store16<BF>(top == -__builtin_inff() ? 0.f : r[e] / sum);
                    }
                }
            }
        }
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

// Joins the pieces of an item that has many (a long request): a workgroup a
// query head, a thread four elements of every 256 / (head_dim / 4)-th piece,
// eight in flight.
template <bool BF>
__global__ __launch_bounds__(256) void join_kernel(AttendArgs g) {
    const int4 s = g.many[blockIdx.x];
    if (s.x < 0) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, D = g.c.head_dim, quads = D / 4, at_once = 256 / quads;
    const int from = s.z >> 1, n = s.w - from + 1, p0 = tid / quads, q = tid - p0 * quads;
    __shared__ f32x4 acc[256];
    __shared__ float weight[256], red[8];
    {
        const int hx = blockIdx.y, hh = hx / g.gt, h = hx - hh * g.gt, ht = s.y * g.nh + hh;
        const int kvh = ht / g.gtiles, gt0 = (ht - kvh * g.gtiles) * 16;
        if (gt0 + h >= g.group) return;
        auto piece = [&](int i) -> int64_t { return (i == 0 ? (int64_t)s.z : ((int64_t)from + i) * 2) * g.nh + hh; };
        float top = -__builtin_inff();
        for (int i = tid; i < n; i += 256) top = fmaxf(top, g.stat[piece(i) * 16 + h].x);
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
        if (lane == 0) red[wave] = top;
        __syncthreads();
        top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        const float base = top == -__builtin_inff() ? 0.f : top;
        f32x4 r = {0.f, 0.f, 0.f, 0.f};
        float sum = 0.f;
        for (int i0 = 0; i0 < n; i0 += 256) {  // 256 weights at a time
            if (i0 > 0) __syncthreads();
            if (i0 + tid < n) {
                const float2 st = g.stat[piece(i0 + tid) * 16 + h];
                const float w = __builtin_amdgcn_exp2f(st.x - base);
                weight[tid] = w;
                sum += w * st.y;
            }
            __syncthreads();
            const int m = n - i0 < 256 ? n - i0 : 256;
            if (p0 < at_once)
                for (int i = p0; i < m; i += 8 * at_once) {
                    f32x4 v[8];
#pragma unroll
                    for (int u = 0; u < 8; u++) {
                        const int x = i + u * at_once < m ? i + u * at_once : i;
                        v[u] = *reinterpret_cast<const f32x4 *>(g.part + (piece(i0 + x) * g.gt + h) * D + 4 * q);
                    }
#pragma unroll
                    for (int u = 0; u < 8; u++) {
                        const bool in = i + u * at_once < m;
                        const float w = in ? weight[i + u * at_once] : 0.f;
#pragma unroll
                        for (int e = 0; e < 4; e++) r[e] += in ? w * v[u][e] : 0.f;
                    }
                }
        }
        acc[tid] = r;
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d, 64);
        if (lane == 0) red[4 + wave] = sum;
        __syncthreads();
        if (tid < quads) {
            const float den = (red[4] + red[5]) + (red[6] + red[7]);
            for (int p = 1; p < at_once; p++)
#pragma unroll
                for (int e = 0; e < 4; e++) r[e] += acc[p * quads + tid][e];
            const int64_t head = (int64_t)kvh * g.group + gt0 + h;
            uint16_t *out = (uint16_t *)g.a.out + s.x * g.a.out_strides[0] + head * g.a.out_strides[1] + 4 * tid;
#pragma unroll
            for (int e = 0; e < 4; e++) out[e] = store16<BF>(top == -__builtin_inff() ? 0.f : r[e] / den);
        }
        __syncthreads();
    }
}

// The most units a token can have.
int64_t attend_units(const AttendArgs &g) {
    const int64_t held = g.a.table_width * g.c.page_size;
    const int64_t keys = g.a.window > 0 && (int64_t)g.a.window + kTile < held ? (int64_t)g.a.window + kTile : held;
    return keys / (kPair * kTile * g.nsub) + 1;
}

// The resident workgroups, and no more than there can be units.
int64_t attend_groups(const AttendArgs &g, int cus) {
    const int64_t groups = (int64_t)cus * (g.c.head_dim > 128 ? 1 : g.c.head_dim > 64 ? 2 : 3);
    const int64_t units = attend_units(g), items = g.a.tokens * (g.c.kv_heads * (int64_t)g.gtiles / g.nh);
    return items > groups / units ? groups : items * units;
}

// What both the workspace and the launch go by.
AttendArgs attend_args(const orth_hip_cache_t &c, const orth_hip_attend_t &a, int cus, int64_t *groups) {
    AttendArgs g;
    g.c = c;
    g.a = a;
    g.page = fast_div((uint32_t)c.page_size);
    g.scale2 = a.scale * 1.4426950408889634f;
    g.group = a.q_heads / c.kv_heads;
    g.gtiles = (g.group + 15) / 16;
    g.gt = g.group < 16 ? g.group : 16;
    // Four or two head tiles a workgroup where there are items enough: its
    // waves then read neighbouring heads of the same keys and need no join
    // (128 requests: 569 us in the kernel, 605 with one tile).  Few items are
    // cut along the keys instead, so that their pieces are few (40 requests of
    // four heads at four tiles a workgroup: 21.9 us, at two 15.9).
    const int64_t tiles = (int64_t)c.kv_heads * g.gtiles;
    g.nh = 1;
    const bool few_keys = a.table_width <= ((int64_t)1 << 28) / c.page_size;  // (block_units)
    while (few_keys && g.nh < kWaves && tiles % (2 * g.nh) == 0 && a.tokens * (tiles / (2 * g.nh)) >= cus / 4) g.nh *= 2;
    g.nsub = kWaves / g.nh;
    *groups = attend_groups(g, cus);
    return g;
}

template <int KS, bool BF>
hipError_t attend_launch(const AttendArgs &g, int64_t groups, size_t lds, hipStream_t stream) {
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
hipError_t attend_by_width(const AttendArgs &g, int64_t groups, hipStream_t stream) {
    const int D = g.c.head_dim, el = D <= 64 ? 4 : D <= 128 ? 8 : 16;
    const size_t lds = (size_t)kWaves * g.gt * (16 * el + 4) * 4 + kWaves * 16 * sizeof(float2);
    hipError_t e = D <= 64 ? attend_launch<2, BF>(g, groups, lds, stream)
                 : D <= 96 ? attend_launch<3, BF>(g, groups, lds, stream)
                 : D <= 128 ? attend_launch<4, BF>(g, groups, lds, stream)
                            : attend_launch<8, BF>(g, groups, lds, stream);
    if (e != hipSuccess) return e;
    // No item has many pieces where none has many units, and of one token's
    // items, which are all of one length, none where they are many.  Requests
    // of several lengths may have: one long among short ones.  (40 requests
    // with windows: 15.3 us without the second launch, 16.8 with it, 17.5
    // where it joined all.  A workgroup alone would take tens of microseconds
    // to join the hundreds of pieces of a long request.)
    const int64_t items = g.a.tokens * (g.c.kv_heads * (int64_t)g.gtiles / g.nh);
    if (attend_units(g) <= kPieces + 1 || (g.a.tokens == 1 && items * kPieces >= groups)) return hipSuccess;
    join_kernel<BF><<<dim3((unsigned)((groups + kPieces - 1) / kPieces), (unsigned)(g.nh * g.gt)), 256, 0, stream>>>(g);
    return hipGetLastError();
}

}  // namespace

int64_t attention_workspace_bytes(const orth_hip_cache_t &c, const orth_hip_attend_t &a, int cus, int64_t *groups) {
    int64_t n = 0;
    const AttendArgs g = attend_args(c, a, cus, &n);
    *groups = attend_units(g) > 1 ? n : 0;  // (items of one unit are not split)
    return n * (2 * g.nh * (g.gt * (int64_t)c.head_dim * 4 + 16 * (int64_t)sizeof(float2))) +
           (n + kPieces - 1) / kPieces * (int64_t)sizeof(int4);
}

hipError_t launch_paged_attention(const orth_hip_cache_t &c, const orth_hip_attend_t &a, int cus, void *work, uint32_t *counters,
                                  hipStream_t stream) {
    int64_t groups = 0;
    AttendArgs g = attend_args(c, a, cus, &groups);
    g.many = static_cast<int4 *>(work);
    g.stat = reinterpret_cast<float2 *>(g.many + (groups + kPieces - 1) / kPieces);
    g.part = reinterpret_cast<float *>(g.stat + groups * 2 * g.nh * 16);
    g.arrived = counters;
    return c.dtype == ORTH_DT_BF16 ? attend_by_width<true>(g, groups, stream) : attend_by_width<false>(g, groups, stream);
}

}  // namespace orth
