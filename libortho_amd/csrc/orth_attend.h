// What the attention kernels over a paged cache share (orth_attn.hip over 16
// bits, orth_attn4.hip over 4): the even cut of the tokens' keys over the
// resident workgroups, and the joining of the pieces that it leaves.
//
// The work is cut by the keys the tokens really see, which only the device
// knows: every wave sums up the tokens' units (two tiles for each wave that
// shares a head tile: 64, 128 or 256 keys) and finds its workgroup's share (of
// 128 tokens in one load and one scan).  A share that ends inside a (token,
// key head) leaves a piece (m, l, o); the workgroup that writes an item's last
// piece joins them, or a second launch where an item has many.  Whole items
// are written at once.
//
// A kernel's arguments G derive from AttendArgs and say how an output is
// rounded (G::round) and whether up to `block` neighbouring tokens of one
// request are taken together, as further columns of their head tiles
// (G::blocks, then g.block, a power of two: tokens block * i .. of one row).
#pragma once

#include "orth_serve.h"

namespace orth {

constexpr int kWaves = 4;
constexpr int kTile = 32;                // keys a wave takes at a time
constexpr int kPair = 2;                 // tiles a wave takes in a unit, the least share of a workgroup
constexpr int kPieces = 16;              // pieces of an item (and one for its ends) that a workgroup joins
constexpr float kLeast = -3.0e38f;       // the maximum of a token that has seen keys, at the least

// Loads run up to two steps of kWaves tiles ahead of the last key: their key
// numbers stay within an int.
static_assert(kMostKeys + (2 * kWaves + 1) * kTile <= INT32_MAX, "a table's keys");

template <class Cache>
struct AttendArgs {
    Cache c;
    orth_hip_attend_t a;
    FastDiv page;
    float scale2;        // scale * log2(e)
    int group, gtiles;   // query heads of a key head, and their tiles of 16
    int gt;              // columns of a tile: min(group, 16), or those of a block of tokens
    FastDiv of_chunks, of_gt;  // by head_dim / 8, by gt
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

// Numbers that all lanes share, known as such: in scalar registers, also where
// a division made them by way of vector ones.
__device__ __forceinline__ int64_t uniform64(int64_t v) {
    return (int64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)v) | (int64_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32;
}
__device__ __forceinline__ Keys uniform(const Keys &k) {
    return Keys{__builtin_amdgcn_readfirstlane(k.begin), __builtin_amdgcn_readfirstlane(k.end),
                __builtin_amdgcn_readfirstlane(k.tile0), __builtin_amdgcn_readfirstlane(k.tiles),
                (uint32_t)__builtin_amdgcn_readfirstlane((int)k.units)};
}

// a / b.  (A 64-bit division takes a quarter of a microsecond, and a short
// call is a chain of such latencies: below 2^22 a product with the reciprocal
// is off by one at the most.)
__device__ __forceinline__ uint64_t div64(uint64_t a, uint64_t b) {
    if ((a | b) >> 32) return a / b;
    const uint32_t n = (uint32_t)a, d = (uint32_t)b;
    if (n >> 22) return n / d;
    uint32_t q = (uint32_t)((float)n * __builtin_amdgcn_rcpf((float)d));
    const int32_t rest = (int32_t)(n - q * d);
    if (rest < 0) q--;
    else if ((uint32_t)rest >= d) q++;
    return q;
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

// Token t's request, and the keys it sees of it.
template <class G>
__device__ __forceinline__ int64_t range_of(const G &g, int64_t t, int64_t *begin, int64_t *end) {
    const int64_t row = g.a.rows ? (int64_t)g.a.rows[t] : t;
    *end = (int64_t)g.a.positions[t] + 1;
    *begin = g.a.window > 0 && *end > g.a.window ? *end - g.a.window : 0;
    const int64_t held = g.a.table_width * g.c.page_size;
    *end = *end < held ? *end : held;
    if (row < 0 || row >= g.a.table_rows || *end <= *begin) *begin = *end = 0;
    return row;
}

template <class G>
__device__ __forceinline__ Keys tiles_of(const G &g, int64_t begin, int64_t end) {
    Keys k;
    k.begin = (int)begin;
    k.end = (int)end;
    k.tile0 = k.begin / kTile;
    k.tiles = (int)(((int64_t)k.end + kTile - 1) / kTile) - k.tile0;
    const int unit = kPair * g.nsub;
    k.units = k.tiles > unit ? (uint32_t)(k.tiles + unit - 1) / unit : 1;  // (one that sees nothing is written too)
    return k;
}

template <class G>
__device__ __forceinline__ Keys keys_of(const G &g, int64_t t) {
    int64_t begin, end;
    range_of(g, t, &begin, &end);
    return tiles_of(g, begin, end);
}

// The tokens of a block, reduced over the lanes that hold them: whether they
// are of one request, and the keys that any of them sees.
struct Block {
    int64_t low, high;    // least and greatest row
    int64_t begin, end;
    __device__ __forceinline__ void add(const Block &o) {
        low = low < o.low ? low : o.low;
        high = high > o.high ? high : o.high;
        begin = begin < o.begin ? begin : o.begin;
        end = end > o.end ? end : o.end;
    }
    __device__ __forceinline__ void across(int from, int to) {
        for (int d = from; d < to; d *= 2)
            add(Block{__shfl_xor(low, d, 64), __shfl_xor(high, d, 64), __shfl_xor(begin, d, 64), __shfl_xor(end, d, 64)});
    }
    __device__ __forceinline__ bool one() const { return low == high; }
};
template <class G>
__device__ __forceinline__ Block block_of(const G &g, int64_t t) {
    if (t >= g.a.tokens) return Block{INT64_MAX, INT64_MIN, INT64_MAX, 0};
    Block b;
    b.low = b.high = range_of(g, t, &b.begin, &b.end);
    if (b.end == 0) b.begin = INT64_MAX;
    return b;
}
template <class G>
__device__ __forceinline__ Keys tiles_of(const G &g, const Block &b) {
    return tiles_of(g, b.end == 0 ? 0 : b.begin, b.end);
}

// The keys of the item that starts with token t, and its tokens.
template <class G>
__device__ __forceinline__ Keys keys_at(const G &g, int64_t t, int lane, int *tokens) {
    *tokens = 1;
    if (g.block > 1 && (t & (g.block - 1)) == 0) {
        Block b = block_of(g, t + (lane & (g.block - 1)));
        b.across(1, g.block);
        if (__all(b.one())) {
            *tokens = (int)(g.a.tokens - t < g.block ? g.a.tokens - t : g.block);
            return uniform(tiles_of(g, b));
        }
    }
    return uniform(keys_of(g, t));
}

// Inclusive sums of the units of tokens t0 + 2 lane, + 1, whose keys are in k[2].  (32 bits
// hold them: a token has at most 2^23 units of 256 keys, or 2^22 of 64 where
// the launch has seen that its table holds no more than 2^28 keys, and a scan
// takes 128 tokens.)  A block's units are its first token's.
constexpr int kScan = 128;
template <class G>
__device__ __forceinline__ uint32_t block_units(const G &g, int64_t t0, int lane, Keys k[2]) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int64_t t = t0 + 2 * lane + i;
        k[i] = Keys{0, 0, 0, 0, 0};
        if (t < g.a.tokens) k[i] = keys_of(g, t);
    }
    if constexpr (G::blocks) {
        if (g.block > 1) {
            Block b = block_of(g, t0 + 2 * lane);
            b.add(block_of(g, t0 + 2 * lane + 1));
            b.across(1, g.block / 2);
            if (b.one()) {
                if ((2 * lane & (g.block - 1)) == 0) k[0] = tiles_of(g, b);
                else k[0].units = 0;
                k[1].units = 0;
            }
        }
    }
    return wave_scan(k[0].units + k[1].units);
}

// A workgroup's share of the work: units cur .. stop - 1, which begin inside
// token t's item `item` at its unit `unit`.
struct Share {
    uint64_t per, cur, stop;
    int64_t t;
    Keys k;
    int item;
    uint32_t unit;
};
__device__ __forceinline__ Share uniform(const Share &s) {
    return Share{(uint64_t)uniform64(s.per), (uint64_t)uniform64(s.cur), (uint64_t)uniform64(s.stop), uniform64(s.t), uniform(s.k),
                 __builtin_amdgcn_readfirstlane(s.item), (uint32_t)__builtin_amdgcn_readfirstlane((int)s.unit)};
}
template <class G>
__device__ __forceinline__ bool share_of(const G &g, int lane, int items, Share *s) {
    Keys mine[2];
    uint32_t incl = 0;
    uint64_t run = 0;
    for (int64_t t0 = 0; t0 < g.a.tokens; t0 += kScan) {
        incl = block_units(g, t0, lane, mine);
        run += (uint32_t)__builtin_amdgcn_readlane((int)incl, 63);
    }
    const uint64_t total = run * items;
    s->per = div64(total + gridDim.x - 1, gridDim.x);
    s->cur = blockIdx.x * s->per;
    s->stop = s->cur + s->per < total ? s->cur + s->per : total;
    const bool marks = blockIdx.x % kPieces == 0 && threadIdx.x == 0;
    if (s->cur >= total) {
        if (marks) g.many[blockIdx.x / kPieces] = int4{-1, 0, 0, 0};
        return false;
    }
    const uint64_t want = div64(s->cur, items);  // the unit, were a token one item
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
            s->t = t0 + 2 * l + (second ? 1 : 0);
            const Keys &x = second ? mine[1] : mine[0];
            s->k.begin = __builtin_amdgcn_readlane(x.begin, l);
            s->k.end = __builtin_amdgcn_readlane(x.end, l);
            s->k.tile0 = __builtin_amdgcn_readlane(x.tile0, l);
            s->k.tiles = __builtin_amdgcn_readlane(x.tiles, l);
            s->k.units = (uint32_t)__builtin_amdgcn_readlane((int)x.units, l);
            before += second ? end - u1 : end - u1 - s->k.units;
            break;
        }
        before += all;
    }
    const uint64_t inside = s->cur - before * items;
    s->item = (int)div64(inside, s->k.units);
    s->unit = (uint32_t)(inside - (uint64_t)s->item * s->k.units);

    if (marks) {
        // an item of more than kPieces + 1 pieces has a workgroup of these
        // behind its first one, and only one within kPieces of it, at whose
        // start no other item lies: it names the item to the second launch
        const uint64_t u0 = s->cur - s->unit;
        const int from = (int)div64(u0, s->per), to = (int)div64(u0 + s->k.units - 1, s->per);
        const bool big = to - from > kPieces && from < (int)blockIdx.x && (int)blockIdx.x - from <= kPieces;
        g.many[blockIdx.x / kPieces] = big ? int4{(int)s->t, s->item, from * 2 + (u0 == from * s->per ? 0 : 1), to} : int4{-1, 0, 0, 0};
    }
    return true;
}

// Where column h of head tile `tile` of an item of `tokens` tokens from t goes
// (NULL: there is no such column).
template <class G>
__device__ __forceinline__ uint16_t *out_of(const G &g, int64_t t, int tokens, int tile, int h) {
    const int kv = g.gtiles == 1 ? tile : tile / g.gtiles, head0 = (tile - kv * g.gtiles) * 16;
    if constexpr (G::blocks) {
        if (tokens > 1) {
            const int j = h / g.group;
            return j >= tokens ? nullptr
                               : (uint16_t *)g.a.out + (t + j) * g.a.out_strides[0] + ((int64_t)kv * g.group + (h - j * g.group)) * g.a.out_strides[1];
        }
    }
    return head0 + h >= g.group ? nullptr
                                : (uint16_t *)g.a.out + t * g.a.out_strides[0] + ((int64_t)kv * g.group + head0 + h) * g.a.out_strides[1];
}

// A column that has seen no key (one of a block may see none where others do).
template <class G>
__device__ __forceinline__ bool unseen(float top, float sum) {
    if constexpr (G::blocks) return sum == 0.f;
    else return top == -__builtin_inff();
}

// Where a piece's row of D elements holds the pair from element e: the first
// pairs of every eight elements, then the second ones, so that the threads of
// a row, eight elements each, write whole lines through.
__device__ __forceinline__ int pair_at(int D, int e) { return (e & 7) / 2 * (D / 4) + e / 8 * 2; }

// Joins the waves' sums of an item, which lie in LDS (o: for each wave, every
// wave_floats, gt rows of row_floats, and (m, l) [waves][16]): units unit .. unit + n - 1 of it, which
// are written if they are all, else left as a piece, joined by the workgroup
// that writes the last one.
template <class G>
__device__ __forceinline__ void finish_item(const G &g, int tid, const float *lds, const float2 *lds_stat, int row_floats, int wave_floats, bool o16,
                                            uint64_t first, uint64_t cur, uint64_t per, int64_t t, int tokens, const Keys &k,
                                            int item, uint32_t unit, uint32_t n) {
    const int D = g.c.head_dim;
    const bool whole = n == k.units;
    const int slot = (int)blockIdx.x * 2 + (cur == first ? 0 : 1);
    const int chunks = D / 8, gt = g.gt;  // eight elements of one query head a thread
    for (int x = tid; x < g.nh * gt * chunks; x += 256) {
        const int hx = (int)quotient(x, g.of_chunks), d = (x - hx * chunks) * 8, hh = (int)quotient(hx, g.of_gt), h = hx - hh * gt;
        uint16_t *out = out_of(g, t, tokens, item * g.nh + hh, h);
        if (!out) continue;
        float top = -__builtin_inff(), sum = 0.f;
        float r[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        for (int v = hh * g.nsub; v < (hh + 1) * g.nsub; v++) top = fmaxf(top, lds_stat[v * 16 + h].x);
        const float base = top == -__builtin_inff() ? 0.f : top;
        for (int v = hh * g.nsub; v < (hh + 1) * g.nsub; v++) {
            const float2 st = lds_stat[v * 16 + h];
            const float w = __builtin_amdgcn_exp2f(st.x - base);
            sum += w * st.y;
            const float *src = lds + v * wave_floats + h * row_floats + d;
#pragma unroll
            for (int i = 0; i < 8; i++) r[i] += w * src[i];
        }
        if (whole) {
            const bool nothing = unseen<G>(top, sum);
            out += d;
            uint16_t y[8];
#pragma unroll
            for (int i = 0; i < 8; i++) y[i] = g.round(nothing ? 0.f : r[i] / sum);
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
            float *dst = g.part + (piece * gt + h) * D;
#pragma unroll
            for (int i = 0; i < 8; i += 2) store_shared(dst + pair_at(D, d + i), r[i], r[i + 1]);
            if (d == 0) store_shared(&g.stat[piece * 16 + h].x, top, sum);
        }
    }
    if (whole) return;
    const uint64_t u0 = cur - unit;
    const int from = (int)div64(u0, per), to = (int)div64(u0 + k.units - 1, per);  // the item's workgroups
    const int slot0 = from * 2 + (u0 == from * per ? 0 : 1);
    if (to - from > kPieces) return;
    // The last of the item's workgroups to arrive joins its
    // pieces.  No fence: the pieces are written through to memory
    // (store_shared), every wave waits for its own to be there,
    // the barrier collects the waves, then one lane counts the
    // workgroup in; the last one reads past its L2.  No workgroup
    // waits for another, and the count is left at zero.
    __shared__ int last_one;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0) {
        const uint32_t there = __hip_atomic_fetch_add(g.arrived + from, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last_one = there == (uint32_t)(to - from);
        if (last_one) __hip_atomic_store(g.arrived + from, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!last_one) return;
    const int quads = D / 4;
    for (int x = tid; x < g.nh * gt * quads; x += 256) {
        const int hx = (int)quotient(x >> 1, g.of_chunks), e4 = (x - hx * quads) * 4, hh = (int)quotient(hx, g.of_gt), h = hx - hh * gt;
        uint16_t *out = out_of(g, t, tokens, item * g.nh + hh, h);
        if (!out) continue;
        float top = -__builtin_inff(), sum = 0.f, r[4] = {0.f, 0.f, 0.f, 0.f};
        for (int i0 = from; i0 <= to; i0 += 4) {
            float2 st[4], v[4][2];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int i = i0 + u < to ? i0 + u : to;
                const int64_t piece = (int64_t)(i == from ? slot0 : 2 * i) * g.nh + hh;
                const float *src = g.part + (piece * gt + h) * D;
                st[u] = load_shared(&g.stat[piece * 16 + h].x);
                v[u][0] = load_shared(src + pair_at(D, e4));
                v[u][1] = load_shared(src + pair_at(D, e4 + 2));
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
        out += e4;
#pragma unroll
        for (int e = 0; e < 4; e++) out[e] = g.round(unseen<G>(top, sum) ? 0.f : r[e] / sum);
    }
}

// Joins the pieces of an item that has many (a long request): a workgroup a
// column, a thread four elements of every 256 / (head_dim / 4)-th piece,
// eight in flight.
template <class G>
__global__ __launch_bounds__(256) void join_kernel(G g) {
    const int4 s = g.many[blockIdx.x];
    if (s.x < 0) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, D = g.c.head_dim, quads = D / 4, at_once = 256 / quads;
    const int from = s.z >> 1, n = s.w - from + 1, p0 = tid / quads, q = tid - p0 * quads;
    __shared__ f32x4 acc[256];
    __shared__ float weight[256], red[8];
    const int hx = blockIdx.y, hh = hx / g.gt, h = hx - hh * g.gt;
    int tokens = 1;
    if constexpr (G::blocks) keys_at(g, s.x, lane, &tokens);
    uint16_t *out = out_of(g, s.x, tokens, s.y * g.nh + hh, h);
    if (!out) return;
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
                    const float *src = g.part + (piece(i0 + x) * g.gt + h) * D;
                    const float2 a = *reinterpret_cast<const float2 *>(src + pair_at(D, 4 * q));
                    const float2 b = *reinterpret_cast<const float2 *>(src + pair_at(D, 4 * q + 2));
                    v[u] = f32x4{a.x, a.y, b.x, b.y};
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
        out += 4 * tid;
#pragma unroll
        for (int e = 0; e < 4; e++) out[e] = g.round(unseen<G>(top, den) ? 0.f : r[e] / den);
    }
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

// ------------------------------------------------------------------- host side

// The most units a token (or a block of `block` ones) can have.
template <class G>
int64_t attend_units(const G &g, int64_t block = 1) {
    const int64_t held = g.a.table_width * g.c.page_size;
    const int64_t span = block > 1 ? held : (int64_t)g.a.window + kTile;  // (a block's tokens may lie apart)
    const int64_t keys = g.a.window > 0 && span < held ? span : held;
    return keys / (kPair * kTile * g.nsub) + 1;
}

// Head tiles a workgroup.
// Four or two where there are items enough: its
// waves then read neighbouring heads of the same keys and need no join
// (128 requests: 569 us in the kernel, 605 with one tile).  Few items are
// cut along the keys instead, so that their pieces are few (40 requests of
// four heads at four tiles a workgroup: 21.9 us, at two 15.9).
// `least`: the items that are enough.
template <class G>
void attend_tiles(G &g, int64_t least, int64_t items_of_a_head) {
    const int64_t tiles = (int64_t)g.c.kv_heads * g.gtiles;
    g.nh = 1;
    const bool few_keys = g.a.table_width <= ((int64_t)1 << 28) / g.c.page_size;  // (block_units)
    while (few_keys && g.nh < kWaves && tiles % (2 * g.nh) == 0 && items_of_a_head * (tiles / (2 * g.nh)) >= least) g.nh *= 2;
    g.nsub = kWaves / g.nh;
    g.of_chunks = fast_div((uint32_t)g.c.head_dim / 8);
    g.of_gt = fast_div((uint32_t)g.gt);
}

// `resident` workgroups, and no more than there can be units.
template <class G>
int64_t attend_groups(const G &g, int64_t resident, int64_t block = 1) {
    const int64_t units = attend_units(g, block), items = g.a.tokens * (g.c.kv_heads * (int64_t)g.gtiles / g.nh);
    return items > resident / units ? resident : items * units;
}

// Whether the second launch is needed.
// No item has many pieces where none has many units, and of one token's
// items, which are all of one length, none where they are many.  Requests
// of several lengths may have: one long among short ones.  (40 requests
// with windows: 15.3 us without the second launch, 16.8 with it, 17.5
// where it joined all.  A workgroup alone would take tens of microseconds
// to join the hundreds of pieces of a long request.)
template <class G>
bool attend_joins(const G &g, int64_t groups, int64_t block = 1) {
    const int64_t items = g.a.tokens * (g.c.kv_heads * (int64_t)g.gtiles / g.nh);
    return !(attend_units(g, block) <= kPieces + 1 || (g.a.tokens == 1 && items * kPieces >= groups));
}
template <class G>
hipError_t launch_join(const G &g, int64_t groups, hipStream_t stream) {
    join_kernel<G><<<dim3((unsigned)((groups + kPieces - 1) / kPieces), (unsigned)(g.nh * g.gt)), 256, 0, stream>>>(g);
    return hipGetLastError();
}

// A call's workspace: the items with many pieces, the pieces' (m, l), the pieces.
template <class G>
int64_t attend_bytes(const G &g, int64_t groups) {
    return groups * (2 * g.nh * (g.gt * (int64_t)g.c.head_dim * 4 + 16 * (int64_t)sizeof(float2))) +
           (groups + kPieces - 1) / kPieces * (int64_t)sizeof(int4);
}
template <class G>
void attend_workspace(G &g, int64_t groups, void *work, uint32_t *counters) {
    g.many = static_cast<int4 *>(work);
    g.stat = reinterpret_cast<float2 *>(g.many + (groups + kPieces - 1) / kPieces);
    g.part = reinterpret_cast<float *>(g.stat + groups * 2 * g.nh * 16);
    g.arrived = counters;
}

}  // namespace orth
