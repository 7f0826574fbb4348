// Low-rank adapters of many requests beside a shared projection:
// out[m] = y[m] + scale_i (x[m] A_i^T) B_i^T with i = adapters[m].
//
// Two launches with the low-rank values between them in FP32, one partial
// per slice of in_features, added in order by the second:
//
//   down  low[m, j] = sum_k x[m, k] A_i[j, k]
//   up    out[m, n] = y[m, n] + sum_j (scale_i low[m, j]) B_i[n, j]
//
// Both go through v_mfma_f32_16x16x32 with 16 tokens as the columns
// (consecutive ones, or neighbours in their adapters' order: Order): x, A and B enter by 16-byte loads as they lie; products are exact,
// sums FP32.  For every adapter among the 16 tokens (found by ballots) the
// product is formed for all columns and kept in those of its own tokens: a
// run of one prompt's tokens is one product, a decode batch of 16 requests
// reads each of their adapters once, and what one adapter holds cannot reach
// another's tokens.  The low-rank values enter the second product as FP32
// values do: as 16-bit parts (three in BF16, two in FP16), whose products with
// B are exact and add up in FP32; FP16 ones are scaled by a power of two per
// token, so that none overflows or loses its low bits.
//
// Bound by reading the adapters (few tokens: workgroups of 16 tokens, a slot
// for each adapter among them, then waves that split the adapters) or x, y
// and out (many: 64 tokens a workgroup share each adapter's loads).
//
// Measured (one MI355X, a call among others): one token, 4096 -> 4096, rank
// 16, FP16: 8.9 us, two chains of latencies (number, weights, join; number,
// partials, store); 48 tokens of 24 adapters, 4096 -> 11008, rank 32, BF16:
// 16.2 us (23.7 MB, 1.5 TB/s; down 6, up 10.5); 2,048 tokens in five runs,
// 11008 -> 4096, rank 64, FP16: 37.5 us (86 MB, 2.3 TB/s; down 19, up 19: the
// partials, which each of the second launch's output blocks adds up again, and
// the launches' starts and ends, with one round of workgroups each).  HBM reads
// by counter: 6.3 MB (A is 6.3) and 17.9 (B and y 17.9) at 48 tokens, 62.6 (x
// and A 52) and 27.4 (B and y 19.4, partials 4) at 2,048.  A wave per low-rank value and a thread per output took
// 12, 57 and 2,500 us.
#include <type_traits>

#include "orth_serve.h"

namespace orth {

namespace {

constexpr int kTokens = 64;    // tokens of a tile, where they are many
constexpr int kFew = 512;      // up to here, tiles of 16: decode batches, whose adapters differ by token
constexpr int kUp = 64;        // outputs a wave takes at a time
constexpr int kShared = 4;     // adapters of a 64-token tile up to which each has a pass of its own
constexpr int kUpWaves = 8;    // waves of an up workgroup of 64 tokens
constexpr int kDown = 8;       // waves of a down workgroup: steps in flight without more partials to add

struct AdapterArgs {
    orth_hip_adapter_t a;
    float *low;        // [slices][tokens][rank]
    int tiles;         // of 16 or 64 tokens
    int slices, steps; // slices of in_features, and steps of 32 in each
    int blocks;        // up: blocks of out_features
    int slots;         // down: workgroups that share the adapters of a tile
    int chunk;         // tiles of an XCD (0: too few to keep together)
    int order_by;      // of 16-token tiles: an Order
    int few;           // 16-token tiles
    int *order;        // [tokens], by the down launch for the up launch (ORDER_GROUP)
};

// Workgroup -> (tile, part of it).  Neighbours in blockIdx go to different
// XCDs, eight in turn, so XCD x takes the x-th eighth of the tiles: tiles of
// one prompt share its adapter in that XCD's L2, and a tile's partials are
// read from the L2 they were written to.
__device__ __forceinline__ void place_of(const AdapterArgs &g, int b, int parts, int *tile, int *part) {
    if (g.chunk > 0) {
        const int x = b & 7, q = b >> 3, at = q / parts;
        *tile = at < g.chunk ? x * g.chunk + at : g.tiles;
        *part = q - at * parts;
    } else {
        *tile = b / parts;
        *part = b - *tile * parts;
    }
}

// The adapter of token m (-1: none).
__device__ __forceinline__ int adapter_of(const AdapterArgs &g, int64_t m) {
    if (m >= g.a.tokens) return -1;
    const int i = g.a.adapters[m];
    return i >= 0 && i < g.a.count ? i : -1;
}

// The tokens of 16-token tiles.  Where the stack has fewer adapters than
// there are tokens, the tiles take the tokens in the order of their adapters
// (those without one last, a stable order), so that the tokens of one adapter
// fall into few tiles and it is read so often: up to 64 tokens each wave
// orders them, more the down launch's workgroups, which leave the order for
// the up launch.
enum Order { ORDER_NONE = 0, ORDER_WAVE = 1, ORDER_GROUP = 2 };
constexpr int kOrdered = 512;  // tokens up to which they are ordered

// The token of column lane & 15 of a tile, and its adapter (-1: none, or no
// token); `order`: the tokens in their order (ORDER_GROUP).  False: the column
// has no token (`m` then is some token's).
__device__ __forceinline__ bool few_token(const AdapterArgs &g, int tile, const int *order, int *m, int *mine) {
    const int lane = threadIdx.x & 63, tokens = (int)g.a.tokens, at = tile * 16 + (lane & 15);
    const bool present = at < tokens;
    if (g.order_by != ORDER_WAVE) {
        *m = present ? (g.order_by == ORDER_GROUP ? order[at] : at) : tokens - 1;
        *mine = present ? adapter_of(g, *m) : -1;
        return present;
    }
    // adapter, then token (adapter_args has seen that the numbers fit)
    const int id = adapter_of(g, lane);
    const uint32_t key = lane < tokens ? (uint32_t)(id >= 0 ? id : 1 << 25) * 64 + lane : 0xffffffc0u + lane;
    int rank = 0;
#pragma unroll
    for (int j = 0; j < 64; j++) rank += (uint32_t)__builtin_amdgcn_readlane((int)key, j) < key;
    const int by = __builtin_amdgcn_ds_permute(rank * 4, lane);  // lane p: the p-th token
    const int t = __shfl(by, at & 63, 64), of = __shfl(id, t, 64);
    *m = present ? t : tokens - 1;
    *mine = present ? of : -1;
    return present;
}

// Orders up to kOrdered tokens: `order` in LDS, room for 2 * kOrdered words.
__device__ __forceinline__ void order_tokens(const AdapterArgs &g, int *order) {
    const int n = (int)g.a.tokens, tid = threadIdx.x, threads = blockDim.x;
    uint32_t *keys = reinterpret_cast<uint32_t *>(order + kOrdered);
    for (int t = tid; t < kOrdered; t += threads) {
        const int id = t < n ? adapter_of(g, t) : -1;
        keys[t] = t < n ? (uint32_t)(id >= 0 ? id : 1 << 22) * kOrdered + t : 0xffffffffu;
        order[t] = 0;
    }
    __syncthreads();
    // `parts` threads a token, each counting the smaller keys of its part
    const int parts = threads / ((n + 63) / 64 * 64), wide = threads / parts, part = tid / wide, t = tid - part * wide;
    const int span = ((n + parts - 1) / parts + 3) / 4 * 4;
    const uint32_t key = t < n ? keys[t] : 0u;
    int rank = 0;
    for (int j = part * span; j < (part + 1) * span && j < kOrdered; j += 4) {
        const u32x4 k = *reinterpret_cast<const u32x4 *>(keys + j);
#pragma unroll
        for (int e = 0; e < 4; e++) rank += k[e] < key;
    }
    if (t < n) atomicAdd(order + t, rank);
    __syncthreads();
    const int place = tid < n ? order[tid] : 0;
    __syncthreads();
    if (tid < n) order[place] = tid;
    __syncthreads();
}

// Eight 16-bit elements from p; those from `left` on are zero, and nothing
// past them is read (`safe` stands in).  W: elements of a load that pointers
// and row lengths allow.  The loads are not behind branches: a branch would
// make the waves wait for every load in flight.
template <int W>
__device__ __forceinline__ u32x4 load8(const uint16_t *p, int64_t left, const uint16_t *safe) {
    u32x4 v = {0u, 0u, 0u, 0u};
    if constexpr (W == 8) {
        v = *reinterpret_cast<const u32x4 *>(left > 0 ? p : safe);
        if (!(left > 0)) v = u32x4{0u, 0u, 0u, 0u};
    } else if constexpr (W == 4) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const uint2 a = *reinterpret_cast<const uint2 *>(left > 4 * h ? p + 4 * h : safe);
            v[2 * h] = left > 4 * h ? a.x : 0u;
            v[2 * h + 1] = left > 4 * h ? a.y : 0u;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (e < left) v[e >> 1] |= (uint32_t)p[e] << (16 * (e & 1));
    }
    return v;
}

// The same with all eight there.
template <int W>
__device__ __forceinline__ u32x4 load8(const uint16_t *p) {
    if constexpr (W == 8) return *reinterpret_cast<const u32x4 *>(p);
    u32x4 v = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int e = 0; e < 8; e++) v[e >> 1] |= (uint32_t)p[e] << (16 * (e & 1));
    return v;
}

template <bool BF>
__device__ __forceinline__ f32x4 mfma(const u32x4 &a, const u32x4 &b, const f32x4 &c) {
    if constexpr (BF)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// ------------------------------------------------------------------------ down

// The workgroup's sum of a product of each wave, 16 RB ranks by 16 tokens,
// joined in LDS ([waves][16 RB][17]); the columns in `own` (column lane & 15 is
// token m) are written as this slice's partial.
template <int RB>
__device__ __forceinline__ void down_join(const AdapterArgs &g, const f32x4 (&acc)[RB], int m, uint32_t own, int rank0,
                                          int slice, float *lds) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, lg = lane >> 4;
    __syncthreads();  // the last use of lds is over
#pragma unroll
    for (int r = 0; r < RB; r++)
#pragma unroll
        for (int i = 0; i < 4; i++) lds[(wave * 16 * RB + 16 * r + 4 * lg + i) * 17 + col] = acc[r][i];
    __syncthreads();
    for (int x = threadIdx.x; x < 256 * RB; x += 64 * kDown) {
        const int j = x % (16 * RB), t = x / (16 * RB), token = __shfl(m, t, 64);
        if (!(own >> t & 1) || rank0 + j >= g.a.rank) continue;
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < kDown; w++) sum += lds[(w * 16 * RB + j) * 17 + t];
        g.low[((int64_t)slice * g.a.tokens + token) * g.a.rank + rank0 + j] = sum;
    }
}

// The whole steps of this wave in a slice: [s, end); true where the step that
// in_features ends inside follows them.
__device__ __forceinline__ bool down_steps(const AdapterArgs &g, int slice, int *s, int *end) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), share = (g.steps + kDown - 1) / kDown, last = (slice + 1) * g.steps;
    const int whole = (int)(g.a.in_features / 32);
    *s = slice * g.steps + wave * share;
    int e = *s + share;
    e = e < last ? e : last;
    *end = e < whole ? e : whole;
    return g.a.in_features % 32 != 0 && *s <= whole && whole < e;
}

// A slice for one of a 16-token tile's adapters: a workgroup reads its part
// of one A, all of a wave's loads in flight.
template <int RB, bool BF, int W>
__device__ __forceinline__ void down_one(const AdapterArgs &g, int m, int id, uint32_t own, int rank0, int slice, float *lds) {
    constexpr int U = 8 / RB;  // steps whose loads are in flight together
    const int lane = threadIdx.x & 63, col = lane & 15, lg = lane >> 4;
    const int64_t K = g.a.in_features;
    const uint16_t *xp = (const uint16_t *)g.a.x + m * g.a.x_stride + 8 * lg, *ap[RB];
#pragma unroll
    for (int r = 0; r < RB; r++) {
        const int j = rank0 + 16 * r + col;
        ap[r] = (const uint16_t *)g.a.a + ((int64_t)id * g.a.rank + (j < g.a.rank ? j : g.a.rank - 1)) * K + 8 * lg;
    }
    f32x4 acc[RB];
#pragma unroll
    for (int r = 0; r < RB; r++) acc[r] = f32x4{0.f, 0.f, 0.f, 0.f};
    int s, end;
    const bool tail = down_steps(g, slice, &s, &end);
    for (; s < end; s += U) {
        u32x4 x[U], a[U][RB];
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (s + u >= end) break;
            const int64_t k = (int64_t)(s + u) * 32;
            x[u] = load8<W>(xp + k);
#pragma unroll
            for (int r = 0; r < RB; r++) a[u][r] = load8<W>(ap[r] + k);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (s + u >= end) break;
#pragma unroll
            for (int r = 0; r < RB; r++) acc[r] = mfma<BF>(a[u][r], x[u], acc[r]);
        }
    }
    if (tail) {
        const int64_t k = K / 32 * 32, left = K - k - 8 * lg;
        const u32x4 x = load8<W>(xp + k, left, xp - 8 * lg);
#pragma unroll
        for (int r = 0; r < RB; r++) acc[r] = mfma<BF>(load8<W>(ap[r] + k, left, ap[r] - 8 * lg), x, acc[r]);
    }
    down_join<RB>(g, acc, m, own, rank0, slice, lds);
}

// A slice for 64 tokens of many adapters: each step's tokens with every
// adapter in turn, the products kept in their own tokens' columns.
template <int RB, bool BF, int W>
__device__ __forceinline__ void down_all(const AdapterArgs &g, int64_t m0, int rank0, int slice, float *lds) {
    // adapters whose loads are in flight together (538 tokens of 24 adapters
    // in turn, 4000 -> 11008, rank 16, BF16, low-rank values in two parts: with
    // eight, and two in the up launch, 82 us, with four and one 91; with the
    // three parts of now 87)
    constexpr int IDS = RB == 1 ? 8 : 2;
    const int lane = threadIdx.x & 63, col = lane & 15, lg = lane >> 4;
    const int64_t K = g.a.in_features;
    const int mine = adapter_of(g, m0 + lane);
    const uint64_t own = __ballot(mine >= 0);
    if (!own) return;
    const uint16_t *xp[4];
#pragma unroll
    for (int c = 0; c < 4; c++) {
        const int64_t m = m0 + 16 * c + col;
        xp[c] = (const uint16_t *)g.a.x + (m < g.a.tokens ? m : g.a.tokens - 1) * g.a.x_stride;
    }
    int64_t row[RB];
#pragma unroll
    for (int r = 0; r < RB; r++) {
        const int j = rank0 + 16 * r + col;
        row[r] = (j < g.a.rank ? j : g.a.rank - 1) * K;
    }
    f32x4 acc[4][RB];
#pragma unroll
    for (int c = 0; c < 4; c++)
#pragma unroll
        for (int r = 0; r < RB; r++) acc[c][r] = f32x4{0.f, 0.f, 0.f, 0.f};
    int s, end;
    if (down_steps(g, slice, &s, &end)) end++;  // (the step that in_features ends inside among them: all loads are checked)
    for (; s < end; s++) {
        const int64_t k = (int64_t)s * 32 + 8 * lg;
        u32x4 x[4];
#pragma unroll
        for (int c = 0; c < 4; c++) x[c] = load8<W>(xp[c] + k, K - k, xp[c]);
        for (uint64_t todo = own; todo;) {
            int id[IDS];
            u32x4 a[IDS][RB];
            uint64_t same[IDS];
#pragma unroll
            for (int i = 0; i < IDS; i++) {
                same[i] = 0;
                id[i] = i > 0 ? id[0] : 0;  // (none left: the first's loads again)
                if (todo) {
                    id[i] = __builtin_amdgcn_readlane(mine, __ffsll((unsigned long long)todo) - 1);
                    same[i] = __ballot(mine == id[i]);
                    todo &= ~same[i];
                }
            }
#pragma unroll
            for (int i = 0; i < IDS; i++) {
                const uint16_t *p = (const uint16_t *)g.a.a + (int64_t)id[i] * g.a.rank * K;
#pragma unroll
                for (int r = 0; r < RB; r++) a[i][r] = load8<W>(p + row[r] + k, K - k, p);
            }
#pragma unroll
            for (int i = 0; i < IDS; i++)
#pragma unroll
                for (int c = 0; c < 4; c++)
#pragma unroll
                    for (int r = 0; r < RB; r++) {
                        const f32x4 t = mfma<BF>(a[i][r], x[c], acc[c][r]);
#pragma unroll
                        for (int e = 0; e < 4; e++) acc[c][r][e] = same[i] >> (16 * c + col) & 1 ? t[e] : acc[c][r][e];
                    }
        }
    }
#pragma unroll
    for (int c = 0; c < 4; c++) {
        const uint32_t o = (uint32_t)(own >> (16 * c)) & 0xffffu;
        if (o) down_join<RB>(g, acc[c], (int)m0 + 16 * c + col, o, rank0, slice, lds);
    }
}

// A slice for 64 tokens and one adapter, through LDS: stages of 64 columns of
// the tokens' rows and of A, read in whole 128-byte lines (16 bytes a lane
// straight into the operands touch each line twice, and the L1 does not hold
// it that long), kAhead stages of them in flight in registers, written to LDS
// with the 16-byte chunks of a row permuted by the row (no bank is hit twice).
// The waves split the product, so there is no sum over them.
constexpr int kAhead = 6;
template <int RB, bool BF>
__device__ __forceinline__ void down_staged(const AdapterArgs &g, int64_t m0, int id, uint64_t own, int rank0, int slice,
                                            u32x4 *lds) {
    constexpr int kRows = 64 + 16 * RB, kLoads = (kRows * 8 + 64 * kDown - 1) / (64 * kDown);  // rows of a stage, chunks a thread
    constexpr int kCols = RB == 4 ? 2 : 1;  // token groups of a wave
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15, lg = lane >> 4;
    const int64_t K = g.a.in_features;
    const int k0 = slice * g.steps * 32;
    const int64_t stop = (int64_t)k0 + g.steps * 32 < K ? (int64_t)k0 + g.steps * 32 : K;
    const int stages = (int)((stop - k0 + 63) / 64);
    const uint16_t *src[kLoads];
    int at[kLoads], chunk[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; i++) {
        int row = (tid + i * 64 * kDown) >> 3;
        chunk[i] = tid & 7;
        if (row >= kRows) row = kRows - 1;  // (a copy, written to the same place)
        at[i] = row * 8 + (chunk[i] ^ (row & 7));
        if (row < 64) {
            const int64_t m = m0 + row < g.a.tokens ? m0 + row : g.a.tokens - 1;
            src[i] = (const uint16_t *)g.a.x + m * g.a.x_stride;
        } else {
            const int j = rank0 + row - 64;
            src[i] = (const uint16_t *)g.a.a + ((int64_t)id * g.a.rank + (j < g.a.rank ? j : g.a.rank - 1)) * K;
        }
    }
    u32x4 held[kAhead][kLoads];
    auto load = [&](int stage, u32x4 v[kLoads]) {
#pragma unroll
        for (int i = 0; i < kLoads; i++) {
            const int64_t k = (int64_t)k0 + 64 * stage + 8 * chunk[i];
            v[i] = load8<8>(src[i] + k, stop - k, src[i]);
        }
    };
    f32x4 acc[kCols];
#pragma unroll
    for (int c = 0; c < kCols; c++) acc[c] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int rb = wave % RB, cg = RB == 4 ? wave / 4 * 2 : wave / RB;  // its ranks and first token group (from four on: none)
    const bool works = cg < 4;
#pragma unroll
    for (int d = 0; d < kAhead; d++) load(d, held[d]);
    for (int s0 = 0; s0 < stages; s0 += kAhead) {
#pragma unroll
        for (int d = 0; d < kAhead; d++) {
            if (s0 + d >= stages) break;
            u32x4 *buf = lds + (d & 1) * kRows * 8;  // (kAhead is even)
#pragma unroll
            for (int i = 0; i < kLoads; i++) buf[at[i]] = held[d][i];
            // every wave has written this stage, and is done with the last
            // one's buffer, which the next stage goes to; loads stay in flight
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            load(s0 + d + kAhead, held[d]);
            if (works) {
                const int ar = 64 + 16 * rb + col;
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const u32x4 a = buf[ar * 8 + ((4 * u + lg) ^ (ar & 7))];
#pragma unroll
                    for (int c = 0; c < kCols; c++) {
                        const int xr = 16 * (cg + c) + col;
                        acc[c] = mfma<BF>(a, buf[xr * 8 + ((4 * u + lg) ^ (xr & 7))], acc[c]);
                    }
                }
            }
        }
    }
    if (works) {
#pragma unroll
        for (int c = 0; c < kCols; c++) {
            const int t = 16 * (cg + c) + col, j = rank0 + 16 * rb + 4 * lg;
            if (!(own >> t & 1)) continue;
            float *dst = g.low + ((int64_t)slice * g.a.tokens + m0 + t) * g.a.rank + j;
            if (g.a.rank % 4 == 0) {
                if (j < g.a.rank) *reinterpret_cast<f32x4 *>(dst) = acc[c];
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (j + i < g.a.rank) dst[i] = acc[c][i];
            }
        }
    }
    __syncthreads();  // the buffers are free for the next pass
}

template <int RB, int CB, bool BF, int W>
__global__ __launch_bounds__(64 * kDown, 4) void adapter_down_kernel(AdapterArgs g) {
    extern __shared__ __align__(16) float down_lds[];
    // (all first slots in front: most others end at once)
    const int per_slot = gridDim.x / g.slots, slot = blockIdx.x / per_slot;
    int tile, slice;
    place_of(g, blockIdx.x - slot * per_slot, g.slices, &tile, &slice);
    if (tile >= g.tiles) return;
    const int64_t m0 = (int64_t)tile * 16 * CB;
    if constexpr (CB == 1) {
        // the slot's adapters: those of every slots-th column that is its
        // adapter's first
        __shared__ __align__(16) int order[CB == 1 ? 2 * kOrdered : 1];  // (its second half is read as vectors)
        if (g.order_by == ORDER_GROUP) {
            order_tokens(g, order);
            if (slice == 0 && slot == 0 && threadIdx.x < 16 && tile * 16 + (int)threadIdx.x < g.a.tokens)
                g.order[tile * 16 + threadIdx.x] = order[tile * 16 + threadIdx.x];
        }
        int m, mine;
        few_token(g, tile, order, &m, &mine);
        bool first = mine >= 0;
        auto unlike = [&](auto d) {  // the adapter d columns before, within the row of 16 lanes
            const int other = __builtin_amdgcn_update_dpp(-1, mine, 0x110 + decltype(d)::value, 0xf, 0xf, false);
            first &= other != mine;
        };
        unlike(std::integral_constant<int, 1>{});
        unlike(std::integral_constant<int, 2>{});
        unlike(std::integral_constant<int, 3>{});
        unlike(std::integral_constant<int, 4>{});
        unlike(std::integral_constant<int, 5>{});
        unlike(std::integral_constant<int, 6>{});
        unlike(std::integral_constant<int, 7>{});
        unlike(std::integral_constant<int, 8>{});
        unlike(std::integral_constant<int, 9>{});
        unlike(std::integral_constant<int, 10>{});
        unlike(std::integral_constant<int, 11>{});
        unlike(std::integral_constant<int, 12>{});
        unlike(std::integral_constant<int, 13>{});
        unlike(std::integral_constant<int, 14>{});
        unlike(std::integral_constant<int, 15>{});
        uint32_t firsts = (uint32_t)__ballot(first) & 0xffffu;
        for (int i = 0; firsts; i++, firsts &= firsts - 1) {
            if (i % g.slots != slot) continue;
            const int id = __builtin_amdgcn_readlane(mine, __ffs(firsts) - 1);
            const uint32_t own = (uint32_t)__ballot(mine == id) & 0xffffu;
            for (int r = 0; r < g.a.rank; r += 16 * RB) down_one<RB, BF, W>(g, m, id, own, r, slice, down_lds);
        }
    } else {
        // up to kShared adapters: the slots take them in turn; more: the
        // first slot takes all at once
        constexpr int kAll = RB < 2 ? RB : 2;
        const int mine = adapter_of(g, m0 + (threadIdx.x & 63));
        const uint64_t own = __ballot(mine >= 0);
        int distinct = 0;
        for (uint64_t todo = own; todo && distinct <= kShared; distinct++)
            todo &= ~__ballot(mine == __builtin_amdgcn_readlane(mine, __ffsll((unsigned long long)todo) - 1));
        if (W != 8 || distinct > kShared) {
            if (slot == 0)
                for (int r = 0; r < g.a.rank; r += kAll * 16) down_all<kAll, BF, W>(g, m0, r, slice, down_lds);
            return;
        }
        int k = 0;
        for (uint64_t todo = own; todo; k++) {
            const int id = __builtin_amdgcn_readlane(mine, __ffsll((unsigned long long)todo) - 1);
            const uint64_t same = __ballot(mine == id);
            todo &= ~same;
            if (k % g.slots != slot) continue;
            for (int r = 0; r < g.a.rank; r += 16 * RB)
                down_staged<RB, BF>(g, m0, id, same, r, slice, reinterpret_cast<u32x4 *>(down_lds));
        }
    }
}

// -------------------------------------------------------------------------- up

// The sum of slices first, first + step, .. of low[m, j0 .. j0 + 7].
template <int U>  // slices whose loads are in flight together
__device__ __forceinline__ void low_sum(const AdapterArgs &g, int64_t m, int j0, int first, int step, f32x4 v[2]) {
    const int r = g.a.rank;
    v[0] = v[1] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int s0 = first; s0 < g.slices; s0 += U * step) {
        f32x4 p[U][2];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int s = s0 + u * step;
            p[u][0] = p[u][1] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (s >= g.slices) continue;
            const float *src = g.low + ((int64_t)s * g.a.tokens + m) * r + j0;
            if (r % 4 == 0) {
                if (j0 < r) p[u][0] = *reinterpret_cast<const f32x4 *>(src);
                if (j0 + 4 < r) p[u][1] = *reinterpret_cast<const f32x4 *>(src + 4);
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (j0 + e < r) p[u][e >> 2][e & 3] = src[e];
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            v[0] += p[u][0];
            v[1] += p[u][1];
        }
    }
}

// Sixteen tokens' low-rank values (of token col, ranks 32 kk + 8 lg .. + 7 in
// a lane), FP32 in the first two of the kLowParts<BF> words of each kk in
// `dst`, become their 16-bit parts there; returns the power of two that the
// lane's token was scaled by.  BF16: three parts of eight bits, cut off, whose
// sum is the value exactly.  FP16: two of eleven bits, rounded to nearest (the
// second one's sign is a bit more): 2^-24 of the value, as an FP32 operation's
// rounding, or 2^-39 of the token's largest where that is more.
template <bool BF>
constexpr int kLowParts = BF ? 3 : 2;
template <bool BF>
__device__ __forceinline__ int low_parts(int kks, u32x4 *dst) {
    const int lane = threadIdx.x & 63;
    int sh = 0;
    if constexpr (!BF) {
        float top = 0.f;
        for (int x = 0; x < 2 * kks; x++) {  // (two parts: no word between)
            const f32x4 v = __builtin_bit_cast(f32x4, dst[x * 64 + lane]);
#pragma unroll
            for (int e = 0; e < 4; e++) top = fabsf(v[e]) < __builtin_inff() ? fmaxf(top, fabsf(v[e])) : top;
        }
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        // the largest finite one to 2^14: its parts are normal numbers and so are those
        // of values 2^-17 of it
        if (top > 0.f) sh = 15 - __builtin_amdgcn_frexp_expf(top);
    }
    for (int kk = 0; kk < kks; kk++) {
        u32x4 *word = dst + kk * kLowParts<BF> * 64 + lane;
        const f32x4 v[2] = {__builtin_bit_cast(f32x4, word[0]), __builtin_bit_cast(f32x4, word[64])};
        u32x4 part[kLowParts<BF>];
#pragma unroll
        for (int i = 0; i < 4; i++) {
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const float x0 = v[i >> 1][(2 * i + e) & 3];
                float x = BF ? x0 : __builtin_amdgcn_ldexpf(x0, sh);
                const bool finite = fabsf(x) < __builtin_inff();
#pragma unroll
                for (int k = 0; k < kLowParts<BF>; k++) {
                    const uint16_t b = !BF ? store16<BF>(x) : x == x ? (uint16_t)(__float_as_uint(x) >> 16) : (uint16_t)0x7fc0;
                    part[k][i] = e == 0 ? b : part[k][i] | (uint32_t)b << 16;
                    x = finite ? x - load16<BF>(b) : 0.f;  // (an infinity or a NaN has no rest)
                }
            }
        }
#pragma unroll
        for (int k = 0; k < kLowParts<BF>; k++) word[64 * k] = part[k];
    }
    return sh;
}

// CB 1: 16 tokens a workgroup of four waves and one unit of kUp outputs; the
// waves split the slices to add, and then the adapters.  CB 4: 64 tokens and
// eight waves; two of them add 16 tokens up, and then each takes a unit of
// its own for all (eight: the sums are read half as often).  Product t's row
// 4 a + i is output 16 a + 4 t + i of the unit, so a lane (rows 4 lg + i of
// all four) holds outputs 16 lg .. 16 lg + 15 of its token.  The loads of y
// and of the first adapters' B go ahead of the low-rank sums.  KB: steps of
// 32 ranks whose loads are in flight together.
template <int CB, bool BF, int W, bool YV, int KB>
__global__ __launch_bounds__(CB == 1 ? 256 : 512, 2) void adapter_up_kernel(AdapterArgs g) {
    constexpr int IDS = (CB == 1 ? 4 : 2) / KB;  // adapters whose loads are in flight together (as many as registers hold)
    constexpr int PT = kLowParts<BF>;
    extern __shared__ u32x4 parts[];             // [4][kks][PT][64]
    __shared__ int shifts[kTokens];
    int tile, block;
    place_of(g, blockIdx.x, g.blocks, &tile, &block);
    if (tile >= g.tiles) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, lg = lane >> 4;
    const int kks = (g.a.rank + 31) / 32, each = kks * PT * 64;
    const int64_t m0 = (int64_t)tile * 16 * CB, N = g.a.out_features;
    // the tokens: CB 1, of column col; CB 4, of lane
    int mine, m1 = 0;
    bool present;
    if constexpr (CB == 1) {
        present = few_token(g, tile, g.order, &m1, &mine);
    } else {
        mine = adapter_of(g, m0 + lane);
        present = m0 + lane < g.a.tokens;
    }
    const uint64_t whole = CB == 1 ? 0xffffull : ~0ull;
    const uint64_t own = __ballot(mine >= 0) & whole, here = __ballot(present) & whole;
    auto token = [&](int c) -> int64_t {  // of column col of group c
        if constexpr (CB == 1) return m1;
        const int64_t m = m0 + 16 * c + col;
        return m < g.a.tokens ? m : g.a.tokens - 1;
    };
    auto take = [&](uint64_t &todo, int &id) -> uint64_t {  // the next adapter and its tokens
        id = __builtin_amdgcn_readlane(mine, __ffsll((unsigned long long)todo) - 1);
        const uint64_t same = __ballot(mine == id) & own;
        todo &= ~same;
        return same;
    };
    // this wave's tokens (those without an adapter are copied) and outputs
    uint64_t held = here;
    if constexpr (CB == 1) {
        held = wave == 0 ? here & ~own : 0;
        int k = 0, id;
        for (uint64_t todo = own; todo; k++) {
            const uint64_t same = take(todo, id);
            if (k % 4 == wave) held |= same;
        }
    }
    const int64_t n0 = CB == 1 ? (int64_t)block * kUp : ((int64_t)block * kUpWaves + wave) * kUp, n = n0 + 16 * lg;
    if (n0 >= N) held = 0;

    u32x4 yv[CB][2];
    uint16_t ys[CB][16];
#pragma unroll
    for (int c = 0; c < CB; c++) {
        const bool on = held >> (16 * c + col) & 1;
        const uint16_t *y = (const uint16_t *)g.a.y + token(c) * g.a.y_stride + n;
        if constexpr (YV) {
            // (also of tokens that are not this wave's)
            yv[c][0] = load8<8>(y, N - n, (const uint16_t *)g.a.y);
            yv[c][1] = load8<8>(y + 8, N - n - 8, (const uint16_t *)g.a.y);
        } else {
#pragma unroll
            for (int e = 0; e < 16; e++) ys[c][e] = on && n + e < N ? y[e] : 0;
        }
    }
    int64_t row[4];
#pragma unroll
    for (int t = 0; t < 4; t++) {
        const int64_t at = n0 + 16 * (col >> 2) + 4 * t + (col & 3);
        row[t] = (at < N ? at : N - 1) * g.a.rank + 8 * lg;
    }
    u32x4 bv[IDS][KB][4];
    int ids[IDS];
    uint64_t same[IDS], todo = held & own;
    auto next = [&]() {
#pragma unroll
        for (int i = 0; i < IDS; i++) {
            same[i] = 0;
            ids[i] = 0;
            if (todo) same[i] = take(todo, ids[i]);
        }
    };
    auto load_b = [&](int kk0) {
#pragma unroll
        for (int i = 0; i < IDS; i++) {
            if (!same[i]) break;
            const uint16_t *b = (const uint16_t *)g.a.b + (int64_t)ids[i] * N * g.a.rank;
#pragma unroll
            for (int k = 0; k < KB; k++)
#pragma unroll
                for (int t = 0; t < 4; t++)
                    bv[i][k][t] = load8<W>(b + row[t] + 32 * (kk0 + k), g.a.rank - 32 * (kk0 + k) - 8 * lg, b);
        }
    };
    next();
    load_b(0);

    // the low-rank values
    const int group = wave & 3, tl = CB == 1 ? mine : __shfl(mine, 16 * group + col, 64);
    const float scale = tl >= 0 ? (g.a.scales ? g.a.scales[tl] : 1.f) : 0.f;
    const bool any = __any(tl >= 0);
    if (any)
        for (int kk = CB == 1 ? 0 : wave >> 2; kk < kks; kk += CB == 1 ? 1 : 2) {
            f32x4 v[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
            if (tl >= 0) low_sum<CB == 1 ? 2 : 4>(g, token(group), 32 * kk + 8 * lg, CB == 1 ? wave : 0, CB == 1 ? 4 : 1, v);
            if (CB > 1) {
                v[0] *= scale;
                v[1] *= scale;
            }
            parts[group * each + (PT * kk) * 64 + lane] = __builtin_bit_cast(u32x4, v[0]);
            parts[group * each + (PT * kk + 1) * 64 + lane] = __builtin_bit_cast(u32x4, v[1]);
        }
    __syncthreads();
    if constexpr (CB == 1) {
        // (x, the rank words, dealt over the waves)
        for (int x = wave; any && x < 2 * kks; x += 4) {
            u32x4 *word = parts + (x / 2 * PT + x % 2) * 64 + lane;
            f32x4 v = __builtin_bit_cast(f32x4, *word);
#pragma unroll
            for (int w = 1; w < 4; w++) v += __builtin_bit_cast(f32x4, word[w * each]);
            *word = __builtin_bit_cast(u32x4, v * scale);
        }
        __syncthreads();
    }
    if (any && wave < CB) {
        const int sh = low_parts<BF>(kks, parts + wave * each);
        if (lane < 16) shifts[16 * wave + lane] = sh;
    }
    __syncthreads();
    if (!held) return;

    f32x4 acc[CB][4];
#pragma unroll
    for (int c = 0; c < CB; c++)
#pragma unroll
        for (int t = 0; t < 4; t++) acc[c][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    while (same[0]) {
        for (int kk0 = 0; kk0 < kks; kk0 += KB) {
            if (kk0 > 0) load_b(kk0);
#pragma unroll
            for (int i = 0; i < IDS; i++)
#pragma unroll
                for (int c = 0; c < CB; c++) {
                    const uint32_t tokens = (uint32_t)(same[i] >> (16 * c)) & 0xffffu;
                    if (!tokens) continue;
                    f32x4 d[4];
#pragma unroll
                    for (int t = 0; t < 4; t++) d[t] = acc[c][t];
#pragma unroll
                    for (int k = 0; k < KB; k++)
                        if (kk0 + k < kks) {
                            const u32x4 *word = parts + c * each + (kk0 + k) * PT * 64 + lane;
#pragma unroll
                            for (int j = 0; j < PT; j++) {
                                const u32x4 p = word[64 * j];
#pragma unroll
                                for (int t = 0; t < 4; t++) d[t] = mfma<BF>(bv[i][k][t], p, d[t]);
                                // (a part at a time: three together take registers that a third wave a
                                // SIMD, or outputs that are not vectors, have need of)
                                if constexpr (BF && (CB == 1 || !YV)) __builtin_amdgcn_sched_barrier(0);
                            }
                        }
                    if (tokens >> col & 1) {
#pragma unroll
                        for (int t = 0; t < 4; t++) acc[c][t] = d[t];
                    }
                }
        }
        next();
        load_b(0);
    }
    // An infinite element of B times a zero part, or one of another sign than
    // the first part, makes a NaN of the sum: those sums are formed again of
    // the whole low-rank values, one a lane at a time.
#pragma unroll
    for (int c = 0; c < CB; c++) {
        float none[2] = {0.f, 0.f};  // (a NaN where a sum is infinite or a NaN)
#pragma unroll
        for (int e = 0; e < 16; e++) none[e & 1] = __builtin_fmaf(acc[c][e >> 2][e & 3], 0.f, none[e & 1]);
        if (!__any(none[0] != none[1])) continue;
        uint32_t odd = 0;
#pragma unroll
        for (int e = 0; e < 16; e++) odd |= (uint32_t)(acc[c][e >> 2][e & 3] != acc[c][e >> 2][e & 3]) << e;
        const int id = CB == 1 ? mine : __shfl(mine, 16 * c + col, 64);
#pragma unroll 1
        for (; __any(odd != 0); odd &= odd - 1) {
            const int at = odd ? __ffs(odd) - 1 : 0;
            float sum = 0.f;
            if (odd && id >= 0 && n + at < N) {
                const uint16_t *b = (const uint16_t *)g.a.b + ((int64_t)id * N + n + at) * g.a.rank;
#pragma unroll 1
                for (int j = 0; j < g.a.rank; j++) {
                    const u32x4 *word = parts + c * each + (j >> 5) * PT * 64 + (j >> 3 & 3) * 16 + col;
                    float low = 0.f;
#pragma unroll
                    for (int k = 0; k < PT; k++) low += load16<BF>(reinterpret_cast<const uint16_t *>(word + 64 * k)[j & 7]);
                    sum += low * load16<BF>(b[j]);
                    if (sum != sum) break;
                }
            }
#pragma unroll
            for (int e = 0; e < 16; e++)
                if (odd && e == at) acc[c][e >> 2][e & 3] = sum;
        }
    }
#pragma unroll
    for (int c = 0; c < CB; c++) {
        if (!(held >> (16 * c + col) & 1)) continue;
        const bool add = own >> (16 * c + col) & 1;
        uint16_t *out = (uint16_t *)g.a.out + token(c) * g.a.out_stride + n;
        const int sh = !BF && add ? shifts[16 * c + col] : 0;
        uint16_t r[16];
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const uint16_t v = YV ? (uint16_t)(yv[c][e >> 3][(e & 7) >> 1] >> (16 * (e & 1))) : ys[c][e];
            const float d = acc[c][e >> 2][e & 3];
            r[e] = add ? store16<BF>(load16<BF>(v) + (BF ? d : __builtin_amdgcn_ldexpf(d, -sh))) : v;
        }
        if constexpr (YV) {
#pragma unroll
            for (int v = 0; v < 2; v++)
                if (n + 8 * v < N) {
                    u32x4 w;
#pragma unroll
                    for (int i = 0; i < 4; i++) w[i] = (uint32_t)r[8 * v + 2 * i] | (uint32_t)r[8 * v + 2 * i + 1] << 16;
                    *reinterpret_cast<u32x4 *>(out + 8 * v) = w;
                }
        } else {
#pragma unroll
            for (int e = 0; e < 16; e++)
                if (n + e < N) out[e] = r[e];
        }
    }
}

// The launches' shapes: from the sizes alone, as the adapter numbers are on
// the device.
AdapterArgs adapter_args(const orth_hip_adapter_t &a, int cus) {
    AdapterArgs g;
    g.a = a;
    g.low = nullptr;
    g.order = nullptr;
    // 16 tokens a tile, also where wider tiles would leave the up launch too
    // few workgroups (911 tokens, 1000 -> 999: 34 us so, 20 with 16; 1,024
    // tokens, 4096 -> 4096: 17 and 36)
    const int64_t wide_tiles = (a.tokens + kTokens - 1) / kTokens, wide_blocks = (a.out_features + kUpWaves * kUp - 1) / (kUpWaves * kUp);
    g.few = a.tokens <= kFew || wide_tiles * wide_blocks < cus / 4;
    const bool few = g.few;
    g.tiles = (int)(few ? (a.tokens + 15) / 16 : wide_tiles);
    const int64_t steps = (a.in_features + 31) / 32;
    g.order_by = !few || a.tokens <= 16 || a.count < 1 || a.count >= a.tokens ? ORDER_NONE
               : a.tokens <= 64 && a.count < (1 << 25) ? ORDER_WAVE
               : a.tokens <= kOrdered && a.count < (1 << 22) ? ORDER_GROUP : ORDER_NONE;
    // slots: as many as a 16-token tile can have adapters; in their order, as
    // a tile has on average and one (the tiles' adapters are then taken in turn)
    int64_t most = a.tokens < 16 ? a.tokens : 16;
    if (a.count < most) most = a.count < 1 ? 1 : a.count;
    const int64_t average = a.count / g.tiles + 1;
    if (g.order_by != ORDER_NONE && average < most) most = average;
    g.slots = few ? (int)most : 2;  // (many tokens: a tile mostly has one adapter, or two where a run ends)
    // down: slices for a workgroup of eight waves a CU, of four steps at
    // least; every slice is a partial more that each workgroup of the second
    // launch adds
    int64_t slices = (int64_t)cus / (g.tiles * (int64_t)(few ? g.slots : 1));
    if (slices > (steps + 3) / 4) slices = (steps + 3) / 4;
    if (slices > 8) slices = 8;
    if (slices < 1) slices = 1;
    g.steps = (int)((steps + slices - 1) / slices);
    if (!few) g.steps += g.steps & 1;  // whole 128-byte lines
    g.slices = (int)((steps + g.steps - 1) / g.steps);
    const int64_t span = few ? kUp : kUpWaves * kUp;
    g.blocks = (int)((a.out_features + span - 1) / span);
    g.chunk = g.tiles >= 8 ? (g.tiles + 7) / 8 : 0;
    return g;
}

bool multiple(const void *p, int64_t stride, int n) { return reinterpret_cast<uintptr_t>(p) % (2 * n) == 0 && stride % n == 0; }

// Launches a kernel with dynamic LDS, past the default limit where it asks for more.
template <class Kernel>
hipError_t launch_lds(Kernel kernel, unsigned groups, int threads, size_t lds, hipStream_t stream, const AdapterArgs &g) {
    if (lds > 48 * 1024) {
        hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                           hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    kernel<<<groups, threads, lds, stream>>>(g);
    return hipGetLastError();
}

template <int RB, bool BF>
hipError_t down_launch(const AdapterArgs &g, unsigned groups, hipStream_t stream) {
    const bool few = g.few, wide = multiple(g.a.x, g.a.x_stride, 8) && multiple(g.a.a, g.a.in_features, 8);
    const size_t join = (size_t)kDown * 16 * RB * 17 * sizeof(float), staged = (size_t)2 * (64 + 16 * RB) * 128;
    const size_t lds = few || join > staged ? join : staged;
    auto go = [&](auto kernel) { return launch_lds(kernel, groups, 64 * kDown, lds, stream, g); };
    if (few) return wide ? go(adapter_down_kernel<RB, 1, BF, 8>) : go(adapter_down_kernel<RB, 1, BF, 1>);
    return wide ? go(adapter_down_kernel<RB, 4, BF, 8>) : go(adapter_down_kernel<RB, 4, BF, 1>);
}

template <int CB, bool BF>
hipError_t up_launch(const AdapterArgs &g, unsigned groups, hipStream_t stream) {
    const size_t lds = (size_t)4 * ((g.a.rank + 31) / 32) * kLowParts<BF> * 64 * sizeof(u32x4);
    const bool yv = g.a.out_features % 8 == 0 && multiple(g.a.y, g.a.y_stride, 8) && multiple(g.a.out, g.a.out_stride, 8);
    const bool one = g.a.rank <= 32;  // one step of ranks: more adapters' loads at a time
    auto go = [&](auto kernel) { return launch_lds(kernel, groups, CB == 1 ? 256 : 64 * kUpWaves, lds, stream, g); };
    if (multiple(g.a.b, g.a.rank, 8)) {
        if (yv) return one ? go(adapter_up_kernel<CB, BF, 8, true, 1>) : go(adapter_up_kernel<CB, BF, 8, true, 2>);
        return one ? go(adapter_up_kernel<CB, BF, 8, false, 1>) : go(adapter_up_kernel<CB, BF, 8, false, 2>);
    }
    if (multiple(g.a.b, g.a.rank, 4)) {
        if (yv) return one ? go(adapter_up_kernel<CB, BF, 4, true, 1>) : go(adapter_up_kernel<CB, BF, 4, true, 2>);
        return go(adapter_up_kernel<CB, BF, 4, false, 2>);
    }
    return go(adapter_up_kernel<CB, BF, 1, false, 2>);
}

template <bool BF>
hipError_t adapter_launch(const AdapterArgs &g, hipStream_t stream) {
    const int64_t padded = g.chunk > 0 ? (int64_t)g.chunk * 8 : g.tiles, parts = (int64_t)g.slices * g.slots;
    if (padded * (g.blocks > parts ? g.blocks : parts) > (int64_t)UINT32_MAX / 512) return hipErrorInvalidConfiguration;
    const unsigned down = (unsigned)(padded * parts), up = (unsigned)(padded * g.blocks);
    if (g.a.count > 0) {
        hipError_t e = g.a.rank <= 16 ? down_launch<1, BF>(g, down, stream)
                     : g.a.rank <= 32 ? down_launch<2, BF>(g, down, stream)
                                      : down_launch<4, BF>(g, down, stream);
        if (e != hipSuccess) return e;
    }
    return g.few ? up_launch<1, BF>(g, up, stream) : up_launch<4, BF>(g, up, stream);
}

// The tokens of a pair of launches: a launch holds fewer than 2^32 threads (one
// past that runs another number of workgroups, without an error), which leaves
// room for 2^5 workgroups a 64-token tile, or for outputs of 512 GB.
constexpr int64_t kLaunchTokens = 1 << 24;

// Tokens t .. of a call, as a call of their own.
orth_hip_adapter_t adapter_part(const orth_hip_adapter_t &a, int64_t t) {
    orth_hip_adapter_t p = a;
    p.x = (const uint16_t *)a.x + t * a.x_stride;
    p.y = (const uint16_t *)a.y + t * a.y_stride;
    p.out = (uint16_t *)a.out + t * a.out_stride;
    p.adapters = a.adapters + t;
    p.tokens = a.tokens - t < kLaunchTokens ? a.tokens - t : kLaunchTokens;
    return p;
}

}  // namespace

int64_t adapter_workspace_bytes(const orth_hip_adapter_t &a, int cus) {
    if (a.count == 0) return 0;
    int64_t most = 0;
    const int64_t last = (a.tokens - 1) / kLaunchTokens * kLaunchTokens;
    for (int64_t t = 0; t <= last; t += last > 0 ? last : 1) {  // (all parts but the last are alike)
        const orth_hip_adapter_t p = adapter_part(a, t);
        const AdapterArgs g = adapter_args(p, cus);
        const int64_t bytes = (int64_t)g.slices * p.tokens * p.rank * 4 + (g.order_by == ORDER_GROUP ? p.tokens * 4 : 0);
        most = bytes > most ? bytes : most;
    }
    return most;
}

hipError_t launch_adapter_add(const orth_hip_adapter_t &a, int cus, void *work, hipStream_t stream) {
    for (int64_t t = 0; t < a.tokens; t += kLaunchTokens) {
        AdapterArgs g = adapter_args(adapter_part(a, t), cus);
        g.low = static_cast<float *>(work);
        if (g.order_by == ORDER_GROUP) g.order = reinterpret_cast<int *>(g.low + (int64_t)g.slices * g.a.tokens * g.a.rank);
        const hipError_t e = a.dtype == ORTH_DT_BF16 ? adapter_launch<true>(g, stream) : adapter_launch<false>(g, stream);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace orth
