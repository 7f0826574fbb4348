// Low-rank adapters of many requests beside a shared projection:
// out[m] = y[m] + scale_i (x[m] A_i^T) B_i^T with i = adapters[m].
//
// Two launches with the low-rank values between them in FP32, one partial
// per slice of in_features, added in order by the second:
//
//   down  low[m, j] = sum_k x[m, k] A_i[j, k]
//   up    out[m, n] = y[m, n] + sum_j (scale_i low[m, j]) B_i[n, j]
//
// Both go through v_mfma_f32_16x16x32 with 16 consecutive tokens as the
// columns: x, A and B enter by 16-byte loads as they lie; products are exact,
// sums FP32.  For every adapter among the 16 tokens (found by ballots) the
// product is formed for all columns and kept in those of its own tokens: a
// run of one prompt's tokens is one product, a decode batch of 16 requests
// reads each of their adapters once, and what one adapter holds cannot reach
// another's tokens.  The low-rank values enter the second product as two
// 16-bit parts (16 bits of them or more; one part would cost as much as the
// output's own rounding), FP16 ones scaled by a power of two per token, so
// that none overflows or loses its low bits.
//
// Bound by reading the adapters (few tokens: workgroups of 16 tokens, whose
// waves split in_features, then the adapters) or x, y and out (many: 64
// tokens a workgroup share each adapter's loads).
#include "orth_serve.h"

namespace orth {

namespace {

constexpr int kTokens = 64;    // tokens of a tile, where they are many
constexpr int kFew = 256;      // up to here, tiles of 16: decode batches, whose adapters differ by token
constexpr int kUp = 64;        // outputs a wave takes at a time
constexpr int kDown = 8;       // waves of a down workgroup: steps in flight without more partials to add
constexpr int kShared = 4;     // adapters of a 64-token tile up to which its tokens are taken together

struct AdapterArgs {
    orth_hip_adapter_t a;
    float *low;        // [slices][tokens][rank]
    int tiles;         // of 16 or 64 tokens
    int slices, steps; // slices of in_features, and steps of 32 in each
    int blocks;        // up: blocks of out_features
    int affine;        // all workgroups of a tile on one XCD
};

// Workgroup -> (tile, part of it): neighbours in blockIdx go to different
// XCDs, eight in turn; a tile's partials are read from the L2 they went to.
__device__ __forceinline__ void place_of(const AdapterArgs &g, int parts, int *tile, int *part) {
    const int b = blockIdx.x;
    if (g.affine) {
        const int x = b & 7, q = b >> 3;
        *tile = (q / parts) * 8 + x;
        *part = q - (q / parts) * parts;
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

// Eight 16-bit elements from p; those from `left` on are zero.  W: elements
// of a load that pointers and row lengths allow.
template <int W>
__device__ __forceinline__ u32x4 load8(const uint16_t *p, int64_t left) {
    u32x4 v = {0u, 0u, 0u, 0u};
    if constexpr (W == 8) {
        if (left > 0) v = *reinterpret_cast<const u32x4 *>(p);
    } else if constexpr (W == 4) {
        if (left > 0) {
            const uint2 a = *reinterpret_cast<const uint2 *>(p);
            v[0] = a.x;
            v[1] = a.y;
        }
        if (left > 4) {
            const uint2 b = *reinterpret_cast<const uint2 *>(p + 4);
            v[2] = b.x;
            v[3] = b.y;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (e < left) v[e >> 1] |= (uint32_t)p[e] << (16 * (e & 1));
    }
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

// The waves' sums of 16 RB ranks by 16 tokens, joined in LDS; those of the
// tokens in `own` are written as this slice's partial.
template <int RB>
__device__ __forceinline__ void down_join(const AdapterArgs &g, const f32x4 acc[RB], int64_t m0, uint32_t own, int rank0,
                                          int slice, float (*lds)[16 * RB][17]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, lg = lane >> 4;
    __syncthreads();  // the last use of lds is over
#pragma unroll
    for (int r = 0; r < RB; r++)
#pragma unroll
        for (int i = 0; i < 4; i++) lds[wave][16 * r + 4 * lg + i][col] = acc[r][i];
    __syncthreads();
    for (int x = threadIdx.x; x < 256 * RB; x += 64 * kDown) {
        const int j = x % (16 * RB), t = x / (16 * RB);
        if (!(own >> t & 1) || rank0 + j >= g.a.rank) continue;
        float sum = lds[0][j][t];
#pragma unroll
        for (int w = 1; w < kDown; w++) sum += lds[w][j][t];
        g.low[((int64_t)slice * g.a.tokens + m0 + t) * g.a.rank + rank0 + j] = sum;
    }
}

// The steps of this wave: [s, end) of this slice.
__device__ __forceinline__ void down_steps(const AdapterArgs &g, int slice, int *s, int *end) {
    const int wave = threadIdx.x >> 6, share = (g.steps + kDown - 1) / kDown;
    const int all = (int)((g.a.in_features + 31) / 32), last = (slice + 1) * g.steps;
    *s = slice * g.steps + wave * share;
    *end = *s + share;
    if (*end > last) *end = last;
    if (*end > all) *end = all;
}

// 16 tokens from m0, every adapter among them.
template <int RB, bool BF, int W>
__device__ __forceinline__ void down16(const AdapterArgs &g, int64_t m0, int rank0, int slice, float (*lds)[16 * RB][17]) {
    constexpr int U = RB == 1 ? 4 : 2;  // steps whose loads are in flight together
    const int lane = threadIdx.x & 63, col = lane & 15, lg = lane >> 4;
    const int64_t K = g.a.in_features;
    const int mine = adapter_of(g, m0 + col);
    const uint32_t own = (uint32_t)__ballot(mine >= 0) & 0xffffu;
    const int64_t m = m0 + col < g.a.tokens ? m0 + col : g.a.tokens - 1;
    const uint16_t *xp = (const uint16_t *)g.a.x + m * g.a.x_stride + 8 * lg;
    const uint16_t *ap = (const uint16_t *)g.a.a + 8 * lg;
    f32x4 acc[RB];
#pragma unroll
    for (int r = 0; r < RB; r++) acc[r] = f32x4{0.f, 0.f, 0.f, 0.f};
    int s, end;
    down_steps(g, slice, &s, &end);
    for (; s < end; s += U) {
        u32x4 xv[U];
        int64_t left[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            left[u] = s + u < end ? K - (int64_t)(s + u) * 32 - 8 * lg : 0;
            xv[u] = load8<W>(xp + (int64_t)(s + u) * 32, left[u]);
        }
        for (uint32_t todo = own; todo;) {
            const int id = __builtin_amdgcn_readlane(mine, __ffs(todo) - 1);
            const uint32_t same = (uint32_t)__ballot(mine == id) & 0xffffu;
            todo &= ~same;
            f32x4 t[RB];
            u32x4 av[U][RB];
#pragma unroll
            for (int r = 0; r < RB; r++) {
                const int j = rank0 + 16 * r + col;
                const uint16_t *p = ap + ((int64_t)id * g.a.rank + (j < g.a.rank ? j : g.a.rank - 1)) * K;
#pragma unroll
                for (int u = 0; u < U; u++) av[u][r] = load8<W>(p + (int64_t)(s + u) * 32, left[u]);
                t[r] = acc[r];
            }
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int r = 0; r < RB; r++) t[r] = mfma<BF>(av[u][r], xv[u], t[r]);
            if (same >> col & 1) {
#pragma unroll
                for (int r = 0; r < RB; r++) acc[r] = t[r];
            }
        }
    }
    down_join<RB>(g, acc, m0, own, rank0, slice, lds);
}

// 64 tokens from m0, the tokens `own` of one adapter: an adapter's loads
// serve four products.
template <int RB, bool BF, int W>
__device__ __forceinline__ void down64(const AdapterArgs &g, int64_t m0, int id, uint64_t own, int rank0, int slice,
                                       float (*lds)[16 * RB][17]) {
    constexpr int U = RB == 1 ? 2 : 1;
    const int lane = threadIdx.x & 63, col = lane & 15, lg = lane >> 4;
    const int64_t K = g.a.in_features;
    const uint16_t *xp[4], *ap[RB];
#pragma unroll
    for (int c = 0; c < 4; c++) {
        const int64_t m = m0 + 16 * c + col;
        xp[c] = (const uint16_t *)g.a.x + (m < g.a.tokens ? m : g.a.tokens - 1) * g.a.x_stride + 8 * lg;
    }
#pragma unroll
    for (int r = 0; r < RB; r++) {
        const int j = rank0 + 16 * r + col;
        ap[r] = (const uint16_t *)g.a.a + ((int64_t)id * g.a.rank + (j < g.a.rank ? j : g.a.rank - 1)) * K + 8 * lg;
    }
    f32x4 acc[4][RB];
#pragma unroll
    for (int c = 0; c < 4; c++)
#pragma unroll
        for (int r = 0; r < RB; r++) acc[c][r] = f32x4{0.f, 0.f, 0.f, 0.f};
    int s, end;
    down_steps(g, slice, &s, &end);
    u32x4 xv[2][U][4], av[2][U][RB];
    auto load = [&](int at, u32x4 x[U][4], u32x4 a[U][RB]) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int64_t k = (int64_t)(at + u) * 32, left = at + u < end ? K - k - 8 * lg : 0;
#pragma unroll
            for (int r = 0; r < RB; r++) a[u][r] = load8<W>(ap[r] + k, left);
#pragma unroll
            for (int c = 0; c < 4; c++) x[u][c] = load8<W>(xp[c] + k, left);
        }
    };
    auto product = [&](const u32x4 x[U][4], const u32x4 a[U][RB]) {
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int r = 0; r < RB; r++)
#pragma unroll
                for (int c = 0; c < 4; c++) acc[c][r] = mfma<BF>(a[u][r], x[u][c], acc[c][r]);
    };
    load(s, xv[0], av[0]);
    for (; s < end; s += 2 * U) {  // (the next step's loads ahead of this one's products)
        load(s + U, xv[1], av[1]);
        product(xv[0], av[0]);
        load(s + 2 * U, xv[0], av[0]);
        product(xv[1], av[1]);
    }
#pragma unroll
    for (int c = 0; c < 4; c++) {
        const uint32_t o = (uint32_t)(own >> (16 * c)) & 0xffffu;
        if (o) down_join<RB>(g, acc[c], m0 + 16 * c, o, rank0, slice, lds);
    }
}

template <int RB, bool BF, int W, bool FEW>
__global__ __launch_bounds__(64 * kDown) void adapter_down_kernel(AdapterArgs g) {
    __shared__ float lds[kDown][16 * RB][17];
    int tile, slice;
    place_of(g, g.slices, &tile, &slice);
    if (tile >= g.tiles) return;
    if constexpr (FEW) {
        for (int r = 0; r < g.a.rank; r += 16 * RB) down16<RB, BF, W>(g, (int64_t)tile * 16, r, slice, lds);
    } else {
        const int64_t m0 = (int64_t)tile * kTokens;
        const int mine = adapter_of(g, m0 + (threadIdx.x & 63));
        const uint64_t all = __ballot(mine >= 0);
        int distinct = 0;
        for (uint64_t todo = all; todo; distinct++)
            todo &= ~__ballot(mine == __builtin_amdgcn_readlane(mine, __ffsll((unsigned long long)todo) - 1));
        for (int r = 0; r < g.a.rank; r += 16 * RB) {
            if (distinct > kShared) {
                for (int c = 0; c < 4 && m0 + 16 * c < g.a.tokens; c++) down16<RB, BF, W>(g, m0 + 16 * c, r, slice, lds);
                continue;
            }
            for (uint64_t todo = all; todo;) {
                const int id = __builtin_amdgcn_readlane(mine, __ffsll((unsigned long long)todo) - 1);
                const uint64_t same = __ballot(mine == id);
                todo &= ~same;
                down64<RB, BF, W>(g, m0, id, same, r, slice, lds);
            }
        }
    }
}

// -------------------------------------------------------------------------- up

// The sum of slices first, first + step, .. of low[m, j0 .. j0 + 7].
__device__ __forceinline__ void low_sum(const AdapterArgs &g, int64_t m, int j0, int first, int step, f32x4 v[2]) {
    const int r = g.a.rank;
    constexpr int U = 4;  // slices whose loads are in flight together
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
// a lane), FP32 in `dst`, become their two parts there; returns the power of
// two that the lane's token was scaled by.
template <bool BF>
__device__ __forceinline__ int low_parts(int kks, u32x4 *dst) {
    const int lane = threadIdx.x & 63;
    int sh = 0;
    if constexpr (!BF) {
        float top = 0.f;
        for (int x = 0; x < 2 * kks; x++) {
            const f32x4 v = __builtin_bit_cast(f32x4, dst[x * 64 + lane]);
            top = fmaxf(fmaxf(top, fmaxf(fabsf(v[0]), fabsf(v[1]))), fmaxf(fabsf(v[2]), fabsf(v[3])));
        }
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        // the largest to 2^14: its parts are normal numbers and so are those
        // of values 2^-17 of it
        if (top > 0.f && top < __builtin_inff()) sh = 15 - __builtin_amdgcn_frexp_expf(top);
    }
    for (int kk = 0; kk < kks; kk++) {
        const f32x4 v[2] = {__builtin_bit_cast(f32x4, dst[(2 * kk) * 64 + lane]),
                            __builtin_bit_cast(f32x4, dst[(2 * kk + 1) * 64 + lane])};
        u32x4 h, l;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            uint32_t hw = 0, lw = 0;
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const float x0 = v[i >> 1][(2 * i + e) & 3], x = BF ? x0 : __builtin_amdgcn_ldexpf(x0, sh);
                const uint16_t hb = store16<BF>(x);
                const float hv = load16<BF>(hb);
                // (an infinity has no rest)
                const uint16_t lb = fabsf(hv) < __builtin_inff() ? store16<BF>(x - hv) : 0;
                hw |= (uint32_t)hb << (16 * e);
                lw |= (uint32_t)lb << (16 * e);
            }
            h[i] = hw;
            l[i] = lw;
        }
        dst[(2 * kk) * 64 + lane] = h;
        dst[(2 * kk + 1) * 64 + lane] = l;
    }
    return sh;
}

// One unit of kUp outputs from n0 of 16 tokens from m0: the adapters of the
// tokens in `own`, every `step`-th of them from `first`.  Product t's row
// 4 a + i is output 16 a + 4 t + i of the unit, so a lane (rows 4 lg + i of
// all four) holds outputs 16 lg .. 16 lg + 15 of its token.  Tokens without
// an adapter are copied with the first ones.
template <bool BF, int W, bool YV>
__device__ __forceinline__ void up_unit(const AdapterArgs &g, int64_t m0, int mine, int sh, int64_t n0, int kks,
                                        const u32x4 *parts, int first, int step) {
    const int lane = threadIdx.x & 63, col = lane & 15, lg = lane >> 4;
    const int64_t N = g.a.out_features, n = n0 + 16 * lg;
    const uint32_t own = (uint32_t)__ballot(mine >= 0) & 0xffffu;
    // this call's tokens
    uint32_t taken = first == 0 ? ~own & 0xffffu : 0;
    int k = 0;
    for (uint32_t todo = own; todo; k++) {
        const uint32_t same = (uint32_t)__ballot(mine == __builtin_amdgcn_readlane(mine, __ffs(todo) - 1)) & 0xffffu;
        todo &= ~same;
        if (k % step == first) taken |= same;
    }
    const bool on = (taken >> col & 1) && m0 + col < g.a.tokens;
    if (!__any(on)) return;
    const int64_t m = m0 + col < g.a.tokens ? m0 + col : g.a.tokens - 1;
    const uint16_t *y = (const uint16_t *)g.a.y + m * g.a.y_stride + n;
    u32x4 yv[2];
    uint16_t ys[16];
    if constexpr (YV) {
        yv[0] = load8<8>(y, on ? N - n : 0);
        yv[1] = load8<8>(y + 8, on ? N - n - 8 : 0);
    } else {
#pragma unroll
        for (int e = 0; e < 16; e++) ys[e] = on && n + e < N ? y[e] : 0;
    }
    f32x4 acc[4];
#pragma unroll
    for (int t = 0; t < 4; t++) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    int64_t row[4];
#pragma unroll
    for (int t = 0; t < 4; t++) {
        const int64_t at = n0 + 16 * (col >> 2) + 4 * t + (col & 3);
        row[t] = (at < N ? at : N - 1) * g.a.rank + 8 * lg;
    }
    for (uint32_t todo = own & taken; todo;) {
        const int id = __builtin_amdgcn_readlane(mine, __ffs(todo) - 1);
        const uint32_t same = (uint32_t)__ballot(mine == id) & 0xffffu;
        todo &= ~same;
        const uint16_t *b = (const uint16_t *)g.a.b + (int64_t)id * N * g.a.rank;
        f32x4 d[4];
#pragma unroll
        for (int t = 0; t < 4; t++) d[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
        for (int kk = 0; kk < kks; kk++) {
            u32x4 bv[4];
#pragma unroll
            for (int t = 0; t < 4; t++) bv[t] = load8<W>(b + row[t] + 32 * kk, g.a.rank - 32 * kk - 8 * lg);
            const u32x4 h = parts[(2 * kk) * 64 + lane], l = parts[(2 * kk + 1) * 64 + lane];
#pragma unroll
            for (int t = 0; t < 4; t++) d[t] = mfma<BF>(bv[t], h, d[t]);
#pragma unroll
            for (int t = 0; t < 4; t++) d[t] = mfma<BF>(bv[t], l, d[t]);
        }
        if (same >> col & 1) {
#pragma unroll
            for (int t = 0; t < 4; t++) acc[t] = d[t];
        }
    }
    if (!on) return;
    uint16_t *out = (uint16_t *)g.a.out + m * g.a.out_stride + n;
    uint16_t r[16];
#pragma unroll
    for (int e = 0; e < 16; e++) {
        const uint16_t v = YV ? (uint16_t)(yv[e >> 3][(e & 7) >> 1] >> (16 * (e & 1))) : ys[e];
        const float d = acc[e >> 2][e & 3];
        r[e] = mine >= 0 ? store16<BF>(load16<BF>(v) + (BF ? d : __builtin_amdgcn_ldexpf(d, -sh))) : v;
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

// FEW: 16 tokens a workgroup, one unit, its waves split the slices to add
// and then the adapters; else 64 tokens, a wave 16 of them to add and then a
// unit for all of them.
template <bool BF, int W, bool YV, bool FEW>
__global__ __launch_bounds__(256) void adapter_up_kernel(AdapterArgs g) {
    extern __shared__ u32x4 parts[];  // [4][kks][2][64]
    __shared__ int shifts[kTokens];
    int tile, block;
    place_of(g, g.blocks, &tile, &block);
    if (tile >= g.tiles) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, lg = lane >> 4;
    const int kks = (g.a.rank + 31) / 32, each = kks * 128;
    const int64_t m0 = (int64_t)tile * (FEW ? 16 : kTokens), mw = FEW ? m0 : m0 + 16 * wave;
    int mine = adapter_of(g, mw + col);
    const float scale = mine >= 0 ? (g.a.scales ? g.a.scales[mine] : 1.f) : 0.f;
    if (__any(mine >= 0)) {
        for (int kk = 0; kk < kks; kk++) {
            f32x4 v[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
            if (mine >= 0) low_sum(g, mw + col, 32 * kk + 8 * lg, FEW ? wave : 0, FEW ? 4 : 1, v);
            if (!FEW) {
                v[0] *= scale;
                v[1] *= scale;
            }
            parts[wave * each + (2 * kk) * 64 + lane] = __builtin_bit_cast(u32x4, v[0]);
            parts[wave * each + (2 * kk + 1) * 64 + lane] = __builtin_bit_cast(u32x4, v[1]);
        }
        if constexpr (FEW) {
            __syncthreads();
            // (x, the rank words, dealt over the waves)
            for (int x = wave; x < 2 * kks; x += 4) {
                f32x4 v = __builtin_bit_cast(f32x4, parts[x * 64 + lane]);
#pragma unroll
                for (int w = 1; w < 4; w++) v += __builtin_bit_cast(f32x4, parts[w * each + x * 64 + lane]);
                parts[x * 64 + lane] = __builtin_bit_cast(u32x4, v * scale);
            }
            __syncthreads();
        }
        if (!FEW || wave == 0) {
            const int sh = low_parts<BF>(kks, parts + (FEW ? 0 : wave * each));
            if (lane < 16) shifts[(FEW ? 0 : 16 * wave) + lane] = sh;
        }
    }
    __syncthreads();
    if constexpr (FEW) {
        up_unit<BF, W, YV>(g, m0, mine, shifts[col], (int64_t)block * kUp, kks, parts, wave, 4);
    } else {
        const int64_t n0 = ((int64_t)block * 4 + wave) * kUp;
        if (n0 >= g.a.out_features) return;
        for (int c = 0; c < 4 && m0 + 16 * c < g.a.tokens; c++) {
            mine = adapter_of(g, m0 + 16 * c + col);
            up_unit<BF, W, YV>(g, m0 + 16 * c, mine, shifts[16 * c + col], n0, kks, parts + c * each, 0, 1);
        }
    }
}

// The launches' shapes: from the sizes alone, as the adapter numbers are on
// the device.
AdapterArgs adapter_args(const orth_hip_adapter_t &a, int cus) {
    AdapterArgs g;
    g.a = a;
    g.low = nullptr;
    const int wide = a.tokens <= kFew ? 16 : kTokens;
    g.tiles = (int)((a.tokens + wide - 1) / wide);
    const int64_t steps = (a.in_features + 31) / 32;
    // down: slices for a workgroup of eight waves a CU
    int64_t slices = (int64_t)cus / g.tiles;
    if (slices > (steps + kDown - 1) / kDown) slices = (steps + kDown - 1) / kDown;
    if (slices > 16) slices = 16;
    if (slices < 1) slices = 1;
    g.steps = (int)((steps + slices - 1) / slices);
    g.slices = (int)((steps + g.steps - 1) / g.steps);
    const int64_t span = a.tokens <= kFew ? kUp : 4 * kUp;
    g.blocks = (int)((a.out_features + span - 1) / span);
    g.affine = g.tiles >= 8;
    return g;
}

bool multiple(const void *p, int64_t stride, int n) { return reinterpret_cast<uintptr_t>(p) % (2 * n) == 0 && stride % n == 0; }

template <int RB, bool BF>
void down_launch(const AdapterArgs &g, unsigned groups, hipStream_t stream) {
    const bool few = g.a.tokens <= kFew;
    if (multiple(g.a.x, g.a.x_stride, 8) && multiple(g.a.a, g.a.in_features, 8)) {
        if (few) adapter_down_kernel<RB, BF, 8, true><<<groups, 64 * kDown, 0, stream>>>(g);
        else adapter_down_kernel<RB, BF, 8, false><<<groups, 64 * kDown, 0, stream>>>(g);
    } else {
        if (few) adapter_down_kernel<RB, BF, 1, true><<<groups, 64 * kDown, 0, stream>>>(g);
        else adapter_down_kernel<RB, BF, 1, false><<<groups, 64 * kDown, 0, stream>>>(g);
    }
}

template <bool BF, int W>
hipError_t up_launch(const AdapterArgs &g, unsigned groups, hipStream_t stream) {
    const size_t lds = (size_t)4 * ((g.a.rank + 31) / 32) * 128 * sizeof(u32x4);
    const bool yv = g.a.out_features % 8 == 0 && multiple(g.a.y, g.a.y_stride, 8) && multiple(g.a.out, g.a.out_stride, 8);
    auto go = [&](auto kernel) -> hipError_t {
        if (lds > 48 * 1024) {
            hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
            if (e != hipSuccess) return e;
        }
        kernel<<<groups, 256, lds, stream>>>(g);
        return hipGetLastError();
    };
    if (g.a.tokens <= kFew) return yv ? go(adapter_up_kernel<BF, W, true, true>) : go(adapter_up_kernel<BF, W, false, true>);
    return yv ? go(adapter_up_kernel<BF, W, true, false>) : go(adapter_up_kernel<BF, W, false, false>);
}

template <bool BF>
hipError_t adapter_launch(const AdapterArgs &g, hipStream_t stream) {
    const int64_t padded = g.affine ? ((int64_t)g.tiles + 7) / 8 * 8 : g.tiles;
    if (padded * (g.blocks > g.slices ? g.blocks : g.slices) > INT32_MAX) return hipErrorInvalidConfiguration;
    const unsigned down = (unsigned)(padded * g.slices), up = (unsigned)(padded * g.blocks);
    if (g.a.count > 0) {
        if (g.a.rank <= 16) down_launch<1, BF>(g, down, stream);
        else if (g.a.rank <= 32) down_launch<2, BF>(g, down, stream);
        else down_launch<4, BF>(g, down, stream);
        hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    if (multiple(g.a.b, g.a.rank, 8)) return up_launch<BF, 8>(g, up, stream);
    if (multiple(g.a.b, g.a.rank, 4)) return up_launch<BF, 4>(g, up, stream);
    return up_launch<BF, 1>(g, up, stream);
}

}  // namespace

int64_t adapter_workspace_bytes(const orth_hip_adapter_t &a, int cus) {
    return a.count > 0 ? (int64_t)adapter_args(a, cus).slices * a.tokens * a.rank * 4 : 0;
}

hipError_t launch_adapter_add(const orth_hip_adapter_t &a, int cus, void *work, hipStream_t stream) {
    AdapterArgs g = adapter_args(a, cus);
    g.low = static_cast<float *>(work);
    return a.dtype == ORTH_DT_BF16 ? adapter_launch<true>(g, stream) : adapter_launch<false>(g, stream);
}

}  // namespace orth
