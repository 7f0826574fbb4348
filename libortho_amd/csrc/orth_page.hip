// Paged cache bookkeeping and filling: page_step (pages, slots and positions
// of a step's tokens from the requests' lengths) and cache_append (rotary
// positions, keys and values into their slots).
#include "orth_serve.h"

namespace orth {

namespace {

// ------------------------------------------------------------------ page step
//
// Two prefix sums over the requests (places, then pages of the requests that
// fit), then one token per thread: its request by binary search in the
// places' starts, its page from the table or the free list.  A request is
// refused for want of places, width or pages by comparing its own prefix
// sum, so no request waits for another's answer; once the pages run out
// every later request that needs one is refused too (the sums run on), so
// the granted ones are a prefix of the list.
//
// Bound by latency: one launch, in which every workgroup repeats the scan of
// all requests (8 bytes each from the L2) instead of waiting for one that
// does it, and then writes a token a thread.  The sums of a scan are 32 bits
// wide where `tokens` allows it (64-bit ones took 2 us more for 16 requests:
// a wave's scan is then a dozen LDS permutes instead of six adds).  Measured:
// 3.3 us in the kernel for 16 requests of one token, 6.3 for 512 with 64
// prompts (13,321 places); 5.6 and 5.8 us a call among others.
constexpr int kStepMost = 1024;  // threads of a workgroup (256 for up to 256 requests)

__device__ __forceinline__ uint32_t scan_in_wave(uint32_t v) { return wave_scan(v); }
__device__ __forceinline__ uint64_t scan_in_wave(uint64_t v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t o = __shfl_up(v, d, 64);
        if (lane >= d) v += o;
    }
    return v;
}

// Inclusive prefix sums over the workgroup; `sums` holds a wave's total each.
template <class Sum>
__device__ __forceinline__ Sum group_scan(Sum v, Sum *sums, Sum *total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    v = scan_in_wave(v);
    __syncthreads();  // the last use of sums is over
    if (lane == 63) sums[wave] = v;
    __syncthreads();
    Sum before = 0, all = 0;
    for (int w = 0; w < waves; w++) {
        before += w < wave ? sums[w] : 0;
        all += sums[w];
    }
    *total = all;
    return v + before;
}

template <class Sum>
__global__ __launch_bounds__(kStepMost) void page_step_kernel(orth_hip_step_t s, FastDiv page) {
    extern __shared__ int32_t lds[];
    int32_t *start = lds, *first = lds + s.requests;  // first place and first page (-1: refused) of each request
    __shared__ Sum sums[kStepMost / 64];
    __shared__ int32_t used, status;
    const int tid = threadIdx.x;
    int64_t head = s.pool[0];
    head = head < 0 ? 0 : (head > s.free_count ? s.free_count : head);
    if (tid == 0) {
        used = (int32_t)head;
        status = 0;
    }
    int64_t places = 0, pages = head;
    for (int64_t r0 = 0; r0 < s.requests; r0 += blockDim.x) {
        const int64_t r = r0 + tid;
        const bool here = r < s.requests;
        const int64_t L = here ? s.lengths[r] : 0, n = here ? s.new_tokens[r] : 0, all = L + n;
        // (a request of more than `tokens` fits nowhere, nor does any after it)
        const int64_t wants = n <= 0 ? 0 : (n <= s.tokens ? n : s.tokens + 1);
        Sum total;
        const int64_t end = places + (int64_t)group_scan<Sum>((Sum)wants, sums, &total);
        const int64_t at = end - wants;
        places += (int64_t)total;
        bool ok = L >= 0 && n >= 0 && all <= INT32_MAX && end <= s.tokens;
        int64_t need = 0;
        if (ok) {
            const int64_t old = quotient((uint32_t)L, page) + (L % s.page_size != 0);
            const int64_t last = quotient((uint32_t)all, page) + (all % s.page_size != 0);
            ok = n == 0 || last <= s.table_width;
            need = ok ? last - old : 0;
        }
        const bool room = ok;
        const int64_t pend = pages + (int64_t)group_scan<Sum>((Sum)need, sums, &total);
        pages += (int64_t)total;
        ok = ok && (need == 0 || pend <= s.free_count);
        if (here) {
            start[r] = (int32_t)(at < s.tokens ? at : s.tokens);
            first[r] = ok ? (int32_t)(need > 0 ? pend - need : 0) : -1;
            if (ok && need > 0) atomicMax(&used, (int32_t)pend);
            if (!ok) atomicOr(&status, room ? ORTH_STEP_NO_PAGES : ORTH_STEP_NO_ROOM);
            if (blockIdx.x == 0) {
                s.query_start[r] = start[r];
                s.lengths_out[r] = (int32_t)(ok ? all : L);
            }
        }
    }
    const int64_t filled = places < s.tokens ? places : s.tokens;
    __syncthreads();
    if (blockIdx.x == 0 && tid == 0) {
        s.query_start[s.requests] = (int32_t)filled;
        s.pool_out[0] = used;
        s.pool_out[1] = status;
    }
    const int64_t t = (int64_t)blockIdx.x * blockDim.x + tid;
    if (t >= s.tokens) return;
    int32_t row = -1, pos = -1;
    int64_t slot = -1;
    if (t < filled) {
        // the last request that starts at or before t (empty ones start where the next does)
        int lo = 0, hi = (int)s.requests - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (start[mid] <= t) lo = mid;
            else hi = mid - 1;
        }
        row = lo;
        if (first[lo] >= 0) {
            const int32_t L = s.lengths[lo];
            pos = L + (int32_t)(t - start[lo]);
            const uint32_t at = quotient((uint32_t)pos, page);
            const uint32_t old = quotient((uint32_t)L, page) + (L % s.page_size != 0);
            const uint32_t in = (uint32_t)pos - at * page.d;
            int32_t *entry = s.block_table + (int64_t)lo * s.table_stride + at;
            int32_t p;
            if (at >= old) {
                p = s.free_pages[first[lo] + (int)(at - old)];
                if (in == 0) *entry = p;  // a new page's first token is one of this step's
            } else {
                p = *entry;
            }
            if (p >= 0) slot = (int64_t)p * s.page_size + in;
        }
    }
    s.rows[t] = row;
    s.positions[t] = pos;
    s.slots[t] = slot;
}

// --------------------------------------------------------------- cache append
//
// Memory-bound: each element is read once and written once.  A head's vector
// is cut into items of 2 V elements: a rotated item is V pairs (V elements of
// each half, or 2 V neighbours when interleaved), the rest are copied.  A
// thread keeps one item and steps through the heads, so its cosines and sines
// (as many bytes as the item's elements read and written) are loaded once for
// all of a token's heads.  Measured: 2,048 tokens of 32 + 8 heads of 128 in
// 9.7 us, 5.3 TB/s; 4 tokens 3.6 us in the kernel (launch and three dependent
// reads: slot, position, cosines).
struct AppendArgs {
    orth_hip_cache_t c;
    orth_hip_append_t a;
    int items, turned;   // items of a head, and how many of them are pairs
    int lanes;           // heads a workgroup takes at a time
    FastDiv per_item, page;
};

template <int V>
struct Vec16 {
    uint16_t e[V];
};

template <int V>
__device__ __forceinline__ Vec16<V> load_vec(const uint16_t *p) {
    Vec16<V> r;
    if constexpr (V == 8) *reinterpret_cast<u32x4 *>(&r) = *reinterpret_cast<const u32x4 *>(p);
    else if constexpr (V == 4) *reinterpret_cast<uint2 *>(&r) = *reinterpret_cast<const uint2 *>(p);
    else r.e[0] = *p;
    return r;
}
template <int V>
__device__ __forceinline__ void store_vec(uint16_t *p, const Vec16<V> &v) {
    if constexpr (V == 8) *reinterpret_cast<u32x4 *>(p) = *reinterpret_cast<const u32x4 *>(&v);
    else if constexpr (V == 4) *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<const uint2 *>(&v);
    else *p = v.e[0];
}

// Where the two vectors of item i start within a head: pairs of the half
// layout lie rot / 2 apart, all others next to each other.
template <int V>
__device__ __forceinline__ void item_at(int i, int turned, int rot, bool interleaved, int *a, int *b) {
    if (i < turned && !interleaved) {
        *a = i * V;
        *b = i * V + rot / 2;
    } else {
        *a = i * 2 * V;
        *b = *a + V;
    }
}

template <int V, bool BF>
__global__ __launch_bounds__(256) void cache_append_kernel(AppendArgs g) {
    const int64_t t = blockIdx.x;
    const int lane_head = (int)quotient(threadIdx.x, g.per_item), item = threadIdx.x - lane_head * g.items;
    if (lane_head >= g.lanes) return;
    const int64_t slot = g.a.slots[t];
    bool write = slot >= 0 && slot < g.c.pages * g.c.page_size;
    bool placed = true;
    const bool pair = item < g.turned;
    float c[V], sn[V];
    if (g.a.cos_sin) {
        const int64_t pos = g.a.positions[t];
        placed = pos >= 0 && pos < g.a.cos_sin_rows;
        write = write && placed;
        if (placed && pair) {
            const float *cs = g.a.cos_sin + pos * g.a.rot + item * V;
#pragma unroll
            for (int j = 0; j < V; j++) {
                c[j] = cs[j];
                sn[j] = cs[j + g.a.rot / 2];
            }
        }
    }
    int64_t pg = 0, in = 0;
    if (write) {
        // (the page of a slot that may pass 2^31: a 64-bit division only there)
        pg = slot <= INT32_MAX ? (int64_t)quotient((uint32_t)slot, g.page) : slot / g.c.page_size;
        in = slot - pg * g.c.page_size;
    }
    int ea, eb;
    item_at<V>(item, g.turned, g.a.rot, g.a.interleaved, &ea, &eb);
    int ca, cb;  // the same of a copied vector
    item_at<V>(item, 0, 0, false, &ca, &cb);
    const int H = g.a.q ? g.a.q_heads : 0, G = g.c.kv_heads, all = H + 2 * G;
    for (int h = blockIdx.y * g.lanes + lane_head; h < all; h += gridDim.y * g.lanes) {
        const uint16_t *src;
        uint16_t *dst;
        bool turn = false;
        if (h < H) {
            src = (const uint16_t *)g.a.q + t * g.a.q_strides[0] + h * g.a.q_strides[1];
            dst = (uint16_t *)g.a.q_out + t * g.a.q_out_strides[0] + h * g.a.q_out_strides[1];
            turn = true;
        } else if (h < H + G) {
            if (!write) continue;
            src = (const uint16_t *)g.a.k + t * g.a.k_strides[0] + (h - H) * g.a.k_strides[1];
            dst = (uint16_t *)g.c.k_cache + pg * g.c.k_strides[0] + in * g.c.k_strides[1] + (h - H) * g.c.k_strides[2];
            turn = true;
        } else {
            if (!write) continue;
            src = (const uint16_t *)g.a.v + t * g.a.v_strides[0] + (h - H - G) * g.a.v_strides[1];
            dst = (uint16_t *)g.c.v_cache + pg * g.c.v_strides[0] + in * g.c.v_strides[1] + (h - H - G) * g.c.v_strides[2];
        }
        const int a = turn ? ea : ca, b = turn ? eb : cb;
        Vec16<V> x = load_vec<V>(src + a), y = load_vec<V>(src + b);
        if (turn && pair && placed) {
            if (!g.a.interleaved) {
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const float u = load16<BF>(x.e[j]), w = load16<BF>(y.e[j]);
                    x.e[j] = store16<BF>(u * c[j] - w * sn[j]);
                    y.e[j] = store16<BF>(w * c[j] + u * sn[j]);
                }
            } else {
                // 2 V neighbours: pair j is elements 2 j and 2 j + 1 of x then y
                uint16_t e[2 * V];
#pragma unroll
                for (int j = 0; j < V; j++) {
                    e[j] = x.e[j];
                    e[V + j] = y.e[j];
                }
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const float u = load16<BF>(e[2 * j]), w = load16<BF>(e[2 * j + 1]);
                    e[2 * j] = store16<BF>(u * c[j] - w * sn[j]);
                    e[2 * j + 1] = store16<BF>(w * c[j] + u * sn[j]);
                }
#pragma unroll
                for (int j = 0; j < V; j++) {
                    x.e[j] = e[j];
                    y.e[j] = e[V + j];
                }
            }
        } else if (!placed) {
            x = Vec16<V>{};
            y = Vec16<V>{};
        }
        store_vec<V>(dst + a, x);
        store_vec<V>(dst + b, y);
    }
}

// The widest vector that pointers, strides and the split of a head allow.
bool append_fits(const orth_hip_cache_t &c, const orth_hip_append_t &a, int V) {
    auto ok = [&](const void *p, const int64_t *s) {
        return reinterpret_cast<uintptr_t>(p) % (2 * V) == 0 && s[0] % V == 0 && s[1] % V == 0;
    };
    const int rot = a.cos_sin ? a.rot : 0;
    return c.head_dim % (2 * V) == 0 && rot % (2 * V) == 0 && ok(a.k, a.k_strides) && ok(a.v, a.v_strides) &&
           (!a.q || (ok(a.q, a.q_strides) && ok(a.q_out, a.q_out_strides)));
}

template <int V>
void append_launch(const AppendArgs &g, dim3 grid, hipStream_t stream) {
    if (g.c.dtype == ORTH_DT_BF16) cache_append_kernel<V, true><<<grid, 256, 0, stream>>>(g);
    else cache_append_kernel<V, false><<<grid, 256, 0, stream>>>(g);
}

}  // namespace

hipError_t launch_page_step(const orth_hip_step_t &s, hipStream_t stream) {
    const int threads = s.requests <= 256 ? 256 : kStepMost;
    const int64_t groups = s.tokens > 0 ? (s.tokens + threads - 1) / threads : 1;
    const size_t lds = (size_t)s.requests * 8;
    const FastDiv page = fast_div((uint32_t)s.page_size);
    auto go = [&](auto kernel) -> hipError_t {
        if (lds > 48 * 1024) {
            hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
            if (e != hipSuccess) return e;
        }
        kernel<<<dim3((unsigned)groups), threads, lds, stream>>>(s, page);
        return hipGetLastError();
    };
    // (1024 requests' places, tokens + 1 at most each, and pages, one more)
    return s.tokens <= (1 << 20) ? go(page_step_kernel<uint32_t>) : go(page_step_kernel<uint64_t>);
}

hipError_t launch_cache_append(const orth_hip_cache_t &c, const orth_hip_append_t &a, int cus, hipStream_t stream) {
    const int V = append_fits(c, a, 8) ? 8 : append_fits(c, a, 4) ? 4 : 1;
    AppendArgs g;
    g.c = c;
    g.a = a;
    if (!a.cos_sin) g.a.rot = 0;
    g.items = c.head_dim / (2 * V);
    g.turned = g.a.rot / (2 * V);
    g.lanes = 256 / g.items;
    g.per_item = fast_div((uint32_t)g.items);
    g.page = fast_div((uint32_t)c.page_size);
    const int heads = (a.q ? a.q_heads : 0) + 2 * c.kv_heads;
    // a workgroup for every head group where tokens alone leave CUs idle,
    // else one a token
    const int parts = (heads + g.lanes - 1) / g.lanes;
    const int y = a.tokens >= 2 * cus ? 1 : parts < 65535 ? parts : 65535;
    // (a launch holds fewer than 2^32 threads along x: one past that runs
    // another number of workgroups, without an error)
    constexpr int64_t kLaunch = 1 << 23;
    for (int64_t t = 0; t < a.tokens; t += kLaunch) {
        const dim3 grid((unsigned)(a.tokens - t < kLaunch ? a.tokens - t : kLaunch), (unsigned)y);
        if (V == 8) append_launch<8>(g, grid, stream);
        else if (V == 4) append_launch<4>(g, grid, stream);
        else append_launch<1>(g, grid, stream);
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

}  // namespace orth
