// Low-rank adapters of many requests beside a shared projection.
#include "orth_serve.h"

namespace orth {

namespace {

// The low-rank products: a wave per (token, rank).
template <bool BF>
__global__ __launch_bounds__(256) void adapter_down_kernel(orth_hip_adapter_t a, float *low) {
    const int64_t t = blockIdx.x;
    const int j = blockIdx.y * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int64_t i = a.adapters[t];
    if (j >= a.rank || i < 0 || i >= a.count) return;
    const uint16_t *x = (const uint16_t *)a.x + t * a.x_stride;
    const uint16_t *w = (const uint16_t *)a.a + (i * a.rank + j) * a.in_features;
    float s = 0.f;
    for (int64_t k = lane; k < a.in_features; k += 64) s += load16<BF>(x[k]) * load16<BF>(w[k]);
    s = wave_sum(s);
    if (lane == 0) low[t * a.rank + j] = s;
}

// An output per thread.
template <bool BF>
__global__ __launch_bounds__(256) void adapter_up_kernel(orth_hip_adapter_t a, const float *low) {
    const int64_t t = blockIdx.x, n = (int64_t)blockIdx.y * 256 + threadIdx.x;
    if (n >= a.out_features) return;
    const int64_t i = a.adapters[t];
    const uint16_t y = ((const uint16_t *)a.y)[t * a.y_stride + n];
    uint16_t *out = (uint16_t *)a.out + t * a.out_stride + n;
    if (i < 0 || i >= a.count) {
        *out = y;
        return;
    }
    const uint16_t *w = (const uint16_t *)a.b + (i * a.out_features + n) * a.rank;
    float s = 0.f;
    for (int j = 0; j < a.rank; j++) s += low[t * a.rank + j] * load16<BF>(w[j]);
    *out = store16<BF>(load16<BF>(y) + (a.scales ? a.scales[i] : 1.f) * s);
}

}  // namespace

int64_t adapter_workspace_bytes(const orth_hip_adapter_t &a, int) { return a.tokens * a.rank * 4; }

hipError_t launch_adapter_add(const orth_hip_adapter_t &a, int, void *work, hipStream_t stream) {
    const dim3 down((unsigned)a.tokens, (unsigned)((a.rank + 3) / 4));
    const dim3 up((unsigned)a.tokens, (unsigned)((a.out_features + 255) / 256));
    float *low = static_cast<float *>(work);
    if (a.dtype == ORTH_DT_BF16) {
        adapter_down_kernel<true><<<down, 256, 0, stream>>>(a, low);
        adapter_up_kernel<true><<<up, 256, 0, stream>>>(a, low);
    } else {
        adapter_down_kernel<false><<<down, 256, 0, stream>>>(a, low);
        adapter_up_kernel<false><<<up, 256, 0, stream>>>(a, low);
    }
    return hipGetLastError();
}

}  // namespace orth
