// The serving operators' launchers (page step, cache append, paged
// attention, adapters): arguments already validated by orth_serve.hip.
#pragma once

#include "orth_common.h"

namespace orth {

// The most keys a block table may hold: the attention's key numbers, and
// those its loads run ahead to, are 32-bit.
constexpr int64_t kMostKeys = ((int64_t)1 << 31) - 512;

hipError_t launch_page_step(const orth_hip_step_t &s, hipStream_t stream);

hipError_t launch_cache_append(const orth_hip_cache_t &c, const orth_hip_append_t &a, int cus, hipStream_t stream);

// (`groups`: the counters that a call takes)
int64_t attention_workspace_bytes(const orth_hip_cache_t &c, const orth_hip_attend_t &a, int cus, int64_t *groups);
hipError_t launch_paged_attention(const orth_hip_cache_t &c, const orth_hip_attend_t &a, int cus, void *work, uint32_t *counters,
                                  hipStream_t stream);

int64_t adapter_workspace_bytes(const orth_hip_adapter_t &a, int cus);
hipError_t launch_adapter_add(const orth_hip_adapter_t &a, int cus, void *work, hipStream_t stream);

// Quotients of 0 <= n < 2^31 by d >= 1 without a division: with l =
// ceil(log2 d) and m = ceil(2^(31 + l) / d) <= 2^32 - 1, n * m >> (31 + l) is
// floor(n / d) (the error n * (m d - 2^(31 + l)) < 2^(31 + l) never reaches
// the next quotient).
struct FastDiv {
    uint32_t m, shift, d;
};
inline FastDiv fast_div(uint32_t d) {
    uint32_t l = 0;
    while (((uint64_t)1 << l) < d) l++;
    return {(uint32_t)((((uint64_t)1 << (31 + l)) + d - 1) / d), 31 + l, d};
}
__device__ __forceinline__ uint32_t quotient(uint32_t n, const FastDiv &f) {
    return (uint32_t)(((uint64_t)n * f.m) >> f.shift);
}

// Inclusive sums over the wave: DPP adds within rows of 16 lanes, then each
// row's last sum to the rows behind it.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false);  // row_bcast 15, 31
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false);
    return v;
}

// 16-bit elements as float, and back (round to nearest even), by type.
template <bool BF>
__device__ __forceinline__ float load16(uint16_t b) {
    if constexpr (BF) return bf16_bits_to_f32(b);
    else return (float)__builtin_bit_cast(f16, b);
}
template <bool BF>
__device__ __forceinline__ uint16_t store16(float v) {
    if constexpr (BF) return f32_to_bf16_bits(v);
    else return __builtin_bit_cast(uint16_t, (f16)v);
}

}  // namespace orth
