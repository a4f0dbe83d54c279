// The INT8-G64 codec of the KV caches on the device (reference contract
// include/ninfer/ops/gqa_attention.h:25-30), eight values per lane.
#pragma once

#include "device_utils.h"

namespace nmi {

// Eight BF16 values per lane, eight consecutive lanes (aligned to eight) per 64-value group:
// s = FP16_RNE(amax / 127), inv = FP32(1 / s), code = clamp(RNE(x * inv), +-127). All eight lanes
// return the group's scale bits; every lane of a group has to be active.
__device__ __forceinline__ i2 quantize_g64(i4 raw, uint16_t& scale_bits) {
    float x[8];
    float amax = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint32_t w = static_cast<uint32_t>(raw[e >> 1]);
        x[e] = bf16_to_f32(static_cast<uint16_t>((e & 1) ? w >> 16 : w & 0xffffu));
        amax = fmaxf(amax, fabsf(x[e]));
    }
    amax = fmaxf(amax, dpp_from<0xB1, 0xf>(amax, 0.0f));  // lane ^ 1
    amax = fmaxf(amax, dpp_from<0x4E, 0xf>(amax, 0.0f));  // lane ^ 2
    amax = fmaxf(amax, dpp_from<0x141, 0xf>(amax, 0.0f)); // the other four of the eight
    scale_bits = f32_to_f16_bits(amax > 0.0f ? amax / 127.0f : 0.0f);
    const float s = f16_bits_to_f32(scale_bits);
    const float inv = s > 0.0f ? 1.0f / s : 0.0f;
    uint32_t code[2] = {0u, 0u};
    if (inv != 0.0f) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float rr = rintf(x[e] * inv);
            rr = fminf(127.0f, fmaxf(-127.0f, rr));
            code[e >> 2] |= (static_cast<uint32_t>(static_cast<int8_t>(rr)) & 0xffu) << (8 * (e & 3));
        }
    }
    return i2{static_cast<int>(code[0]), static_cast<int>(code[1])};
}

} // namespace nmi
