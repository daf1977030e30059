// attention_tiles.h -- the 32 x 32 x 16 bf16 MFMA and accumulator helpers of the attention kernels (attention.hip, attention_varlen.hip).
#pragma once
#include "dpipe_common.h"

namespace dpipe_tiles {
using namespace dpipe;

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

__device__ __forceinline__ f32x16 mfma16(bf16x8_t a, bf16x8_t b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_mfma, a), __builtin_bit_cast(bf16x8_mfma, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int e = 0; e < 16; ++e) z[e] = 0.f;
    return z;
}
__device__ __forceinline__ bf16x8_t zero_frag() {
    bf16x8_t z;
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] = 0;
    return z;
}
// 8 consecutive accumulator entries (e0 .. e0+7) -> bf16 MFMA operand
__device__ __forceinline__ bf16x8_t pack_frag(const f32x16& s, int e0) {
    uint4 u;
    u.x = pack_bf16x2(s[e0 + 0], s[e0 + 1]); u.y = pack_bf16x2(s[e0 + 2], s[e0 + 3]);
    u.z = pack_bf16x2(s[e0 + 4], s[e0 + 5]); u.w = pack_bf16x2(s[e0 + 6], s[e0 + 7]);
    return __builtin_bit_cast(bf16x8_t, u);
}

}  // namespace dpipe_tiles
