// bq_attn_dev.hpp -- device helpers of the attention kernels for a few rows
// (bq_attn.hip, bq_attn_shared.hip).
#pragma once
#include "bq_kv.hpp"

namespace bq {

constexpr int kWaves = 4;          // per workgroup
constexpr int kRound = 512;        // 32-token steps whose pages are staged at once
constexpr float kNone = -3.402823466e38f;  // the running maximum before any token
constexpr float kLazy = 8.f;       // it moves when a score passes it by more (log2)

// 32-token steps that a tile's rows see: [b, b + ns) for the sinks, then
// [lo_step, lo_step + n - ns)
struct Steps {
    int b, lo, lo_step, ns, n;
};

// four int8 codes -> bf16 (exact)
BQ_DEV u32x2 codes_bf16(uint32_t w) {
    const float a = (float)(int8_t)w, b = (float)(int8_t)(w >> 8), c = (float)(int8_t)(w >> 16), d = (float)((int32_t)w >> 24);
    auto hi2 = [](float x, float y) {  // the high halves: small integers are exact in bf16
        return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, y), __builtin_bit_cast(uint32_t, x), 0x07060302u);
    };
    return u32x2{hi2(a, b), hi2(c, d)};
}
BQ_DEV bf16x8 codes8(uint32_t lo, uint32_t hi) {
    const u32x2 a = codes_bf16(lo), b = codes_bf16(hi);
    return __builtin_bit_cast(bf16x8, u32x4{a[0], a[1], b[0], b[1]});
}
BQ_DEV f16x8 codes8h(uint32_t lo, uint32_t hi) {
    f16x2 v[4];
    codes_f16(lo, v[0], v[1]);
    codes_f16(hi, v[2], v[3]);
    return f16x8{v[0][0], v[0][1], v[1][0], v[1][1], v[2][0], v[2][1], v[3][0], v[3][1]};
}
BQ_DEV f32x4 mfma16h(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
BQ_DEV f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// largest and sum over the four lane groups that share lane & 15
BQ_DEV float groups_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
BQ_DEV float groups_sum(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

}  // namespace bq
