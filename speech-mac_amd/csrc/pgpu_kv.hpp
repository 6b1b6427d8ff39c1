// What the attentions and the writes of the quantised KV caches (pgpu_kv8.hip,
// pgpu_kv4.hip) share: loads, the fixed-point numbers that the int8 matrix
// instruction takes, fp16 terms, reductions without LDS.
#pragma once

#include "pgpu_common.hpp"

namespace pgpu {

// Rows that a call reads or writes once, past the caches.
__device__ inline float4 once_load(const float *p) {
    const f32x4 v = __builtin_nontemporal_load((const f32x4 *)p);
    return make_float4(v.x, v.y, v.z, v.w);
}
__device__ inline void once_store(float *p, float4 v) {
    __builtin_nontemporal_store(f32x4{v.x, v.y, v.z, v.w}, (f32x4 *)p);
}

// Memory that no work-group of a launch writes, at an address that is the same
// for a wave: read through the scalar cache.
template <typename T>
__device__ inline T uniform_load(const T *p) {
    return *(const __attribute__((address_space(4))) T *)p;
}

// Byte b of four numbers -> a word; sel = b | (4 + b) << 8.
__device__ inline uint32_t pick4(uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t sel) {
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, sel),
                                 __builtin_amdgcn_perm(b, a, sel), 0x05040100u);
}
// LDS between the lanes of one wave: nothing is moved across it.
__device__ inline void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr float kNone = -3.0e38f;  // the maximum of no scores

__device__ inline float row16_max(float v) {
    // v_max of the lane 8, 4, 2, 1 apart within each row of 16.
    v = fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(
                     0, __builtin_bit_cast(int, v), 0x128, 0xf, 0xf, false)));
    v = fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(
                     0, __builtin_bit_cast(int, v), 0x124, 0xf, 0xf, false)));
    v = fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(
                     0, __builtin_bit_cast(int, v), 0x4E, 0xf, 0xf, false)));
    v = fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(
                     0, __builtin_bit_cast(int, v), 0xB1, 0xf, 0xf, false)));
    return v;
}

// Fixed point below `top` (>= 0, the largest magnitude): the power of two that
// takes it above 2^30 / 1.004 and not above 127 * (2^24 + 2^16 + 2^8 + 1), the
// largest sum of four signed bytes (0x11000 carries a significand above 1.992
// into the exponent). Below 2^-96 the step stays at 2^-126.
__device__ inline int fix_exponent(float top) {
    return min(126, 157 - (int)((fbits(top) + 0x11000u) >> 23));
}
__device__ inline float power_of_2(int e) { return bitsf((uint32_t)(127 + e) << 23); }
// The four bytes of the number, each signed: n = sum of byte t * 256^t.
__device__ inline uint32_t fix_bytes(float x, float mul) {
    return ((uint32_t)(int)rintf(x * mul) + 0x80808080u) ^ 0x80808080u;
}
// Which byte of a number stands in row t of its query: the highest in row 0.
__device__ inline uint32_t row_byte(int t) { return 3u - t; }
// At most 128 products of 2^14 to a byte: two bytes' sums together stay below 2^30.
__device__ inline float fix_sum(i32x4 c) {
    return fmaf((float)(c.x * 256 + c.y), 65536.0f, (float)(c.z * 256 + c.w));
}

__device__ inline float lane_value(float v, int lane) {
    return bitsf((uint32_t)__builtin_amdgcn_readlane((int)fbits(v), lane));
}

template <int P>
__device__ inline uint32_t quad_lane(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, P * 0x55, 0xf, 0xf, false);
}

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

// x, y -> two fp16 terms, both truncated: hi + lo has 22 bits of them. The
// remainder is one v_fma_mix_f32, which reads an fp16 half as it stands.
__device__ inline void split_pair(float x, float y, f16x2 &hi, f16x2 &lo) {
    const auto h = __builtin_amdgcn_cvt_pkrtz(x, y);
    const uint32_t u = __builtin_bit_cast(uint32_t, h);
    float rx, ry;
    asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel_hi:[1,0,0]" : "=v"(rx) : "v"(u), "v"(x));
    asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]"
        : "=v"(ry) : "v"(u), "v"(y));
    hi = __builtin_bit_cast(f16x2, h);
    lo = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_pkrtz(rx, ry));
}

// Pairs of terms -> an operand of 8.
__device__ inline f16x8 join_pairs(f16x2 a, f16x2 b, f16x2 c, f16x2 d) {
    const i32x4 x = {__builtin_bit_cast(int, a), __builtin_bit_cast(int, b),
                     __builtin_bit_cast(int, c), __builtin_bit_cast(int, d)};
    return __builtin_bit_cast(f16x8, x);
}

// The largest of three; NaN does not count.
__device__ inline float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// The largest over lanes 16 and 32 apart, without the quieting of NaN that fmaxf adds
// to each operand (8187 rows over the 8-bit cache 164.9 us, 166.8 with it).
__device__ inline float quarters_max(float v) {
    auto x = __builtin_amdgcn_permlane16_swap(fbits(v), fbits(v), false, false);
    v = max3(__builtin_bit_cast(float, (uint32_t)x[0]), __builtin_bit_cast(float, (uint32_t)x[1]),
             __builtin_bit_cast(float, (uint32_t)x[1]));
    x = __builtin_amdgcn_permlane32_swap(fbits(v), fbits(v), false, false);
    return max3(__builtin_bit_cast(float, (uint32_t)x[0]), __builtin_bit_cast(float, (uint32_t)x[1]),
                __builtin_bit_cast(float, (uint32_t)x[1]));
}

}  // namespace pgpu
