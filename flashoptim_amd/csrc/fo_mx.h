// The MXFP4 format's device pieces: a group's scale and its values' codes (the format itself is described in fo_mx.hip).
#pragma once

#include "fo_device.h"

namespace fo {

constexpr int kBlock = 128;    // values that rows are filled up to
constexpr int kMxGroup = 32;

// 8-bit scale of a group from the bits of its largest magnitude as fp32.  Infinities and NaNs have the largest bits.
__device__ __forceinline__ u32 scale_byte(u32 magnitude_bits) {
    const u32 e = magnitude_bits >> 23;
    return e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
}
// The scale as the converting instructions take it; they look at the exponent alone.
__device__ __forceinline__ float scale_value(u32 byte) { return as_f32(byte << 23); }

__device__ __forceinline__ u32 largest_of_quad(u32 x) {
    const u32 a = (u32)__builtin_amdgcn_mov_dpp((int)x, 0xb1, 0xf, 0xf, true);   // lanes 1 0 3 2
    x = x > a ? x : a;
    const u32 b = (u32)__builtin_amdgcn_mov_dpp((int)x, 0x4e, 0xf, 0xf, true);   // lanes 2 3 0 1
    return x > b ? x : b;
}

// Two values next to each other, as they are stored.
template <int DT> struct Pair;
template <> struct Pair<DT_BF16> {
    u32 v;
    __device__ __forceinline__ u32 magnitude() const {   // the larger, as fp32 bits
        const u32 a = (v & 0x7fffu) << 16, b = v & 0x7fff0000u;
        return a > b ? a : b;
    }
    template <int BYTE> __device__ __forceinline__ u32 encode(u32 into, float scale) const {
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(into, __builtin_bit_cast(bf16x2, v), scale, BYTE);
    }
};
template <> struct Pair<DT_F16> {
    u32 v;
    __device__ __forceinline__ u32 magnitude() const {
        const u32 a = v & 0x7fffu, b = (v >> 16) & 0x7fffu, m = a > b ? a : b;
        return as_u32((float)__builtin_bit_cast(_Float16, (uint16_t)m));
    }
    template <int BYTE> __device__ __forceinline__ u32 encode(u32 into, float scale) const {
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(into, __builtin_bit_cast(f16x2, v), scale, BYTE);
    }
};
template <> struct Pair<DT_F32> {
    float a, b;
    __device__ __forceinline__ u32 magnitude() const {
        const u32 x = as_u32(a) & 0x7fffffffu, y = as_u32(b) & 0x7fffffffu;
        return x > y ? x : y;
    }
    template <int BYTE> __device__ __forceinline__ u32 encode(u32 into, float scale) const {
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(into, a, b, scale, BYTE);
    }
};

template <int DT> __device__ __forceinline__ u32 encode8(const Pair<DT>* p, float scale) {
    u32 w = p[0].template encode<0>(0u, scale);
    w = p[1].template encode<1>(w, scale);
    w = p[2].template encode<2>(w, scale);
    return p[3].template encode<3>(w, scale);
}

}  // namespace fo
