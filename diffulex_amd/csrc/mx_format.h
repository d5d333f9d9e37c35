// Microscaled (MX) KV-cache elements: blocks of 32 consecutive elements of a head row share one power-of-two scale.
//
//   code value c, scale byte b:  element = c * 2^(b - 127)          (b == 255: the block is NaN)
//   E4M3 codes (one byte, largest magnitude M = 448) or E2M1 codes (four bits, M = 6; element 2 i in the low half of byte i).
//   Writing a block with largest magnitude A: b - 127 = the smallest e with A <= M 2^e (at least -127), codes = the multiples
//   of the code's grid nearest to x 2^-e, ties to even, among those whose element is below 2^128 (MxLast).  A block that holds
//   an infinity or NaN gets b = 255 and codes 0.
//
// With a power of two as the scale, x 2^-e is exact in fp32 (the codes round once, from the exact quotient), and every
// code * scale that a finite block is written with, 4 or 2 significant bits, is exactly a finite bf16 (a subnormal one too: x is a
// multiple of 2^-133, and so is what it is rounded to): widening loses nothing and the matrix instructions see what the cache
// holds.  Codes and scales from elsewhere may stand for elements that bf16 has not: those below its smallest subnormal are rounded,
// those from 2^128 on are infinities.  gfx950 converts two codes and applies the scale in one instruction
// (v_cvt_scalef32_pk_bf16_fp8 / _fp4), whose scale operand is read as its exponent field: the byte shifted to bit 23 is the
// E8M0 scale for all 256 bytes (byte 0 is 2^-127, byte 255 NaN) -- compared with 64-bit arithmetic for every byte and every code.
#pragma once

#include "dfx_common.h"

namespace dfx {

constexpr int kMxBlock = 32;

// Bytes of a head row's codes.
DFX_HD constexpr int mx_row_bytes(bool e2m1, int head_dim) { return e2m1 ? head_dim / 2 : head_dim; }

// Scale byte of a block whose largest magnitude has the bf16 bits `a` (sign cleared; the largest of the bits is the largest
// of the magnitudes, and an infinity or NaN is larger still).  A = 1.m * 2^(E - 127): one binade lower than the largest code's if
// the mantissa does not exceed the largest code's (448 = 1.75 * 2^8, 6 = 1.5 * 2^2).
template <bool E2M1>
DFX_HD uint32_t mx_scale_byte(uint32_t a) {
    const int e = static_cast<int>(a >> 7) - (E2M1 ? 2 : 8) + ((a & 0x7fu) > (E2M1 ? 0x40u : 0x60u) ? 1 : 0);
    return a >= 0x7f80u ? 255u : static_cast<uint32_t>(e < 0 ? 0 : e);
}

// Largest magnitude bits of 8 bf16.
DFX_D uint32_t abs_max8(u32x4 w) {
    uint32_t m = 0;
    const uint32_t d[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        m = max(m, d[i] & 0x7fffu);
        m = max(m, (d[i] >> 16) & 0x7fffu);
    }
    return m;
}

// Maximum over the lane's pair / quad of lanes (all of them active).
DFX_D uint32_t max_pair(uint32_t v) {
    return max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0xB1, 0xf, 0xf, true)));  // lanes 1 0 3 2
}
DFX_D uint32_t max_quad(uint32_t v) {
    v = max_pair(v);
    return max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x4E, 0xf, 0xf, true)));  // lanes 2 3 0 1
}

// The scale byte of blocks whose largest magnitudes round up to a code that stands for 2^128 (255 to 256 with 2^120, 3.98 to 4 with 2^126),
// and the last code whose element is a finite bf16.  (Blocks of smaller maxima have smaller bytes, and M 2^e below 2^128.)
template <bool E2M1>
struct MxLast {
    static constexpr uint32_t kByte = E2M1 ? 253 : 247;
    static constexpr float kCode = E2M1 ? 3.0f : 240.0f;
};

// 2^-e as a float for scale byte b (0 for the byte of a non-finite block: its codes are written as zeros).
DFX_D float mx_inverse_scale(uint32_t b) { return b == 255u ? 0.0f : __builtin_bit_cast(float, (254u - b) << 23); }

template <bool E2M1>
DFX_D void mx_scaled8(u32x4 w, uint32_t scale_byte, float (&y)[8]) {
    const float s = mx_inverse_scale(scale_byte);
    const bool bad = scale_byte == 255u;
    const uint32_t d[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float lo = __builtin_bit_cast(float, d[i] << 16) * s, hi = __builtin_bit_cast(float, d[i] & 0xffff0000u) * s;
        y[2 * i] = bad ? 0.0f : lo;  // (an infinity times 0 would be a NaN)
        y[2 * i + 1] = bad ? 0.0f : hi;
    }
    if (scale_byte == MxLast<E2M1>::kByte) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = __builtin_amdgcn_fmed3f(y[i], -MxLast<E2M1>::kCode, MxLast<E2M1>::kCode);
    }
}

// 8 bf16 -> 8 E4M3 codes.  v_cvt_pk_fp8_f32 rounds to nearest even (compared with a library cast for all bf16 up to 448).
DFX_D u32x2 mx_codes8_e4m3(u32x4 w, uint32_t scale_byte) {
    float y[8];
    mx_scaled8<false>(w, scale_byte, y);
    u32x2 r;
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    r.x = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], v, true));
    v = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], 0, false);
    r.y = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], v, true));
    return r;
}

// 8 bf16 -> 8 E2M1 codes (a dword).
DFX_D uint32_t mx_codes8_e2m1(u32x4 w, uint32_t scale_byte) {
    float y[8];
    mx_scaled8<true>(w, scale_byte, y);
    uint32_t r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, y[0], y[1], 1.0f, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, y[2], y[3], 1.0f, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, y[4], y[5], 1.0f, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, y[6], y[7], 1.0f, 3);
}

// Writes 8 elements' codes of a head row (dst: the row's first byte; c: element / 8) and, from the lane that `leads` its block, the
// block's scale byte.  `a`: the block's largest magnitude bits.
template <bool E2M1>
DFX_D void mx_put8(u32x4 w, uint32_t a, uint8_t* codes, uint8_t* scales, int c, bool leads) {
    const uint32_t b = mx_scale_byte<E2M1>(a);
    if constexpr (E2M1) *reinterpret_cast<uint32_t*>(codes + c * 4) = mx_codes8_e2m1(w, b);
    else *reinterpret_cast<u32x2*>(codes + c * 8) = mx_codes8_e4m3(w, b);
    if (leads) scales[c >> 2] = static_cast<uint8_t>(b);
}

DFX_D float mx_scale_operand(uint32_t scale_byte) { return __builtin_bit_cast(float, scale_byte << 23); }

// 8 E4M3 codes -> 8 bf16
DFX_D u32x4 mx_widen8_e4m3(u32x2 w, float scale) {
    return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.x, scale, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.x, scale, true)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.y, scale, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.y, scale, true))};
}

// 8 E2M1 codes -> 8 bf16
DFX_D u32x4 mx_widen8_e2m1(uint32_t w, float scale) {
    return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3))};
}

}  // namespace dfx
