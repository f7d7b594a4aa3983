// e4m3 values with a scale for each block of 128: the rounding shared by the
// quantization kernel and by the epilogues that write 8-bit operands.
//
// A block with largest magnitude a holds q = e4m3(x * (448 / a)) and the scale
// a / 448, so its largest value sits at e4m3's largest finite one.  Both
// quotients are correctly rounded and the product is one fp32 multiplication:
// the codes are a function of the block's fp32 values alone.  a is at least
// 2^-100, which keeps 448 / a finite and gives an empty block zeros.
// Magnitudes are compared as bit patterns, where NaN > inf > finite: a block
// that holds a NaN or an infinity gets that as its scale and stands for NaN
// as a whole (finite * 0 * inf), instead of hiding it.
#pragma once

#include "ptx.cuh"

namespace s3t {

constexpr float kE4M3Max = 448.f;
constexpr uint32_t kAmaxFloorBits = 0x0D800000u;   // 2^-100

S3T_DEV uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

struct BlockScale {
    float scale, inv;
};

S3T_DEV BlockScale block_scale(uint32_t amax_bits) {
    const float a = __uint_as_float(max(amax_bits, kAmaxFloorBits));
    return {__fdiv_rn(a, kE4M3Max), __fdiv_rn(kE4M3Max, a)};
}

// Two values to e4m3 (round to nearest even, saturating, NaN kept), `lo` in the low byte.
S3T_DEV uint16_t pack_e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

S3T_DEV uint32_t pack_e4m3x4(float a, float b, float c, float d) {
    return uint32_t(pack_e4m3x2(a, b)) | (uint32_t(pack_e4m3x2(c, d)) << 16);
}

}  // namespace s3t
