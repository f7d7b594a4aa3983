// Elements of fp32, fp16 or bf16 in memory, fp32 in registers.
#pragma once

#include "ptx.cuh"

namespace s3t {

S3T_DEV float to_float(float v) { return v; }
S3T_DEV float to_float(__half v) { return __half2float(v); }
S3T_DEV float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
S3T_DEV T from_float(float v);
template <>
S3T_DEV float from_float<float>(float v) { return v; }
template <>
S3T_DEV __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
S3T_DEV __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

S3T_DEV float2 unpack2(uint32_t u, __half) {
    return __half22float2(*reinterpret_cast<const __half2*>(&u));
}
S3T_DEV float2 unpack2(uint32_t u, __nv_bfloat16) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u));
}
S3T_DEV uint32_t pack2(float a, float b, __half) { return pack_half2(a, b); }
S3T_DEV uint32_t pack2(float a, float b, __nv_bfloat16) { return pack_bf162(a, b); }

}  // namespace s3t
