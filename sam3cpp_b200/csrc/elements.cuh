// Loads and stores of runs of consecutive elements (fp32, fp16 or bf16 in
// memory, fp32 in registers).
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

// Eight consecutive elements at a 16-byte boundary.
S3T_DEV void load8(const float* p, float (&v)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <typename T>
S3T_DEV void load8(const T* p, float (&v)[8]) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = unpack2(w[i], T());
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
S3T_DEV void store8(float* p, const float (&v)[8]) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
template <typename T>
S3T_DEV void store8(T* p, const float (&v)[8]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack2(v[0], v[1], T()), pack2(v[2], v[3], T()), pack2(v[4], v[5], T()),
                                              pack2(v[6], v[7], T()));
}

}  // namespace s3t
