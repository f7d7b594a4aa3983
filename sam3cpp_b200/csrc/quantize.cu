// 8-bit block quantization: rows of fp32, fp16 or bf16 to e4m3 with one fp32
// scale per 128 columns of a row (activations) or per 128 x 128 block
// (weights).  The arithmetic is in fp8.cuh.
//
// Bound by HBM: each element is read once and one byte of it written.  Sixteen
// lanes hold the 128 columns of a group, eight consecutive elements each, so
// the group's maximum is four shuffles away and nothing is read twice.  82944 x
// 4736 fp16: 183 us, 6.5 TB/s (469 us with a division per lane and group and
// the maxima in fp32: bound by its instructions; 208 us at five CTAs an SM).
#include "elements.cuh"
#include "fp8.cuh"
#include "kernels.h"

namespace s3t {

namespace {

constexpr int kThreads = 256;
constexpr int kGroupLanes = 16;     // lanes of a 128-column group
constexpr int kRowsPerWarp = 4;     // activation rows a warp has in flight
constexpr int kRowsPerCta = kRowsPerWarp * kThreads / 32;

// A lane's eight elements of a group as they lie in memory.
template <typename T>
struct Raw {
    uint32_t w[2 * sizeof(T)];
};

// Elements 2 i and 2 i + 1.
template <typename T>
S3T_DEV float2 elements(const Raw<T>& v, int i) {
    if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(v.w[2 * i]), __uint_as_float(v.w[2 * i + 1]));
    else return unpack2(v.w[i], T());
}

// Columns of element i of a lane's eight: consecutive where the rows are
// 16-byte aligned (VEC), else 16 apart so that a load of the half warp still
// covers consecutive addresses.
template <bool VEC>
S3T_DEV int lane_col(int lane16, int i) {
    return VEC ? lane16 * 8 + i : lane16 + 16 * i;
}

template <typename T, bool VEC>
S3T_DEV void load_group(const T* row, int64_t c0, int64_t cols, int lane16, Raw<T>& v) {
    if (VEC && c0 + lane16 * 8 + 8 <= cols) {
        const uint4* p = reinterpret_cast<const uint4*>(row + c0 + lane16 * 8);
#pragma unroll
        for (int i = 0; i < int(sizeof(T)) / 2; ++i) {
            const uint4 u = p[i];
            v.w[4 * i] = u.x; v.w[4 * i + 1] = u.y; v.w[4 * i + 2] = u.z; v.w[4 * i + 3] = u.w;
        }
        return;
    }
    T e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t c = c0 + lane_col<VEC>(lane16, i);
        e[i] = c < cols ? row[c] : from_float<T>(0.f);
    }
    memcpy(v.w, e, sizeof(e));
}

template <typename T>
S3T_DEV void no_group(Raw<T>& v) {
#pragma unroll
    for (int i = 0; i < int(2 * sizeof(T)); ++i) v.w[i] = 0;
}

template <typename T, bool VEC>
S3T_DEV void store_group(uint8_t* row, int64_t c0, int64_t cols, int lane16, const Raw<T>& v, float inv) {
    float2 f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __fmul2_rn(elements(v, i), make_float2(inv, inv));
    const uint32_t lo = pack_e4m3x4(f[0].x, f[0].y, f[1].x, f[1].y), hi = pack_e4m3x4(f[2].x, f[2].y, f[3].x, f[3].y);
    if (VEC && c0 + lane16 * 8 + 8 <= cols) {
        *reinterpret_cast<uint2*>(row + c0 + lane16 * 8) = make_uint2(lo, hi);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t c = c0 + lane_col<VEC>(lane16, i);
        if (c < cols) row[c] = uint8_t((i < 4 ? lo : hi) >> (8 * (i & 3)));
    }
}

// Largest magnitude of a lane's eight elements as bits of T: the bits of 16-bit
// types order like their magnitudes too, and two compare at once.
template <typename T>
S3T_DEV uint32_t peak_bits(const Raw<T>& v) {
    if constexpr (sizeof(T) == 4) {
        uint32_t m = v.w[0] & 0x7fffffffu;
#pragma unroll
        for (int i = 1; i < 8; ++i) m = max(m, v.w[i] & 0x7fffffffu);
        return m;
    } else {
        uint32_t m = v.w[0] & 0x7fff7fffu;
#pragma unroll
        for (int i = 1; i < 4; ++i) m = __vmaxu2(m, v.w[i] & 0x7fff7fffu);
        return max(m & 0xffffu, m >> 16);
    }
}

template <typename T>
S3T_DEV uint32_t float_bits(uint32_t peak) {
    if constexpr (sizeof(T) == 4) return peak;
    else return __float_as_uint(unpack2(peak, T()).x);
}

// A warp takes two groups (256 columns) of four consecutive rows.  The maxima
// of two 16-bit rows share a word in the reduction, and each lane does one of
// the eight divisions (a / 448 and 448 / a of four rows) of its half warp.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 4 ? 4 : 8) quantize_rows_kernel(const QuantizeArgs a, uint32_t col_blocks) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rb = blockIdx.x / col_blocks, cb = blockIdx.x - rb * col_blocks;
    const int64_t r0 = int64_t(rb) * kRowsPerCta + warp * kRowsPerWarp;
    const int lane16 = lane % kGroupLanes;
    const int64_t g = int64_t(cb) * 2 + lane / kGroupLanes;
    const int64_t c0 = g * kScaleBlock;
    const T* x = static_cast<const T*>(a.x) + r0 * a.x_stride;
    Raw<T> v[kRowsPerWarp];
    // Rows and columns past the end read nothing and count as zeros.
#pragma unroll
    for (int r = 0; r < kRowsPerWarp; ++r) {
        if (r0 + r < a.rows) load_group<T, VEC>(x + r * a.x_stride, c0, a.cols, lane16, v[r]);
        else no_group(v[r]);
    }
    uint32_t peak[kRowsPerWarp];
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int r = 0; r < kRowsPerWarp; ++r) peak[r] = peak_bits(v[r]);
#pragma unroll
        for (int o = kGroupLanes / 2; o; o >>= 1)
#pragma unroll
            for (int r = 0; r < kRowsPerWarp; ++r) peak[r] = max(peak[r], __shfl_xor_sync(0xffffffffu, peak[r], o));
    } else {
        uint32_t two[kRowsPerWarp / 2];
#pragma unroll
        for (int r = 0; r < kRowsPerWarp / 2; ++r) two[r] = peak_bits(v[2 * r]) | (peak_bits(v[2 * r + 1]) << 16);
#pragma unroll
        for (int o = kGroupLanes / 2; o; o >>= 1)
#pragma unroll
            for (int r = 0; r < kRowsPerWarp / 2; ++r) two[r] = __vmaxu2(two[r], __shfl_xor_sync(0xffffffffu, two[r], o));
#pragma unroll
        for (int r = 0; r < kRowsPerWarp; ++r) peak[r] = r & 1 ? two[r / 2] >> 16 : two[r / 2] & 0xffffu;
    }
    static_assert(kRowsPerWarp == 4, "lane pattern of the divisions");
    const int row = lane16 & 3;
    const uint32_t mine = row & 2 ? (row & 1 ? peak[3] : peak[2]) : (row & 1 ? peak[1] : peak[0]);
    const float top = __uint_as_float(max(float_bits<T>(mine), kAmaxFloorBits));
    const bool inverse = lane16 & 4;
    const float quotient = __fdiv_rn(inverse ? kE4M3Max : top, inverse ? top : kE4M3Max);
#pragma unroll
    for (int r = 0; r < kRowsPerWarp; ++r) {
        const float inv = __shfl_sync(0xffffffffu, quotient, 4 + r, kGroupLanes);
        if (r0 + r < a.rows && c0 < a.cols) store_group<T, VEC>(a.q + (r0 + r) * a.q_stride, c0, a.cols, lane16, v[r], inv);
    }
    if (lane16 < 4 && r0 + row < a.rows && c0 < a.cols) a.scale[g * a.scale_stride + r0 + row] = quotient;
}

// A CTA takes one 128 x 128 block: 16 rows at a time, eight times, all in registers.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) quantize_blocks_kernel(const QuantizeArgs a, uint32_t col_blocks) {
    constexpr int kPasses = kScaleBlock / (kThreads / kGroupLanes);
    __shared__ uint32_t warp_max[kThreads / 32];
    const uint32_t rb = blockIdx.x / col_blocks, cb = blockIdx.x - rb * col_blocks;
    const int lane16 = threadIdx.x % kGroupLanes;
    const int64_t r0 = int64_t(rb) * kScaleBlock + threadIdx.x / kGroupLanes;
    const int64_t c0 = int64_t(cb) * kScaleBlock;
    const T* x = static_cast<const T*>(a.x);
    Raw<T> v[kPasses];
    uint32_t m = 0;
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
        const int64_t r = r0 + p * (kThreads / kGroupLanes);
        if (r < a.rows) load_group<T, VEC>(x + r * a.x_stride, c0, a.cols, lane16, v[p]);
        else no_group(v[p]);
    }
#pragma unroll
    for (int p = 0; p < kPasses; ++p) m = max(m, peak_bits(v[p]));
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) m = max(m, warp_max[w]);
    const BlockScale s = block_scale(float_bits<T>(m));
    if (threadIdx.x == 0) a.scale[int64_t(cb) * a.scale_stride + rb] = s.scale;
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
        const int64_t r = r0 + p * (kThreads / kGroupLanes);
        if (r < a.rows) store_group<T, VEC>(a.q + r * a.q_stride, c0, a.cols, lane16, v[p], s.inv);
    }
}

template <typename T, bool VEC>
cudaError_t launch(const QuantizeArgs& a, cudaStream_t stream) {
    const bool blocks = a.block_rows != 1;
    const int64_t cb = (a.cols + (blocks ? kScaleBlock : 2 * kScaleBlock) - 1) / (blocks ? kScaleBlock : 2 * kScaleBlock);
    const int64_t rb = (a.rows + (blocks ? kScaleBlock : kRowsPerCta) - 1) / (blocks ? kScaleBlock : kRowsPerCta);
    if (rb > 0x7fffffff / cb) return cudaErrorInvalidValue;
    if (blocks)
        quantize_blocks_kernel<T, VEC><<<uint32_t(rb * cb), kThreads, 0, stream>>>(a, uint32_t(cb));
    else
        quantize_rows_kernel<T, VEC><<<uint32_t(rb * cb), kThreads, 0, stream>>>(a, uint32_t(cb));
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_quantize_fp8(const QuantizeArgs& a, cudaStream_t stream) {
    switch (a.kind) {
        case kF32: return a.vec ? launch<float, true>(a, stream) : launch<float, false>(a, stream);
        case kF16: return a.vec ? launch<__half, true>(a, stream) : launch<__half, false>(a, stream);
        case kBF16:
            return a.vec ? launch<__nv_bfloat16, true>(a, stream) : launch<__nv_bfloat16, false>(a, stream);
    }
    return cudaErrorInvalidValue;
}

}  // namespace s3t
