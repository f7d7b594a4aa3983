// 8-bit block quantization: rows of fp32, fp16 or bf16 to e4m3 with one fp32
// scale per 128 columns of a row (activations) or per 128 x 128 block
// (weights).  The arithmetic is in fp8.cuh.
//
// Bound by HBM: each element is read once and one byte of it written.  Sixteen
// lanes hold the 128 columns of a group, eight consecutive elements each, so
// the group's maximum is four shuffles away and nothing is read twice.
#include "elements.cuh"
#include "fp8.cuh"
#include "kernels.h"

namespace s3t {

namespace {

constexpr int kThreads = 256;
constexpr int kGroupLanes = 16;     // lanes of a 128-column group
constexpr int kRowsPerWarp = 4;     // activation rows a warp has in flight
constexpr int kRowsPerCta = kRowsPerWarp * kThreads / 32;

// Columns of element i of a lane's eight: consecutive where the rows are
// 16-byte aligned (VEC), else 16 apart so that a load of the half warp still
// covers consecutive addresses.
template <bool VEC>
S3T_DEV int lane_col(int lane16, int i) {
    return VEC ? lane16 * 8 + i : lane16 + 16 * i;
}

template <typename T, bool VEC>
S3T_DEV void load_group(const T* row, int64_t c0, int64_t cols, int lane16, float (&v)[8]) {
    if (VEC && c0 + lane16 * 8 + 8 <= cols) {
        load8(row + c0 + lane16 * 8, v);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t c = c0 + lane_col<VEC>(lane16, i);
        v[i] = c < cols ? to_float(row[c]) : 0.f;
    }
}

template <bool VEC>
S3T_DEV void store_group(uint8_t* row, int64_t c0, int64_t cols, int lane16, const float (&v)[8], float inv) {
    const uint32_t lo = pack_e4m3x4(__fmul_rn(v[0], inv), __fmul_rn(v[1], inv), __fmul_rn(v[2], inv),
                                    __fmul_rn(v[3], inv));
    const uint32_t hi = pack_e4m3x4(__fmul_rn(v[4], inv), __fmul_rn(v[5], inv), __fmul_rn(v[6], inv),
                                    __fmul_rn(v[7], inv));
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

S3T_DEV uint32_t amax8(const float (&v)[8]) {
    uint32_t a = abs_bits(v[0]);
#pragma unroll
    for (int i = 1; i < 8; ++i) a = max(a, abs_bits(v[i]));
    return a;
}

// A warp takes two groups (256 columns) of kRowsPerWarp consecutive rows.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const QuantizeArgs a, uint32_t col_blocks) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rb = blockIdx.x / col_blocks, cb = blockIdx.x - rb * col_blocks;
    const int64_t r0 = int64_t(rb) * kRowsPerCta + warp * kRowsPerWarp;
    const int64_t g = int64_t(cb) * 2 + lane / kGroupLanes;
    const int64_t c0 = g * kScaleBlock;
    const int lane16 = lane % kGroupLanes;
    const T* x = static_cast<const T*>(a.x);
    float v[kRowsPerWarp][8];
#pragma unroll
    for (int r = 0; r < kRowsPerWarp; ++r) {
        // Rows and columns past the end read nothing and count as zeros.
        if (r0 + r < a.rows) {
            load_group<T, VEC>(x + (r0 + r) * a.x_stride, c0, a.cols, lane16, v[r]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[r][i] = 0.f;
        }
    }
#pragma unroll
    for (int r = 0; r < kRowsPerWarp; ++r) {
        uint32_t m = amax8(v[r]);
#pragma unroll
        for (int o = kGroupLanes / 2; o; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (r0 + r < a.rows && c0 < a.cols) {
            const BlockScale s = block_scale(m);
            store_group<VEC>(a.q + (r0 + r) * a.q_stride, c0, a.cols, lane16, v[r], s.inv);
            if (lane16 == 0) a.scale[g * a.scale_stride + r0 + r] = s.scale;
        }
    }
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
    float v[kPasses][8];
    uint32_t m = 0;
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
        const int64_t r = r0 + p * (kThreads / kGroupLanes);
        if (r < a.rows) {
            load_group<T, VEC>(x + r * a.x_stride, c0, a.cols, lane16, v[p]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[p][i] = 0.f;
        }
    }
#pragma unroll
    for (int p = 0; p < kPasses; ++p) m = max(m, amax8(v[p]));
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) m = max(m, warp_max[w]);
    const BlockScale s = block_scale(m);
    if (threadIdx.x == 0) a.scale[int64_t(cb) * a.scale_stride + rb] = s.scale;
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
        const int64_t r = r0 + p * (kThreads / kGroupLanes);
        if (r < a.rows) store_group<VEC>(a.q + r * a.q_stride, c0, a.cols, lane16, v[p], s.inv);
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
