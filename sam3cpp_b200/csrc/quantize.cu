// 8-bit block quantization: rows of fp32, fp16 or bf16 to e4m3 with one fp32
// scale per 128 columns of a row (activations) or per 128 x 128 block
// (weights).  The arithmetic is in fp8.cuh.
//
// Bound by HBM: each element is read once and one byte of it written.  Sixteen
// lanes hold the 128 columns of a group, eight consecutive elements each, so
// the group's maximum is four shuffles away and nothing is read twice.  82944 x
// 4736 fp16: 172 us, 6.9 TB/s (469 us with a division per lane and group and
// the maxima in fp32: bound by its instructions; 189 us with four rows a warp
// and every access guarded, 220 us once the 1 kW cap lowers the clocks).
#include "elements.cuh"
#include "fp8.cuh"
#include "kernels.h"

namespace s3t {

namespace {

constexpr int kThreads = 256;
constexpr int kGroupLanes = 16;     // lanes of a 128-column group
// Activation rows a warp has in flight: the 16 lanes of a half warp do the two
// divisions of eight 16-bit rows; four fp32 rows are as many registers.
template <typename T>
constexpr int kRowsPerWarp = sizeof(T) == 4 ? 4 : 8;
template <typename T>
constexpr int kRowsPerCta = kRowsPerWarp<T> * kThreads / 32;

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

template <typename T>
S3T_DEV void load_raw(const T* p, Raw<T>& v) {
#pragma unroll
    for (int i = 0; i < int(sizeof(T)) / 2; ++i) {
        const uint4 u = reinterpret_cast<const uint4*>(p)[i];
        v.w[4 * i] = u.x; v.w[4 * i + 1] = u.y; v.w[4 * i + 2] = u.z; v.w[4 * i + 3] = u.w;
    }
}

// Eight consecutive elements at any address, from the whole 16-byte units that
// hold them (a unit with one of the row's bytes lies in the row's allocation).
template <typename T>
S3T_DEV void load_shifted(const T* p, Raw<T>& v) {
    constexpr int WORDS = 2 * int(sizeof(T));
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    const uint32_t shift = uint32_t(at) & 15;
    const uint4* units = reinterpret_cast<const uint4*>(at - shift);
    uint32_t c[WORDS + 4];
#pragma unroll
    for (int i = 0; i <= WORDS / 4; ++i) {
        const uint4 u = i < WORDS / 4 || shift ? units[i] : make_uint4(0, 0, 0, 0);
        c[4 * i] = u.x; c[4 * i + 1] = u.y; c[4 * i + 2] = u.z; c[4 * i + 3] = u.w;
    }
    if (shift & 8) {
#pragma unroll
        for (int i = 0; i + 2 < WORDS + 4; ++i) c[i] = c[i + 2];
    }
    if (shift & 4) {
#pragma unroll
        for (int i = 0; i + 1 < WORDS + 4; ++i) c[i] = c[i + 1];
    }
#pragma unroll
    for (int i = 0; i < WORDS; ++i) v.w[i] = sizeof(T) < 4 && (shift & 2) ? __funnelshift_r(c[i], c[i + 1], 16) : c[i];
}

template <typename T, bool VEC>
S3T_DEV void load_group(const T* row, int64_t c0, int64_t cols, int lane16, Raw<T>& v) {
    if (VEC && c0 + lane16 * 8 + 8 <= cols) {
        load_raw(row + c0 + lane16 * 8, v);
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

template <typename T>
S3T_DEV uint2 codes(const Raw<T>& v, float inv) {
    float2 f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __fmul2_rn(elements(v, i), make_float2(inv, inv));
    return make_uint2(pack_e4m3x4(f[0].x, f[0].y, f[1].x, f[1].y), pack_e4m3x4(f[2].x, f[2].y, f[3].x, f[3].y));
}

template <typename T, bool VEC>
S3T_DEV void store_group(uint8_t* row, int64_t c0, int64_t cols, int lane16, const Raw<T>& v, float inv) {
    const uint2 c = codes(v, inv);
    if (VEC && c0 + lane16 * 8 + 8 <= cols) {
        *reinterpret_cast<uint2*>(row + c0 + lane16 * 8) = c;
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t at = c0 + lane_col<VEC>(lane16, i);
        if (at < cols) row[at] = uint8_t((i < 4 ? c.x : c.y) >> (8 * (i & 3)));
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

// A warp takes two groups (256 columns) of kRowsPerWarp consecutive rows.  The
// maxima of two 16-bit rows share a word in the reduction, and each lane does
// one of the divisions (a / 448 and 448 / a of each row) of its half warp.
// INSIDE: all of the warp's rows and columns are there (nearly every warp of a
// large matrix), so no access is guarded: at 6.5 TB/s the kernel issues on four
// of five clocks, and its instructions are what the 1 kW cap slows down.
template <typename T, bool VEC, bool INSIDE>
S3T_DEV void quantize_rows(const QuantizeArgs& a, int64_t r0, int64_t g, int lane16) {
    constexpr int ROWS = kRowsPerWarp<T>;
    const int64_t c0 = g * kScaleBlock;
    Raw<T> v[ROWS];
    {
        const T* x = static_cast<const T*>(a.x) + r0 * a.x_stride;
        if constexpr (INSIDE) x += c0 + lane16 * 8;
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            // Rows and columns past the end read nothing and count as zeros.
            if constexpr (INSIDE && VEC) load_raw(x, v[r]);
            else if constexpr (INSIDE) load_shifted(x, v[r]);
            else if (r0 + r < a.rows) load_group<T, VEC>(x, c0, a.cols, lane16, v[r]);
            else no_group(v[r]);
            x += a.x_stride;
        }
    }
    // Bits of row k's largest magnitude: a word each, or two rows a word.
    constexpr int WORDS = sizeof(T) == 4 ? ROWS : ROWS / 2;
    uint32_t peak[WORDS];
#pragma unroll
    for (int k = 0; k < WORDS; ++k) {
        if constexpr (sizeof(T) == 4) peak[k] = peak_bits(v[k]);
        else peak[k] = peak_bits(v[2 * k]) | (peak_bits(v[2 * k + 1]) << 16);
    }
#pragma unroll
    for (int o = kGroupLanes / 2; o; o >>= 1)
#pragma unroll
        for (int k = 0; k < WORDS; ++k) {
            const uint32_t other = __shfl_xor_sync(0xffffffffu, peak[k], o);
            peak[k] = sizeof(T) == 4 ? max(peak[k], other) : __vmaxu2(peak[k], other);
        }
    const int row = lane16 & (ROWS - 1);
    uint32_t mine = peak[0];
#pragma unroll
    for (int k = 1; k < WORDS; ++k)
        if (row / (ROWS / WORDS) == k) mine = peak[k];
    if constexpr (sizeof(T) != 4) mine = row & 1 ? mine >> 16 : mine & 0xffffu;
    const float top = __uint_as_float(max(float_bits<T>(mine), kAmaxFloorBits));
    const bool inverse = lane16 & ROWS;
    const float quotient = __fdiv_rn(inverse ? kE4M3Max : top, inverse ? top : kE4M3Max);
    uint8_t* q = a.q + r0 * a.q_stride;
    if constexpr (INSIDE) q += c0 + lane16 * 8;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        const float inv = __shfl_sync(0xffffffffu, quotient, ROWS + r, kGroupLanes);
        if constexpr (INSIDE) *reinterpret_cast<uint2*>(q) = codes(v[r], inv);
        else if (r0 + r < a.rows && c0 < a.cols) store_group<T, VEC>(q, c0, a.cols, lane16, v[r], inv);
        q += a.q_stride;
    }
    if (lane16 < ROWS && (INSIDE || (r0 + row < a.rows && c0 < a.cols))) a.scale[g * a.scale_stride + r0 + row] = quotient;
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads, 4) quantize_rows_kernel(const QuantizeArgs a, uint32_t col_blocks) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rb = blockIdx.x / col_blocks, cb = blockIdx.x - rb * col_blocks;
    const int64_t r0 = int64_t(rb) * kRowsPerCta<T> + warp * kRowsPerWarp<T>;
    const int64_t g = int64_t(cb) * 2 + lane / kGroupLanes;
    if (r0 + kRowsPerWarp<T> <= a.rows && int64_t(cb + 1) * 2 * kScaleBlock <= a.cols)
        quantize_rows<T, VEC, true>(a, r0, g, lane % kGroupLanes);
    else
        quantize_rows<T, VEC, false>(a, r0, g, lane % kGroupLanes);
}

// Threads of a CTA that takes one 128 x 128 block, all of it in registers: 512
// for fp32 (20000 x 4097: 65 us, with 256 76 us; aligned rows the same), 256 for
// 16 bits (16384 x 16384: 117 us, 6.9 TB/s, with 512 143 us; every access
// guarded 128 us).
template <typename T>
constexpr int kBlockThreads = sizeof(T) == 4 ? 512 : 256;

// INSIDE: the whole block is there, so no access is guarded.
template <typename T, bool VEC, bool INSIDE>
S3T_DEV void quantize_block(const QuantizeArgs& a, uint32_t rb, uint32_t cb, uint32_t* warp_max) {
    constexpr int kRows = kBlockThreads<T> / kGroupLanes, kPasses = kScaleBlock / kRows;   // rows at a time
    const int lane16 = threadIdx.x % kGroupLanes;
    const int64_t r0 = int64_t(rb) * kScaleBlock + threadIdx.x / kGroupLanes;
    const int64_t c0 = int64_t(cb) * kScaleBlock;
    const bool columns = INSIDE || c0 + kScaleBlock <= a.cols;   // all columns are there
    Raw<T> v[kPasses];
    {
        const T* x = static_cast<const T*>(a.x) + r0 * a.x_stride;
        const int64_t step = kRows * a.x_stride;
#pragma unroll
        for (int p = 0; p < kPasses; ++p, x += step) {
            if (!INSIDE && r0 + p * kRows >= a.rows) no_group(v[p]);
            else if (INSIDE && VEC) load_raw(x + c0 + lane16 * 8, v[p]);
            else if (!VEC && columns) load_shifted(x + c0 + lane16 * 8, v[p]);
            else load_group<T, VEC>(x, c0, a.cols, lane16, v[p]);
        }
    }
    uint32_t m = 0;
#pragma unroll
    for (int p = 0; p < kPasses; ++p) m = max(m, peak_bits(v[p]));
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kBlockThreads<T> / 32; ++w) m = max(m, warp_max[w]);
    const BlockScale s = block_scale(float_bits<T>(m));
    if (threadIdx.x == 0) a.scale[int64_t(cb) * a.scale_stride + rb] = s.scale;
    uint8_t* q = a.q + r0 * a.q_stride;
    const int64_t step = kRows * a.q_stride;
#pragma unroll
    for (int p = 0; p < kPasses; ++p, q += step) {
        if (INSIDE) *reinterpret_cast<uint2*>(q + c0 + lane16 * 8) = codes(v[p], s.inv);
        else if (r0 + p * kRows >= a.rows) continue;
        else if (!VEC && columns) store_group<T, true>(q, c0, a.cols, lane16, v[p], s.inv);
        else store_group<T, VEC>(q, c0, a.cols, lane16, v[p], s.inv);
    }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kBlockThreads<T>) quantize_blocks_kernel(const QuantizeArgs a, uint32_t col_blocks) {
    __shared__ uint32_t warp_max[kBlockThreads<T> / 32];
    const uint32_t rb = blockIdx.x / col_blocks, cb = blockIdx.x - rb * col_blocks;
    if (int64_t(rb + 1) * kScaleBlock <= a.rows && int64_t(cb + 1) * kScaleBlock <= a.cols)
        quantize_block<T, VEC, true>(a, rb, cb, warp_max);
    else
        quantize_block<T, VEC, false>(a, rb, cb, warp_max);
}

template <typename T, bool VEC>
cudaError_t launch(const QuantizeArgs& a, cudaStream_t stream) {
    const bool blocks = a.block_rows != 1;
    const int64_t cb = (a.cols + (blocks ? kScaleBlock : 2 * kScaleBlock) - 1) / (blocks ? kScaleBlock : 2 * kScaleBlock);
    const int64_t rb = (a.rows + (blocks ? kScaleBlock : kRowsPerCta<T>) - 1) / (blocks ? kScaleBlock : kRowsPerCta<T>);
    if (rb > 0x7fffffff / cb) return cudaErrorInvalidValue;
    if (blocks)
        return launch_on(quantize_blocks_kernel<T, VEC>, uint32_t(rb * cb), kBlockThreads<T>, 0, stream, a, uint32_t(cb));
    return launch_on(quantize_rows_kernel<T, VEC>, uint32_t(rb * cb), kThreads, 0, stream, a, uint32_t(cb));
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
