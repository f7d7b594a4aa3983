// The step between two transformer blocks in one pass over the rows:
//   h  = post-norm(y)            (or y itself)
//   x' = resid_scale x + branch_scale channel * act(gate) * h
//   u  = pre-norm(x')            (fp32 / fp16 / bf16, or e4m3 with a scale per 128 columns)
// with RMSNorm, v / sqrt(mean(v^2) + eps) * w, or LayerNorm,
// (v - mean(v)) / sqrt(var(v) + eps) * w + b.  The pre-norm reads the fp32 x',
// before its rounding to the residual's type: the rounding then enters the
// residual stream once and the branch not at all.
//
// Bound by HBM: y, x and the gate are read once, x' and u written once, and a
// row stays in registers between the two norms.  A chunk is 256 columns, eight
// consecutive ones per lane; a row's chunks are dealt out to the warps of a
// CTA.  A LayerNorm warp reduces its own mean and centred square sum M2 and
// the warps' are merged by the pairwise update of Chan, Golub and LeVeque
// (1979), so there is one exchange per norm and no cancellation.
#include "elements.cuh"
#include "fp8.cuh"
#include "kernels.h"

namespace s3t {

namespace {

constexpr int kChunk = 256;
constexpr int kLaneElems = 8;
constexpr int kMaxWarps = 16;          // of a CTA: 16 x 4 chunks hold kNormMaxDim columns

// Columns of a lane's eight elements of a chunk: consecutive (VEC), or 16
// apart within the lane's half-warp group of 128, so that scalar accesses of
// a half warp still cover consecutive addresses.
template <bool VEC>
S3T_DEV int chunk_col(int lane, int i) {
    return VEC ? lane * kLaneElems + i : (lane >> 4) * kScaleBlock + (lane & 15) + 16 * i;
}

template <bool VEC, typename T>
S3T_DEV void load_chunk(const T* p, int c0, int dim, int lane, float (&v)[kLaneElems]) {
    if (VEC) {
        if (c0 + lane * kLaneElems < dim) {
            load8(p + c0 + lane * kLaneElems, v);
            return;
        }
#pragma unroll
        for (int i = 0; i < kLaneElems; ++i) v[i] = 0.f;
        return;
    }
#pragma unroll
    for (int i = 0; i < kLaneElems; ++i) {
        const int c = c0 + chunk_col<VEC>(lane, i);
        v[i] = c < dim ? to_float(p[c]) : 0.f;
    }
}

template <bool VEC, typename T>
S3T_DEV void store_chunk(T* p, int c0, int dim, int lane, const float (&v)[kLaneElems]) {
    if (VEC) {
        if (c0 + lane * kLaneElems < dim) store8(p + c0 + lane * kLaneElems, v);
        return;
    }
#pragma unroll
    for (int i = 0; i < kLaneElems; ++i) {
        const int c = c0 + chunk_col<VEC>(lane, i);
        if (c < dim) p[c] = from_float<T>(v[i]);
    }
}

S3T_DEV float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Mean (0 for RMSNorm) and 1 / sqrt(mean square or variance + eps) of a row
// whose chunks c = warp, warp + WARPS, ... this warp holds; columns past dim
// hold 0.
struct RowStats {
    float mean, rstd;
};

template <int CPW, bool VEC>
S3T_DEV RowStats row_stats(const float (&v)[CPW][kLaneElems], int layer, int dim, float eps, int warp, int warps, int lane,
                           float2* exchange) {
    float n = 0.f, mean = 0.f, m2 = 0.f;
    if (layer) {
        float s = 0.f;
        int held = 0;
#pragma unroll
        for (int j = 0; j < CPW; ++j) {
            const int c0 = (warp + j * warps) * kChunk;
            held += max(0, min(kChunk, dim - c0));
#pragma unroll
            for (int i = 0; i < kLaneElems; ++i) s += v[j][i];
        }
        n = float(held);
        mean = held ? warp_sum(s) / n : 0.f;
    }
#pragma unroll
    for (int j = 0; j < CPW; ++j) {
        const int c0 = (warp + j * warps) * kChunk;
#pragma unroll
        for (int i = 0; i < kLaneElems; ++i) {
            const float d = v[j][i] - mean;
            if (!layer || c0 + chunk_col<VEC>(lane, i) < dim) m2 = fmaf(d, d, m2);
        }
    }
    m2 = warp_sum(m2);
    if (warps > 1) {
        __syncthreads();   // the exchange of the norm before has been read
        if (lane == 0) exchange[warp] = make_float2(mean, m2);
        __syncthreads();
        // Every warp merges all partials in the same order.
        n = mean = m2 = 0.f;
        for (int w = 0; w < warps; ++w) {
            const float2 e = exchange[w];
            if (!layer) {
                m2 += e.y;
                continue;
            }
            int held = 0;
#pragma unroll
            for (int j = 0; j < CPW; ++j) held += max(0, min(kChunk, dim - (w + j * warps) * kChunk));
            const float nb = float(held);
            if (nb == 0.f) continue;
            const float d = e.x - mean, nn = n + nb;
            m2 += e.y + d * d * (n * nb / nn);
            mean += d * (nb / nn);
            n = nn;
        }
    }
    return {mean, rsqrtf(m2 / float(dim) + eps)};
}

template <bool VEC>
S3T_DEV void load_weight(const float* w, float otherwise, int c0, int dim, int lane, float (&v)[kLaneElems]) {
    if (w) {
        load_chunk<VEC>(w, c0, dim, lane, v);
    } else {
#pragma unroll
        for (int i = 0; i < kLaneElems; ++i) v[i] = otherwise;
    }
}

// A CTA takes blockDim.y rows, each by blockDim.x / 32 warps (blockDim.y = 1
// where a row has more than one warp).
template <typename T, typename R, int CPW, bool VEC>
__global__ void __launch_bounds__(32 * kMaxWarps) norm_residual_kernel(const NormResidualArgs a) {
    __shared__ float2 exchange[kMaxWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int64_t row = int64_t(blockIdx.x) * blockDim.y + threadIdx.y;
    if (row >= a.rows) return;   // whole rows: no barrier is shared between rows
    const int dim = a.dim;
    const R* xr = static_cast<const R*>(a.x) + row * a.x_stride;
    float x[CPW][kLaneElems], h[CPW][kLaneElems];
#pragma unroll
    for (int j = 0; j < CPW; ++j) load_chunk<VEC>(xr, (warp + j * warps) * kChunk, dim, lane, x[j]);
    if (a.y) {
        const T* yr = static_cast<const T*>(a.y) + row * a.y_stride;
#pragma unroll
        for (int j = 0; j < CPW; ++j) load_chunk<VEC>(yr, (warp + j * warps) * kChunk, dim, lane, h[j]);
        if (a.post) {
            const RowStats st = row_stats<CPW, VEC>(h, a.layer, dim, a.eps, warp, warps, lane, exchange);
#pragma unroll
            for (int j = 0; j < CPW; ++j) {
                const int c0 = (warp + j * warps) * kChunk;
                float w[kLaneElems], b[kLaneElems];
                load_weight<VEC>(a.post_weight, 1.f, c0, dim, lane, w);
                load_weight<VEC>(a.post_bias, 0.f, c0, dim, lane, b);
#pragma unroll
                for (int i = 0; i < kLaneElems; ++i) h[j][i] = fmaf((h[j][i] - st.mean) * st.rstd, w[i], b[i]);
            }
        }
        if (a.gate) {
            const T* gr = static_cast<const T*>(a.gate) + (uint32_t(row) / uint32_t(a.gate_rows)) * a.gate_stride;
#pragma unroll
            for (int j = 0; j < CPW; ++j) {
                float g[kLaneElems];
                load_chunk<VEC>(gr, (warp + j * warps) * kChunk, dim, lane, g);
#pragma unroll
                for (int i = 0; i < kLaneElems; ++i) {
                    if (a.gate_act == kGateSigmoid) g[i] = 1.f / (1.f + expf(-g[i]));
                    if (a.gate_act == kGateTanh) g[i] = tanhf(g[i]);
                    h[j][i] *= g[i];
                }
            }
        }
#pragma unroll
        for (int j = 0; j < CPW; ++j) {
            const int c0 = (warp + j * warps) * kChunk;
            float ch[kLaneElems];
            load_weight<VEC>(a.channel, 1.f, c0, dim, lane, ch);
#pragma unroll
            for (int i = 0; i < kLaneElems; ++i) {
                // Columns past dim stay out of the row's sums.
                const bool in = c0 + chunk_col<VEC>(lane, i) < dim;
                x[j][i] = in ? fmaf(a.branch_scale * ch[i], h[j][i], a.resid_scale * x[j][i]) : 0.f;
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < CPW; ++j)
#pragma unroll
            for (int i = 0; i < kLaneElems; ++i) x[j][i] *= a.resid_scale;
    }
    if (a.x_out) {
        R* xo = static_cast<R*>(a.x_out) + row * a.x_out_stride;
#pragma unroll
        for (int j = 0; j < CPW; ++j) store_chunk<VEC>(xo, (warp + j * warps) * kChunk, dim, lane, x[j]);
    }
    if (!a.u) return;
    const RowStats st = row_stats<CPW, VEC>(x, a.layer, dim, a.eps, warp, warps, lane, exchange);
#pragma unroll
    for (int j = 0; j < CPW; ++j) {
        const int c0 = (warp + j * warps) * kChunk;
        float w[kLaneElems], b[kLaneElems];
        load_weight<VEC>(a.pre_weight, 1.f, c0, dim, lane, w);
        load_weight<VEC>(a.pre_bias, 0.f, c0, dim, lane, b);
#pragma unroll
        for (int i = 0; i < kLaneElems; ++i) w[i] = fmaf((x[j][i] - st.mean) * st.rstd, w[i], b[i]);
        if (!a.u_eight) {
            store_chunk<VEC>(static_cast<T*>(a.u) + row * a.u_stride, c0, dim, lane, w);
            continue;
        }
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < kLaneElems; ++i)
            if (c0 + chunk_col<VEC>(lane, i) < dim) m = max(m, abs_bits(w[i]));
#pragma unroll
        for (int o = 8; o; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        const BlockScale s = block_scale(m);
        uint8_t* q = static_cast<uint8_t*>(a.u) + row * a.u_stride;
        const uint32_t lo = pack_e4m3x4(w[0] * s.inv, w[1] * s.inv, w[2] * s.inv, w[3] * s.inv);
        const uint32_t hi = pack_e4m3x4(w[4] * s.inv, w[5] * s.inv, w[6] * s.inv, w[7] * s.inv);
        if (VEC) {
            if (c0 + lane * kLaneElems < dim) *reinterpret_cast<uint2*>(q + c0 + lane * kLaneElems) = make_uint2(lo, hi);
        } else {
#pragma unroll
            for (int i = 0; i < kLaneElems; ++i) {
                const int c = c0 + chunk_col<VEC>(lane, i);
                if (c < dim) q[c] = uint8_t((i < 4 ? lo : hi) >> (8 * (i & 3)));
            }
        }
        const int g0 = c0 + (lane >> 4) * kScaleBlock;
        if ((lane & 15) == 0 && g0 < dim) a.u_scale[int64_t(g0 / kScaleBlock) * a.u_scale_stride + row] = s.scale;
    }
}

template <typename T, typename R, int CPW>
cudaError_t launch_cpw(const NormResidualArgs& a, dim3 grid, dim3 block, cudaStream_t stream) {
    if (a.vec) norm_residual_kernel<T, R, CPW, true><<<grid, block, 0, stream>>>(a);
    else norm_residual_kernel<T, R, CPW, false><<<grid, block, 0, stream>>>(a);
    return cudaGetLastError();
}

template <typename T, typename R>
cudaError_t launch_types(const NormResidualArgs& a, cudaStream_t stream) {
    const int chunks = (a.dim + kChunk - 1) / kChunk;
    // Many rows: as few warps a row as hold it, for whole rows in flight
    // without barriers.  Few rows: one chunk a warp, for latency.
    const int cpw = a.rows >= 2048 || chunks > 16 ? 4 : 1;
    const int warps = (chunks + cpw - 1) / cpw;
    const int rows_per_cta = warps == 1 ? 4 : 1;
    const int64_t ctas = (a.rows + rows_per_cta - 1) / rows_per_cta;
    if (ctas > 0x7fffffff || warps > kMaxWarps) return cudaErrorInvalidValue;
    const dim3 grid{uint32_t(ctas)}, block(32 * warps, rows_per_cta);
    return cpw == 4 ? launch_cpw<T, R, 4>(a, grid, block, stream) : launch_cpw<T, R, 1>(a, grid, block, stream);
}

}  // namespace

cudaError_t launch_norm_residual(const NormResidualArgs& a, cudaStream_t stream) {
    switch (a.kind) {
        case kF32: return launch_types<float, float>(a, stream);
        case kF16:
            return a.resid_kind == kF32 ? launch_types<__half, float>(a, stream) : launch_types<__half, __half>(a, stream);
        case kBF16:
            return a.resid_kind == kF32 ? launch_types<__nv_bfloat16, float>(a, stream)
                                        : launch_types<__nv_bfloat16, __nv_bfloat16>(a, stream);
    }
    return cudaErrorInvalidValue;
}

}  // namespace s3t
