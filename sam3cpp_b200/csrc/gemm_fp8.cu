// Matrix product of 8-bit operands with a scale for each block of 128:
//   y[m][n] = act( sum_g xs[g][m] ws[g][n / 128] P_g[m][n] + bias[n] ),
//   P_g[m][n] = sum over the 128 columns k of group g of x[m][k] w[n][k],
// x and w e4m3 row-major.  The scales change with g, so a tensor-memory
// accumulator holds one group's P_g only (four K = 32 UMMAs) and the promotion
// warps add xs ws P_g to fp32 registers while the next group's UMMAs run into
// another accumulator.  Rows, columns and K beyond the matrices are zero-filled
// by TMA and their scales read as 0.
//
// gemm_fp8_pair_kernel: tiles of 256 x 256 by a CTA pair, for many rows.  Per
// group a pair's UMMAs take 512 clocks at the nominal rate; the promotion of a
// CTA's 128 x 256 share is 64 packed FMAs and 128 TMEM columns per thread of
// eight warps.  A warp's 128 columns lie in one weight block, so its factor is
// one number per row and group.
//
// gemm_fp8_tile_kernel: for few rows, with the operands swapped: 128 rows of w
// are the UMMA's M and 16 to 128 rows of x its N, so one token costs one pass
// over the weights at full load width.  The groups are split over the CTAs of a
// cluster, which add their fp32 tiles through distributed shared memory in a
// fixed order: no workspace, no atomics, the same result every time.
#include "fp8.cuh"
#include "elements.cuh"
#include "kernels.h"

namespace s3t {

namespace {

constexpr int kTileM = 128;
constexpr uint32_t kStageRow = kScaleBlock;                    // bytes of a K group of one row
constexpr uint32_t kHalfBytes = kTileM * kStageRow;            // 128 rows of a group

template <int OUT>
struct OutType;
template <>
struct OutType<kF32> { using T = float; };
template <>
struct OutType<kF16> { using T = __half; };
template <>
struct OutType<kBF16> { using T = __nv_bfloat16; };
template <>
struct OutType<kE4M3> { using T = uint8_t; };

S3T_DEV float2 packed_fma(float a0, float a1, float2 s, float2 c) { return __ffma2_rn(make_float2(a0, a1), s, c); }

// ------------------------------------------------------------- few rows ---

template <int BN>
struct TileCfg {
    static constexpr int STAGES = BN == 16 ? 6 : BN == 32 ? 5 : BN == 64 ? 4 : 3;
    static constexpr int ACCS = BN == 128 ? 2 : 4;             // accumulators in flight
    static constexpr uint32_t TMEM_COLS = ACCS * BN;
    static constexpr uint32_t X_BYTES = BN * kStageRow;
    static constexpr uint32_t STAGE_BYTES = kHalfBytes + X_BYTES;
    static constexpr uint32_t RING = STAGES * STAGE_BYTES;
    static constexpr uint32_t RED_BYTES = BN * kTileM * 4;     // the fp32 tile, over the drained ring
    static constexpr uint32_t SCALE_BYTES = 4 * 2 * BN * 4;    // [promotion warp][parity][column]
    static constexpr size_t SMEM = RING + SCALE_BYTES + 1024 + 256;
    static constexpr int THREADS = 192;
    static_assert(RED_BYTES <= RING, "the fp32 tile replaces the ring");
    // Two CTAs fit an SM and a third does not, whichever instances they are:
    // their tensor memory (at most 2 x 256 columns) never runs out, so no CTA
    // of a cluster waits for an allocation that another cluster holds.
    static_assert(TMEM_COLS <= 256 && SMEM <= 113 * 1024 && SMEM > 76 * 1024, "two CTAs per SM");
};

template <int BN, int OUT>
__global__ void __launch_bounds__(192)
    gemm_fp8_tile_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                         const GemmFp8Args args) {
    using Cfg = TileCfg<BN>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sW = smem;
    uint8_t* sX = smem + Cfg::STAGES * kHalfBytes;
    float* scales = reinterpret_cast<float*>(smem + Cfg::RING);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + Cfg::RING + Cfg::SCALE_BYTES);
    uint64_t* empty = full + Cfg::STAGES;
    uint64_t* tfull = empty + Cfg::STAGES;
    uint64_t* tempty = tfull + Cfg::ACCS;
    uint64_t* drain = tempty + Cfg::ACCS;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = int(cluster_ctarank()), splits = int(cluster_nctarank());
    const int tiles_n = (args.N + kTileM - 1) / kTileM;
    const int tile = int(blockIdx.x) / splits;
    const int n0 = (tile % tiles_n) * kTileM, m0 = (tile / tiles_n) * BN;
    const int groups = (args.K + kScaleBlock - 1) / kScaleBlock;
    const int g0 = int(int64_t(groups) * rank / splits), g1 = int(int64_t(groups) * (rank + 1) / splits);

    if (threadIdx.x == 0) {
        for (int s = 0; s < Cfg::STAGES; ++s) {
            mbar_init(full + s, 1);
            mbar_init(empty + s, 1);
        }
        for (int i = 0; i < Cfg::ACCS; ++i) {
            mbar_init(tfull + i, 1);
            mbar_init(tempty + i, 4);
        }
        mbar_init(drain, 1);
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, Cfg::TMEM_COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    if (warp == 0) {
        if (lane == 0) {
            int s = 0;
            uint32_t ph = 0, armed = 0, armed_parity = 0;
            bool ok = true;
            for (int g = g0; g < g1; ++g) {
                if (!mbar_wait(empty + s, ph ^ 1, args.status, kErrTimeoutProducer, abort_flag)) {
                    ok = false;
                    break;
                }
                mbar_arrive_expect_tx(full + s, Cfg::STAGE_BYTES);
                armed |= 1u << s;
                armed_parity = (armed_parity & ~(1u << s)) | (ph << s);
                tma_load_2d(sW + s * kHalfBytes, &tmW, full + s, g * kScaleBlock, n0);
                tma_load_2d(sX + s * Cfg::X_BYTES, &tmX, full + s, g * kScaleBlock, m0);
                if (++s == Cfg::STAGES) {
                    s = 0;
                    ph ^= 1;
                }
            }
            if (!ok) {
                for (int i = 0; i < Cfg::STAGES; ++i)
                    if (armed & (1u << i))
                        mbar_wait(full + i, (armed_parity >> i) & 1u, args.status, kErrTimeoutDrain, nullptr);
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t idesc = umma_idesc_e4m3(kTileM, BN);
            const uint64_t dW0 = umma_desc_sw128(smem_u32(sW), 16, 1024);
            const uint64_t dX0 = umma_desc_sw128(smem_u32(sX), 16, 1024);
            int s = 0;
            uint32_t ph = 0;
            bool ok = true, issued = false;
            for (int i = 0; i < g1 - g0; ++i) {
                const int acc = i % Cfg::ACCS;
                const uint32_t aph = (i / Cfg::ACCS) & 1;
                if (!mbar_wait(tempty + acc, aph ^ 1, args.status, kErrTimeoutMma, abort_flag) ||
                    !mbar_wait(full + s, ph, args.status, kErrTimeoutMma, abort_flag)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint64_t dw = dW0 + uint64_t(s) * (kHalfBytes >> 4), dx = dX0 + uint64_t(s) * (Cfg::X_BYTES >> 4);
#pragma unroll
                for (int k = 0; k < 4; ++k) umma_f8_ss(tmem_base + acc * BN, dw + 2 * k, dx + 2 * k, idesc, k != 0);
                issued = true;
                umma_commit(empty + s);
                umma_commit(tfull + acc);
                if (++s == Cfg::STAGES) {
                    s = 0;
                    ph ^= 1;
                }
            }
            if (!ok && issued) {
                umma_commit(drain);
                mbar_wait(drain, 0, args.status, kErrTimeoutDrain, nullptr);
            }
        }
    } else {
        // Promotion warp w: TMEM lanes (rows of w) 32 * (w % 4) .. + 31, all BN columns (rows of x).
        const int quarter = warp & 3;
        float* my_scales = scales + (warp - 2) * 2 * BN;
        constexpr int PER_LANE = (BN + 31) / 32;
        float next[PER_LANE];
        const int nb = n0 / kScaleBlock;
        auto fetch = [&](int g) {
            const float sw = __ldg(args.ws + int64_t(g) * args.ws_stride + nb);
#pragma unroll
            for (int i = 0; i < PER_LANE; ++i) {
                const int j = lane + 32 * i, m = m0 + j;
                next[i] = j < BN && m < args.M ? __ldg(args.xs + int64_t(g) * args.xs_stride + m) * sw : 0.f;
            }
        };
        fetch(g0);
        float2 sum[BN / 2];
#pragma unroll
        for (int i = 0; i < BN / 2; ++i) sum[i] = make_float2(0.f, 0.f);
        for (int i = 0; i < g1 - g0; ++i) {
            const int acc = i % Cfg::ACCS;
            const uint32_t aph = (i / Cfg::ACCS) & 1;
            float* sc = my_scales + (i & 1) * BN;
#pragma unroll
            for (int q = 0; q < PER_LANE; ++q)
                if (lane + 32 * q < BN) sc[lane + 32 * q] = next[q];
            __syncwarp();
            if (i + 1 < g1 - g0) fetch(g0 + i + 1);
            if (!mbar_wait(tfull + acc, aph, args.status, kErrTimeoutEpilogue, abort_flag)) break;
            tc_fence_after();
            const uint32_t t = tmem_base + (uint32_t(quarter * 32) << 16) + acc * BN;
            if constexpr (BN == 16) {
                uint32_t r[16];
                tmem_ld16(t, r);
                tmem_wait_ld();
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    sum[c] = packed_fma(__uint_as_float(r[2 * c]), __uint_as_float(r[2 * c + 1]),
                                        *reinterpret_cast<const float2*>(sc + 2 * c), sum[c]);
            } else {
#pragma unroll
                for (int b = 0; b < BN / 32; ++b) {
                    uint32_t r[32];
                    tmem_ld32(t + 32 * b, r);
                    tmem_wait_ld();
#pragma unroll
                    for (int c = 0; c < 16; ++c)
                        sum[16 * b + c] = packed_fma(__uint_as_float(r[2 * c]), __uint_as_float(r[2 * c + 1]),
                                                     *reinterpret_cast<const float2*>(sc + 32 * b + 2 * c), sum[16 * b + c]);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(tempty + acc);
        }
        // Every UMMA of this CTA has completed (the last accumulator is full),
        // so the ring is free: the tile goes there as [x row][w row].
        float* red = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int j = 0; j < BN / 2; ++j) {
            red[(2 * j) * kTileM + quarter * 32 + lane] = sum[j].x;
            red[(2 * j + 1) * kTileM + quarter * 32 + lane] = sum[j].y;
        }
    }
    __syncwarp();
    cluster_sync();
    // Each CTA of the cluster finishes BN / splits rows of x: a warp takes one
    // row, a lane four consecutive columns of y.
    {
        using T = typename OutType<OUT>::T;
        const uint32_t red = smem_u32(smem);
        const int j1 = BN * (rank + 1) / splits;
        for (int j = BN * rank / splits + warp; j < j1; j += Cfg::THREADS / 32) {
            const int m = m0 + j, n = n0 + lane * 4;
            if (m >= args.M) break;
            float v[4] = {0.f, 0.f, 0.f, 0.f};
            for (int q = 0; q < splits; ++q) {
                const float4 p = ld_cluster_f4(mapa_shared(red, q) + (j * kTileM + lane * 4) * 4);
                v[0] += p.x; v[1] += p.y; v[2] += p.z; v[3] += p.w;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (args.bias && n + i < args.N) v[i] += __ldg(args.bias + n + i);
            }
            if (args.gelu) {
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = gelu_erf_as(v[i]);
            }
            T* row = static_cast<T*>(args.y) + int64_t(m) * args.y_stride;
            const bool whole = args.vec && n + 4 <= args.N;
            if constexpr (OUT == kE4M3) {
                uint32_t a = max(max(abs_bits(v[0]), abs_bits(v[1])), max(abs_bits(v[2]), abs_bits(v[3])));
                a = __reduce_max_sync(0xffffffffu, a);
                const BlockScale s = block_scale(a);
                if (lane == 0) args.ys[int64_t(n0 / kScaleBlock) * args.ys_stride + m] = s.scale;
                const uint32_t c = pack_e4m3x4(v[0] * s.inv, v[1] * s.inv, v[2] * s.inv, v[3] * s.inv);
                if (whole) {
                    *reinterpret_cast<uint32_t*>(row + n) = c;
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (n + i < args.N) row[n + i] = uint8_t(c >> (8 * i));
                }
            } else if (whole) {
                if constexpr (OUT == kF32)
                    *reinterpret_cast<float4*>(row + n) = make_float4(v[0], v[1], v[2], v[3]);
                else
                    *reinterpret_cast<uint2*>(row + n) = make_uint2(pack2(v[0], v[1], T()), pack2(v[2], v[3], T()));
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (n + i < args.N) row[n + i] = from_float<T>(v[i]);
            }
        }
    }
    tc_fence_before();
    __syncwarp();
    cluster_sync();   // no CTA leaves while another still reads its tile
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, Cfg::TMEM_COLS);
    }
}

template <int BN, int OUT>
cudaError_t launch_tile(const GemmFp8Args& a, int num_sms, cudaStream_t stream) {
    using Cfg = TileCfg<BN>;
    CUtensorMap tw, tx;
    if (!make_tmap_rows(&tw, a.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.K, a.N, a.w_stride, kStageRow, kTileM) ||
        !make_tmap_rows(&tx, a.x, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.K, a.M, a.x_stride, kStageRow, BN))
        return cudaErrorInvalidValue;
    const int64_t tiles = (int64_t(a.N) + kTileM - 1) / kTileM * ((int64_t(a.M) + BN - 1) / BN);
    if (tiles > (1 << 27)) return cudaErrorInvalidValue;
    const int groups = (a.K + kScaleBlock - 1) / kScaleBlock;
    int splits = 1;
    while (splits < 8 && 2 * splits <= groups && tiles * 2 * splits <= 2 * num_sms) splits *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(uint32_t(tiles) * splits);
    cfg.blockDim = dim3(Cfg::THREADS);
    cfg.dynamicSmemBytes = Cfg::SMEM;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = splits;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, gemm_fp8_tile_kernel<BN, OUT>, tw, tx, a);
}

template <int OUT>
cudaError_t launch_out(const GemmFp8Args& a, int num_sms, cudaStream_t stream) {
    if (a.M <= 16) return launch_tile<16, OUT>(a, num_sms, stream);
    if (a.M <= 32) return launch_tile<32, OUT>(a, num_sms, stream);
    if (a.M <= 64) return launch_tile<64, OUT>(a, num_sms, stream);
    return launch_tile<128, OUT>(a, num_sms, stream);
}

template <int BN, int OUT>
cudaError_t prepare_tile() {
    return cudaFuncSetAttribute(gemm_fp8_tile_kernel<BN, OUT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                int(TileCfg<BN>::SMEM));
}

template <int OUT>
cudaError_t prepare_out() {
    cudaError_t e;
    if ((e = prepare_tile<16, OUT>()) != cudaSuccess) return e;
    if ((e = prepare_tile<32, OUT>()) != cudaSuccess) return e;
    if ((e = prepare_tile<64, OUT>()) != cudaSuccess) return e;
    return prepare_tile<128, OUT>();
}

}  // namespace

cudaError_t fp8_prepare() {
    cudaError_t e;
    if ((e = prepare_out<kF32>()) != cudaSuccess) return e;
    if ((e = prepare_out<kF16>()) != cudaSuccess) return e;
    if ((e = prepare_out<kBF16>()) != cudaSuccess) return e;
    return prepare_out<kE4M3>();
}

cudaError_t launch_gemm_fp8(const GemmFp8Args& a, int num_sms, cudaStream_t stream) {
    switch (a.out) {
        case kF32: return launch_out<kF32>(a, num_sms, stream);
        case kF16: return launch_out<kF16>(a, num_sms, stream);
        case kBF16: return launch_out<kBF16>(a, num_sms, stream);
        case kE4M3: return launch_out<kE4M3>(a, num_sms, stream);
    }
    return cudaErrorInvalidValue;
}

}  // namespace s3t
