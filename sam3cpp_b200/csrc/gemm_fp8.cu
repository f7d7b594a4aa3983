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
// group a pair's UMMAs take 514 clocks alone (two of N = 128 instead took 958:
// x is read again), a promotion warp loads 128 TMEM columns and does 64 packed
// FMAs a thread.  A warp's 128 columns lie in one weight block, so its factor
// is one number per row and group.  Measured (82944 x 1024 x 4736, fp16 out):
// 386 us, 2.09 PFLOP/s; with the promotion's FMAs left out 344 us, its loads
// 366 us, both 307 us, which the 1 kW cap holds.  So it is bound by the tensor
// pipe and the promotion together: the accumulators fill tensor memory, two
// groups are in flight, and a group's accumulator is free again about 700
// clocks after it is full.  A tile's epilogue is not overlapped with the next
// mainloop beyond those two groups (2700 clocks for fp16, 5000 with GELU and
// e4m3, when the bias was still added there; now it begins the sums), which is
// what K = 1024 pays for: 5184 x 4736 x 1024, GELU, e4m3 46-49 us, 36-39 us
// without GELU.
//
// gemm_fp8_tile_kernel: for few rows, with the operands swapped: 128 rows of w
// are the UMMA's M and 16 to 64 rows of x its N, so one token costs one pass
// over the weights at full load width.  The groups are split over the CTAs of a
// cluster, which add their fp32 tiles through distributed shared memory in a
// fixed order: no workspace, no atomics, the same result every time.  1 x 4736
// x 1024 5.5 us (bound by its chain of latencies: launch, load, UMMA, cluster
// exchange), 1 x 8192 x 8192 12.4 us (5.4 TB/s of weights).
#include "fp8.cuh"
#include "elements.cuh"
#include "kernels.h"

namespace s3t {

namespace {

constexpr int kTileM = 128;
constexpr uint32_t kStageRow = kScaleBlock;                    // bytes of a K group of one row
constexpr uint32_t kHalfBytes = kTileM * kStageRow;            // 128 rows of a group
constexpr int kMaxSplits = 8;                                  // CTAs that share a tile's groups

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

// Four accumulator columns times their factors, added to two sums.
S3T_DEV void add4(const uint32_t* r, const float* factors, float2& a, float2& b) {
    const float4 f = *reinterpret_cast<const float4*>(factors);
    a = __ffma2_rn(make_float2(__uint_as_float(r[0]), __uint_as_float(r[1])), make_float2(f.x, f.y), a);
    b = __ffma2_rn(make_float2(__uint_as_float(r[2]), __uint_as_float(r[3])), make_float2(f.z, f.w), b);
}

S3T_DEV float2 packed_fma(float a0, float a1, float2 s, float2 c) { return __ffma2_rn(make_float2(a0, a1), s, c); }

// ------------------------------------------------------------- few rows ---

template <int BN>
struct TileCfg {
    static constexpr int STAGES = BN <= 32 ? 5 : 4;
    static constexpr int ACCS = 4;                             // accumulators in flight
    static constexpr uint32_t TMEM_COLS = ACCS * BN;
    static constexpr uint32_t X_BYTES = BN * kStageRow;
    static constexpr uint32_t STAGE_BYTES = kHalfBytes + X_BYTES;
    static constexpr uint32_t RING = STAGES * STAGE_BYTES;
    static constexpr uint32_t RED_BYTES = BN * kTileM * 4;     // the fp32 tile, over the drained ring
    // Per promotion warp: a ring of raw scales (the block's and a row's per lane)
    // and two buffers of their products.
    static constexpr int SCALE_SLOTS = 4;
    static constexpr int SCALE_WORDS = SCALE_SLOTS * 32 * ((BN + 31) / 32 + 1) + 2 * BN;
    static constexpr uint32_t SCALE_BYTES = 4 * SCALE_WORDS * 4;
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

    // The producer makes the barriers and asks for the first stages before the
    // other warps are ready: a call of one token is all latency.
    int s = 0, g = g0;
    uint32_t ph = 0, armed = 0, armed_parity = 0;
    auto load = [&]() {
        mbar_arrive_expect_tx(full + s, Cfg::STAGE_BYTES);
        armed |= 1u << s;
        armed_parity = (armed_parity & ~(1u << s)) | (ph << s);
        tma_load_2d(sW + s * kHalfBytes, &tmW, full + s, g * kScaleBlock, n0);
        tma_load_2d(sX + s * Cfg::X_BYTES, &tmX, full + s, g * kScaleBlock, m0);
        ++g;
        if (++s == Cfg::STAGES) {
            s = 0;
            ph ^= 1;
        }
    };
    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tmW);
        tma_prefetch_desc(&tmX);
        for (int i = 0; i < Cfg::STAGES; ++i) {
            mbar_init(full + i, 1);
            mbar_init(empty + i, 1);
        }
        for (int i = 0; i < Cfg::ACCS; ++i) {
            mbar_init(tfull + i, 1);
            mbar_init(tempty + i, 4);
        }
        mbar_init(drain, 1);
        *abort_flag = 0;
        fence_barrier_init();
        while (g < g1 && g - g0 < Cfg::STAGES) load();
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
            bool ok = true;
            while (g < g1) {
                if (!mbar_wait(empty + s, ph ^ 1, args.status, kErrTimeoutProducer, abort_flag)) {
                    ok = false;
                    break;
                }
                load();
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
        constexpr int PER_LANE = (BN + 31) / 32;
        // The scales of the BN rows and of the weight block come by cp.async,
        // SCALE_SLOTS - 1 groups ahead, into words that only this lane reads: a
        // load into a register would stall the warp at its first use.
        float* raw = scales + (warp - 2) * Cfg::SCALE_WORDS + lane;
        float* products = scales + (warp - 2) * Cfg::SCALE_WORDS + Cfg::SCALE_SLOTS * 32 * (PER_LANE + 1);
        const float* ahead_w = args.ws + int64_t(g0) * args.ws_stride + n0 / kScaleBlock;
        const float* ahead_x = args.xs + int64_t(g0) * args.xs_stride + (m0 + lane < args.M ? m0 + lane : 0);
        auto fetch = [&](int g) {
            float* slot = raw + ((g - g0) % Cfg::SCALE_SLOTS) * 32 * (PER_LANE + 1);
            if (g < g1) {
                cp_async4(slot, ahead_w, true);
#pragma unroll
                for (int i = 0; i < PER_LANE; ++i) {
                    const int j = lane + 32 * i;
                    const bool take = j < BN && m0 + j < args.M;
                    cp_async4(slot + 32 * (i + 1), ahead_x + (take ? 32 * i : 0), take);
                }
                if (g + 1 < g1) {
                    ahead_w += args.ws_stride;
                    ahead_x += args.xs_stride;
                }
            }
            cp_async_commit();
        };
        for (int i = 0; i < Cfg::SCALE_SLOTS - 1; ++i) fetch(g0 + i);
        float2 sum[BN / 2];
#pragma unroll
        for (int i = 0; i < BN / 2; ++i) sum[i] = make_float2(0.f, 0.f);
        for (int i = 0; i < g1 - g0; ++i) {
            const int acc = i % Cfg::ACCS;
            const uint32_t aph = (i / Cfg::ACCS) & 1;
            fetch(g0 + i + Cfg::SCALE_SLOTS - 1);
            cp_async_wait<Cfg::SCALE_SLOTS - 1>();
            const float* slot = raw + (i % Cfg::SCALE_SLOTS) * 32 * (PER_LANE + 1);
            float* sc = products + (i & 1) * BN;
#pragma unroll
            for (int q = 0; q < PER_LANE; ++q)
                if (lane + 32 * q < BN) sc[lane + 32 * q] = slot[32 * (q + 1)] * slot[0];
            __syncwarp();
            if (!mbar_wait(tfull + acc, aph, args.status, kErrTimeoutEpilogue, abort_flag)) break;
            tc_fence_after();
            const uint32_t t = tmem_base + (uint32_t(quarter * 32) << 16) + acc * BN;
            if constexpr (BN == 16) {
                uint32_t r[16];
                tmem_ld16(t, r);
                tmem_wait_ld();
#pragma unroll
                for (int c = 0; c < 4; ++c) add4(r + 4 * c, sc + 4 * c, sum[2 * c], sum[2 * c + 1]);
            } else {
#pragma unroll
                for (int b = 0; b < BN / 32; ++b) {
                    uint32_t r[32];
                    tmem_ld32(t + 32 * b, r);
                    tmem_wait_ld(r);
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        add4(r + 4 * c, sc + 32 * b + 4 * c, sum[16 * b + 2 * c], sum[16 * b + 2 * c + 1]);
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
            // All the cluster's parts at once (one after the other is a remote
            // latency each), added in the order of the ranks.
            float4 part[kMaxSplits];
#pragma unroll
            for (int q = 0; q < kMaxSplits; ++q)
                if (q < splits) part[q] = ld_cluster_f4(mapa_shared(red, q) + (j * kTileM + lane * 4) * 4);
            float v[4] = {part[0].x, part[0].y, part[0].z, part[0].w};
#pragma unroll
            for (int q = 1; q < kMaxSplits; ++q)
                if (q < splits) {
                    v[0] += part[q].x; v[1] += part[q].y; v[2] += part[q].z; v[3] += part[q].w;
                }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (args.bias && n + i < args.N) v[i] += __ldg(args.bias + n + i);
            }
            if (args.gelu) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float2 t = gelu_erf_poly2(make_float2(v[2 * i], v[2 * i + 1]));
                    v[2 * i] = t.x;
                    v[2 * i + 1] = t.y;
                }
            }
            T* row = static_cast<T*>(args.y) + int64_t(m) * args.y_stride;
            const bool whole = args.vec && n + 4 <= args.N;
            if constexpr (OUT == kE4M3) {
                // Columns past N take no part in the block: their products are 0,
                // and NaN under an infinite scale.
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (n + i >= args.N) v[i] = 0.f;
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

int groups_of(int K) { return K / kScaleBlock + (K % kScaleBlock != 0); }

// CTAs that share a tile's groups: as many as give every SM one CTA, or two
// while each has eight groups and more.  (1 x 4736 x 1024: 5.5 us with 148
// CTAs, 8.1 us with 296 of one group; 1 x 8192 x 8192: 12.8 us with 256 CTAs
// of 16 groups, 16.7 us with 128 of 32.)
int tile_splits(int64_t tiles, int groups, int num_sms) {
    int splits = 1;
    while (2 * splits <= kMaxSplits && 2 * splits <= groups &&
           tiles * 2 * splits <= (groups >= 16 * splits ? 2 * num_sms : num_sms))
        splits *= 2;
    return splits;
}

int64_t tiles_of(int M, int N, int bm, int bn) {
    return (int64_t(M) + bm - 1) / bm * ((int64_t(N) + bn - 1) / bn);
}

template <int BN, int OUT>
cudaError_t launch_tile(const GemmFp8Args& a, int num_sms, cudaStream_t stream) {
    using Cfg = TileCfg<BN>;
    CUtensorMap tw, tx;
    if (!make_tmap_rows(&tw, a.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.K, a.N, a.w_stride, kStageRow, kTileM) ||
        !make_tmap_rows(&tx, a.x, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.K, a.M, a.x_stride, kStageRow, BN))
        return cudaErrorInvalidValue;
    const int64_t tiles = tiles_of(a.M, a.N, BN, kTileM);
    if (tiles > (1 << 27)) return cudaErrorInvalidValue;
    const int splits = tile_splits(tiles, groups_of(a.K), num_sms);
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

// -------------------------------------------------------------- many rows ---

struct PairCfg8 {
    static constexpr int BN = 256;
    static constexpr int STAGES = 4;
    static constexpr int WARPS = 8;                            // promotion and epilogue
    static constexpr int WARP_COLS = BN * 4 / WARPS;           // 128: one weight block
    static constexpr uint32_t STAGE_BYTES = 2 * kHalfBytes;    // 128 rows of x, 128 rows of w per CTA
    static constexpr uint32_t RING = STAGES * STAGE_BYTES;
    static constexpr uint32_t OUT_ROW = 128;                   // bytes of a row of y staged at a time
    static constexpr uint32_t OUT_BUF = 32 * OUT_ROW;
    static constexpr int OUT_BUFS = 2;                         // per warp: all of a 16-bit tile
    static constexpr uint32_t OUT_BYTES = WARPS * OUT_BUFS * OUT_BUF;
    static constexpr int RAW_SLOTS = 6;                        // groups of scales on their way
    static constexpr int RAW_WORDS = 64 * 4;                   // two row and two block scales per factor thread
    static constexpr int FACTOR_SLOTS = 4;
    static constexpr int FACTOR_WORDS = 2 * kTileM;            // a factor per row and weight block
    static constexpr uint32_t SMALL_BYTES = 4 * (RAW_SLOTS * RAW_WORDS + FACTOR_SLOTS * FACTOR_WORDS + 2 * WARPS * WARP_COLS);
    static constexpr uint32_t TMEM_COLS = 2 * BN;
    static constexpr size_t SMEM = RING + OUT_BYTES + SMALL_BYTES + 1024 + 256;
    // Warpgroup 0: TMA producer, UMMA issuer and two factor warps; warpgroups 1
    // and 2: promotion.  The launch gives each of the 384 threads 168 registers
    // (64,512 in all); 128 sums and 64 columns in flight need more, so
    // warpgroup 0 keeps 72 (9,216) and the others take 216 (55,296).
    static constexpr int THREADS = 128 + 32 * WARPS;
    static constexpr int FEW_REGS = 72, MANY_REGS = 216;
    static_assert(128 * FEW_REGS + 32 * WARPS * MANY_REGS <= THREADS * 168, "the split stays within the launch");
};
static_assert(PairCfg8::WARP_COLS == kScaleBlock, "a warp's columns are one weight block");

template <int OUT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PairCfg8::THREADS, 1)
    gemm_fp8_pair_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW,
                         const __grid_constant__ CUtensorMap tmY, const GemmFp8Args args) {
    using Cfg = PairCfg8;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sX = smem;
    uint8_t* sW = smem + Cfg::STAGES * kHalfBytes;
    uint8_t* sOut = smem + Cfg::RING;
    float* raw = reinterpret_cast<float*>(sOut + Cfg::OUT_BYTES);
    float* factors = raw + Cfg::RAW_SLOTS * Cfg::RAW_WORDS;
    float* biases = factors + Cfg::FACTOR_SLOTS * Cfg::FACTOR_WORDS;
    uint64_t* full = reinterpret_cast<uint64_t*>(biases + 2 * Cfg::WARPS * Cfg::WARP_COLS);
    uint64_t* done = full + Cfg::STAGES;
    uint64_t* tempty = done + Cfg::STAGES;
    uint64_t* drain = tempty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    const int tiles_n = (args.N + Cfg::BN - 1) / Cfg::BN;
    const int n_tiles = ((args.M + 2 * kTileM - 1) / (2 * kTileM)) * tiles_n;
    const int pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;
    const int groups = (args.K + kScaleBlock - 1) / kScaleBlock;

    if (threadIdx.x == 0) {
        for (int s = 0; s < Cfg::STAGES; ++s) {
            mbar_init(full + s, 1);
            mbar_init(done + s, 1 + 2);              // the UMMAs and this CTA's factor warps
        }
        for (int i = 0; i < 2; ++i) mbar_init(tempty + i, 2 * Cfg::WARPS);   // every promotion warp of the pair
        mbar_init(drain, 1);
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc_pair(tmem_slot, Cfg::TMEM_COLS);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    cluster_sync();   // both CTAs' barriers exist before any cross-CTA arrive
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    if (warp < 4) {
        setmaxnreg_dec<Cfg::FEW_REGS>();
        if (warp == 0) {
            if (lane == 0) {
                int s = 0;
                uint32_t ph = 0, armed = 0, armed_parity = 0;
                bool ok = true;
                for (int tile = pair; ok && tile < n_tiles; tile += n_pairs) {
                    const int m0 = (tile / tiles_n) * 2 * kTileM + int(rank) * kTileM;
                    const int n0 = (tile % tiles_n) * Cfg::BN + int(rank) * kTileM;
                    for (int g = 0; g < groups; ++g) {
                        if (!mbar_wait(done + s, ph ^ 1, args.status, kErrTimeoutProducer, abort_flag)) {
                            ok = false;
                            break;
                        }
                        const uint32_t lfull = mapa_shared(smem_u32(full + s), 0);
                        if (leader) {
                            mbar_arrive_expect_tx(full + s, 2 * Cfg::STAGE_BYTES);
                            armed |= 1u << s;
                            armed_parity = (armed_parity & ~(1u << s)) | (ph << s);
                        }
                        tma_load_2d_pair(sX + s * kHalfBytes, &tmX, lfull, g * kScaleBlock, m0);
                        tma_load_2d_pair(sW + s * kHalfBytes, &tmW, lfull, g * kScaleBlock, n0);
                        if (++s == Cfg::STAGES) {
                            s = 0;
                            ph ^= 1;
                        }
                    }
                }
                if (!ok && leader) {
                    // Gave up: wait (bounded) for the pair's copies counted on these barriers.
                    for (int i = 0; i < Cfg::STAGES; ++i)
                        if (armed & (1u << i))
                            mbar_wait(full + i, (armed_parity >> i) & 1u, args.status, kErrTimeoutDrain, nullptr);
                }
            }
        } else if (warp == 1) {
            if (leader) {
                constexpr uint32_t idesc = umma_idesc_e4m3(2 * kTileM, Cfg::BN);
                const uint64_t dX0 = umma_desc_sw128(smem_u32(sX), 16, 1024);
                const uint64_t dW0 = umma_desc_sw128(smem_u32(sW), 16, 1024);
                int s = 0, it = 0;
                uint32_t ph = 0;
                bool ok = true, issued = false;
                for (int tile = pair; ok && tile < n_tiles; tile += n_pairs) {
                    for (int g = 0; g < groups; ++g, ++it) {
                        const int acc = it & 1;
                        const uint32_t aph = (it >> 1) & 1;
                        if (!mbar_wait(full + s, ph, args.status, kErrTimeoutMma, abort_flag) ||
                            !mbar_wait(tempty + acc, aph ^ 1, args.status, kErrTimeoutMma, abort_flag)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        const uint64_t dx = dX0 + uint64_t(s) * (kHalfBytes >> 4), dw = dW0 + uint64_t(s) * (kHalfBytes >> 4);
                        if (elect_one()) {
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                umma_f8_ss_pair(tmem_base + acc * Cfg::BN, dx + 2 * k, dw + 2 * k, idesc, k != 0);
                            // One commit per group (a second cost 61 clocks of the tensor
                            // pipe): the stage is free and its sums are in the accumulator.
                            umma_commit_pair(done + s, 0x3);
                        }
                        __syncwarp();
                        issued = true;
                        if (++s == Cfg::STAGES) {
                            s = 0;
                            ph ^= 1;
                        }
                    }
                }
                if (!ok && issued) {
                    if (elect_one()) umma_commit_pair(drain, 0x1);
                    __syncwarp();
                    mbar_wait(drain, 0, args.status, kErrTimeoutDrain, nullptr);
                }
            }
        } else {
            // Factor warps: xs ws of this CTA's 128 rows and two weight blocks, for
            // each group, so that a promotion warp reads one word.  The raw scales
            // come by cp.async, RAW_SLOTS - 1 groups ahead, into words of the
            // thread's own.  A group's done barrier counts these warps too.
            const int ft = int(threadIdx.x) - 64;
            float* mine = raw + ft * 4;
            int ahead_tile = pair - n_pairs, ahead_left = 0, ahead_slot = 0;
            const float *x0 = args.xs, *x1 = args.xs, *w0 = args.ws, *w1 = args.ws;
            bool in_x0 = false, in_x1 = false, in_w0 = false, in_w1 = false;
            auto fetch = [&]() {
                if (ahead_left == 0) {
                    ahead_tile += n_pairs;
                    const bool tile_ok = ahead_tile < n_tiles;
                    const int m = tile_ok ? (ahead_tile / tiles_n) * 2 * kTileM + int(rank) * kTileM + ft : 0;
                    const int n = tile_ok ? (ahead_tile % tiles_n) * Cfg::BN : 0;
                    in_x0 = tile_ok && m < args.M;
                    in_x1 = tile_ok && m + 64 < args.M;
                    in_w0 = tile_ok;
                    in_w1 = tile_ok && n + kScaleBlock < args.N;
                    x0 = args.xs + (in_x0 ? m : 0);
                    x1 = args.xs + (in_x1 ? m + 64 : 0);
                    w0 = args.ws + n / kScaleBlock;
                    w1 = in_w1 ? w0 + 1 : w0;
                    ahead_left = groups;
                }
                float* to = mine + ahead_slot * Cfg::RAW_WORDS;
                cp_async4(to, x0, in_x0);
                cp_async4(to + 1, x1, in_x1);
                cp_async4(to + 2, w0, in_w0);
                cp_async4(to + 3, w1, in_w1);
                cp_async_commit();
                ahead_slot = ahead_slot + 1 == Cfg::RAW_SLOTS ? 0 : ahead_slot + 1;
                if (--ahead_left > 0) {   // the pointers stop at a tile's last group
                    x0 += args.xs_stride;
                    x1 += args.xs_stride;
                    w0 += args.ws_stride;
                    w1 += args.ws_stride;
                }
            };
            for (int i = 0; i < Cfg::RAW_SLOTS - 1; ++i) fetch();
            int slot = 0, s = 0, lag = 0;          // lag: stage of group it - 2
            uint32_t lag_ph = 0;
            int it = 0;
            bool ok = true;
            for (int tile = pair; ok && tile < n_tiles; tile += n_pairs) {
                for (int g = 0; g < groups; ++g, ++it) {
                    fetch();
                    cp_async_wait<Cfg::RAW_SLOTS - 1>();
                    const float4 v = *reinterpret_cast<const float4*>(mine + slot * Cfg::RAW_WORDS);
                    slot = slot + 1 == Cfg::RAW_SLOTS ? 0 : slot + 1;
                    // Group it - 2 is in its accumulator, so the promotion of group
                    // it - 4, which this slot held, is over.
                    if (it >= 2) {
                        if (!mbar_wait(done + lag, lag_ph, args.status, kErrTimeoutProducer, abort_flag)) {
                            ok = false;
                            break;
                        }
                        if (++lag == Cfg::STAGES) {
                            lag = 0;
                            lag_ph ^= 1;
                        }
                    }
                    float* f = factors + (it % Cfg::FACTOR_SLOTS) * Cfg::FACTOR_WORDS + ft;
                    f[0] = v.x * v.z;
                    f[64] = v.y * v.z;
                    f[128] = v.x * v.w;
                    f[192] = v.y * v.w;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(done + s);
                    s = s + 1 == Cfg::STAGES ? 0 : s + 1;
                }
            }
            cp_async_wait<0>();
        }
    } else {
        setmaxnreg_inc<Cfg::MANY_REGS>();
        // Warp w reads TMEM lane quarter w % 4 (rows 32 * (w % 4) .. + 31 of this
        // CTA's half) and one half of the 256 columns.
        const int quarter = warp & 3, half = (warp - 4) >> 2;
        const uint32_t lanes = uint32_t(quarter * 32) << 16;
        uint8_t* stage = sOut + (warp - 4) * Cfg::OUT_BUFS * Cfg::OUT_BUF;
        float* my_bias = biases + (warp - 4) * 2 * Cfg::WARP_COLS;   // this tile's and the next one's
        const uint32_t my_factor = smem_u32(factors + half * kTileM + quarter * 32 + lane);
        int it = 0, out = 0, s = 0;   // groups promoted, the next buffer of y, the group's stage
        uint32_t ph = 0;
        bool ok = true;
        auto fetch_bias = [&](int tile, int which) {
            const int n0 = (tile % tiles_n) * Cfg::BN + half * Cfg::WARP_COLS;
#pragma unroll
            for (int i = 0; i < Cfg::WARP_COLS / 32; ++i) {
                const int n = n0 + lane + 32 * i;
                const bool take = tile < n_tiles && n < args.N;
                cp_async4(my_bias + which * Cfg::WARP_COLS + lane + 32 * i, args.bias + (take ? n : 0), take);
            }
            cp_async_commit();
        };
        int which = 0;
        if (args.bias) fetch_bias(pair, 0);
        for (int tile = pair; ok && tile < n_tiles; tile += n_pairs) {
            const int row0 = (tile / tiles_n) * 2 * kTileM + int(rank) * kTileM + quarter * 32;
            const int n0 = (tile % tiles_n) * Cfg::BN + half * Cfg::WARP_COLS;
            // The sums begin with the bias, which came during the tile before.
            float2 sum[Cfg::WARP_COLS / 2];
            if (args.bias) {
                cp_async_wait<0>();
                __syncwarp();
#pragma unroll
                for (int i = 0; i < Cfg::WARP_COLS / 4; ++i) {
                    const float4 b = ld_shared_f4(smem_u32(my_bias) + which * Cfg::WARP_COLS * 4 + 16 * i);
                    sum[2 * i] = make_float2(b.x, b.y);
                    sum[2 * i + 1] = make_float2(b.z, b.w);
                }
                which ^= 1;
                fetch_bias(tile + n_pairs, which);   // every lane left that buffer a tile ago
            } else {
#pragma unroll
                for (int i = 0; i < Cfg::WARP_COLS / 2; ++i) sum[i] = make_float2(0.f, 0.f);
            }
            // 64 columns on their way at a time, across groups too: the next
            // group's first columns are asked for before the last of this one
            // are added.  The accumulator goes back to the UMMA issuer once its
            // last columns are in registers, before half of them are added.
            uint32_t r[2][32];
            float f = 0.f;
            uint32_t t = 0;
            auto add = [&](const uint32_t (&v)[32], int b) {
#pragma unroll
                for (int c = 0; c < 16; ++c)
                    sum[16 * b + c] = packed_fma(__uint_as_float(v[2 * c]), __uint_as_float(v[2 * c + 1]), make_float2(f, f),
                                                 sum[16 * b + c]);
            };
            auto next_group = [&]() {   // waits for the next group's accumulator
                if (!mbar_wait(done + s, ph, args.status, kErrTimeoutEpilogue, abort_flag)) return false;
                if (++s == Cfg::STAGES) {
                    s = 0;
                    ph ^= 1;
                }
                tc_fence_after();
                t = tmem_base + lanes + (it & 1) * Cfg::BN + half * Cfg::WARP_COLS;
                return true;
            };
            ok = next_group();
            if (!ok) break;
            tmem_ld32(t, r[0]);
            tmem_ld32(t + 32, r[1]);
            f = ld_shared_f(my_factor + (it % Cfg::FACTOR_SLOTS) * Cfg::FACTOR_WORDS * 4);
#pragma unroll 1
            for (int g = 0; g < groups; ++g) {
                tmem_wait_ld(r[0]);
                tmem_wait_ld(r[1]);
                add(r[0], 0);
                tmem_ld32(t + 64, r[0]);
                add(r[1], 1);
                tmem_ld32(t + 96, r[1]);
                tmem_wait_ld(r[0]);
                tmem_wait_ld(r[1]);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(tempty + (it & 1)), 0));
                ++it;
                add(r[0], 2);
                if (g + 1 == groups) {
                    add(r[1], 3);
                    break;
                }
                ok = next_group();
                if (!ok) break;
                tmem_ld32(t, r[0]);
                const float f_next = ld_shared_f(my_factor + (it % Cfg::FACTOR_SLOTS) * Cfg::FACTOR_WORDS * 4);
                add(r[1], 3);
                tmem_ld32(t + 32, r[1]);
                f = f_next;
            }
            if (!ok) break;
            if (n0 >= args.N || row0 >= args.M) continue;   // warp-uniform: nothing of y here
            if (args.gelu) {
#pragma unroll
                for (int i = 0; i < Cfg::WARP_COLS / 2; ++i) sum[i] = gelu_erf_poly2(sum[i]);
            }
            // Each lane writes 128 bytes of its row at a time to a swizzled stage,
            // and one TMA store per warp takes the 32 rows while the next tile is
            // computed (every pair ends its tile at about the same time: stores that
            // the warps waited for cost 2 us a tile).  Where rows of y are not
            // 16-byte aligned, or the last columns end inside 16 bytes (a tiled
            // store wrote those whole: zeros behind the matrix), the warp copies
            // the stage element by element.
            using T = typename OutType<OUT>::T;
            constexpr int ELEM = int(sizeof(T));
            constexpr int CHUNK_COLS = int(Cfg::OUT_ROW) / ELEM;
            BlockScale bs{0.f, 0.f};
            if constexpr (OUT == kE4M3) {
                float a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < Cfg::WARP_COLS / 2; ++i) a[i & 3] = absmax3_nan(a[i & 3], sum[i].x, sum[i].y);
                float top = absmax3_nan(absmax3_nan(a[0], a[1], a[2]), a[3], a[3]);
                // As in the tile kernel, columns past N take no part.  Looked at again only
                // where they can matter, and by steps that stay in this branch:
                // masks that the compiler may compute ahead spill (fc1 48.9 -> 62.8 us).
                const int left = args.N - n0;
                if (left < Cfg::WARP_COLS && top != top) {
                    top = 0.f;
#pragma unroll
                    for (int i = 0; i < Cfg::WARP_COLS / 2; ++i) {
                        absmax_nan_if(top, sum[i].x, 2 * i, left);
                        absmax_nan_if(top, sum[i].y, 2 * i + 1, left);
                    }
                }
                bs = block_scale(abs_bits(top));
                if (row0 + lane < args.M) args.ys[int64_t(n0 / kScaleBlock) * args.ys_stride + row0 + lane] = bs.scale;
            }
#pragma unroll
            for (int c = 0; c < Cfg::WARP_COLS / CHUNK_COLS; ++c) {
                const int n = n0 + c * CHUNK_COLS;
                if (n >= args.N) break;
                uint8_t* buf = stage + out * Cfg::OUT_BUF;
                out = out + 1 == Cfg::OUT_BUFS ? 0 : out + 1;
                if (lane == 0) bulk_wait_group_read<Cfg::OUT_BUFS - 1>();   // the chunk that was in buf has left it
                __syncwarp();
                const uint32_t rowp = smem_u32(buf + lane * Cfg::OUT_ROW);
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    uint32_t w[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if constexpr (OUT == kF32) {
                            const float2 v = sum[c * 16 + q * 2 + i / 2];
                            w[i] = __float_as_uint(i & 1 ? v.y : v.x);
                        } else if constexpr (OUT == kE4M3) {
                            const float2 v0 = sum[q * 8 + 2 * i], v1 = sum[q * 8 + 2 * i + 1];
                            w[i] = pack_e4m3x4(v0.x * bs.inv, v0.y * bs.inv, v1.x * bs.inv, v1.y * bs.inv);
                        } else {
                            const float2 v = sum[c * 32 + q * 4 + i];
                            w[i] = pack2(v.x, v.y, T());
                        }
                    }
                    st_shared_u4(rowp + ((q ^ (lane & 7)) << 4), w[0], w[1], w[2], w[3]);
                }
                if (args.vec && (n + CHUNK_COLS <= args.N || int64_t(args.N) * ELEM % 16 == 0)) {
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) tma_store_2d(&tmY, buf, n, row0);
                } else {
                    __syncwarp();
#pragma unroll 8
                    for (int rr = 0; rr < 32; ++rr) {
                        T* y = static_cast<T*>(args.y) + int64_t(row0 + rr) * args.y_stride + n;
#pragma unroll
                        for (int k = 0; k < CHUNK_COLS / 32; ++k) {
                            const int col = lane + 32 * k, byte = col * ELEM;
                            const T v = *reinterpret_cast<const T*>(buf + rr * Cfg::OUT_ROW +
                                                                    (((byte >> 4) ^ (rr & 7)) << 4) + (byte & 15));
                            if (row0 + rr < args.M && n + col < args.N) y[col] = v;
                        }
                    }
                    __syncwarp();
                }
                if (lane == 0) bulk_commit_group();   // one group a chunk, empty where the warp copied
            }
        }
        cp_async_wait<0>();
        if (lane == 0) bulk_wait_group_all();
    }

    tc_fence_before();
    __syncwarp();
    cluster_sync();   // no CTA leaves while its pair may still signal or read it
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, Cfg::TMEM_COLS);
    }
}

template <int OUT>
cudaError_t launch_pair(const GemmFp8Args& a, int num_sms, cudaStream_t stream) {
    using Cfg = PairCfg8;
    constexpr int ELEM = OUT == kF32 ? 4 : OUT == kE4M3 ? 1 : 2;
    constexpr CUtensorMapDataType DT = OUT == kF32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                       : OUT == kE4M3 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                       : OUT == kF16  ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                      : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    CUtensorMap tx, tw;
    if (!make_tmap_rows(&tx, a.x, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.K, a.M, a.x_stride, kStageRow, kTileM) ||
        !make_tmap_rows(&tw, a.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.K, a.N, a.w_stride, kStageRow, kTileM))
        return cudaErrorInvalidValue;
    CUtensorMap ty = tx;
    if (a.vec && !make_tmap_rows(&ty, a.y, DT, a.N, a.M, uint64_t(a.y_stride) * ELEM, Cfg::OUT_ROW / ELEM, 32))
        return cudaErrorInvalidValue;
    const int64_t tiles = (int64_t(a.M) + 2 * kTileM - 1) / (2 * kTileM) * ((int64_t(a.N) + Cfg::BN - 1) / Cfg::BN);
    if (tiles > (1 << 30)) return cudaErrorInvalidValue;
    const int pairs = int(tiles < num_sms / 2 ? tiles : num_sms / 2);
    return launch_on(gemm_fp8_pair_kernel<OUT>, 2 * pairs, Cfg::THREADS, Cfg::SMEM, stream, tx, tw, ty, a);
}

// Up to 32 rows the narrow tiles.  Above, what takes less by the two kernels'
// measured steps: a 128 x 64 tile's CTA takes about 0.6 us a group after 5.5 us
// of set-up and joining, a 256 x 256 tile's pair 0.42 us after 6.5 us.  (us,
// tiles against pairs: 201 x 1024 x 4736 11.2 / 22.5, 400 x 1024 x 1024 8.5 /
// 9.9, 201 x 4736 x 1024 11.5 / 9.6, 1600 x 1024 x 4736 36.9 / 22.9, 201 x 8192
// x 8192 58 / 35.)
template <int OUT>
cudaError_t launch_out(const GemmFp8Args& a, int num_sms, cudaStream_t stream) {
    if (a.M <= 16) return launch_tile<16, OUT>(a, num_sms, stream);
    if (a.M <= 32) return launch_tile<32, OUT>(a, num_sms, stream);
    const int64_t groups = groups_of(a.K);
    const int64_t tiles = tiles_of(a.M, a.N, 64, kTileM), pairs = tiles_of(a.M, a.N, 2 * kTileM, PairCfg8::BN);
    const int splits = tile_splits(tiles, int(groups), num_sms);
    const int64_t rounds = (tiles * splits + num_sms - 1) / num_sms, waves = (pairs + num_sms / 2 - 1) / (num_sms / 2);
    const int64_t tile_time = 550 + 60 * rounds * ((groups + splits - 1) / splits), pair_time = 650 + 42 * waves * groups;
    if (tile_time <= pair_time) return launch_tile<64, OUT>(a, num_sms, stream);
    return launch_pair<OUT>(a, num_sms, stream);
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
    return cudaFuncSetAttribute(gemm_fp8_pair_kernel<OUT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                int(PairCfg8::SMEM));
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
