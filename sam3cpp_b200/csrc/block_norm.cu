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
// row stays in registers between the two norms.  A chunk is 256 columns, two
// groups of 128, four consecutive columns of each per lane (so that every
// access of a warp is contiguous and a scale group's maximum is one warp
// reduction); warp w of a row's team holds CPW consecutive chunks.
//
// Many rows (STREAM): persistent CTAs, up to four chunks a warp, so that a
// reduction or a barrier is paid once for 32 columns a lane; the vectors wait in
// shared memory (the branch's scales folded into the post-norm's: one multiply
// less a value) and the next row comes there by bulk copies while the second
// half of a row is computed.  82944 x 1024, LayerNorm twice, gate, e4m3 out:
// 155-162 us, 5.8-6.0 TB/s with 16 warps an SM and one row ahead (12 warps and
// two rows: 174 us, 20 warps of fewer registers: 168 us); in runs of seconds
// under the 1 kW cap 172 us, where instructions count (178 us with 5% more).
// Whole rows per warp read straight into registers took 398 us (the loads'
// latency), one chunk a warp with the next row in registers 269 us (four times
// the reductions).
// Few rows: one chunk a warp up to 4096 columns, everything asked for at once,
// for the latency of one row; up to 32 warps of one or two chunks above (2 x
// 16384: 6.7 us, with 16 warps of four chunks 7.8 us; 4 x 6791 7.6 and 11.6 us).
//
// Up to 256 columns: eight a lane, several rows a warp (norm_narrow_kernel).
//
// A LayerNorm warp reduces its own mean and centred square sum and the warps'
// are merged about the row's mean (Chan, Golub and LeVeque, 1979), so there is
// one exchange per norm and no cancellation.
#include "elements.cuh"
#include "fp8.cuh"
#include "kernels.h"

#include <type_traits>

namespace s3t {

namespace {

constexpr int kChunk = 2 * kScaleBlock;
constexpr int kMaxWarps = 16;          // of a row whose vectors stay in registers; twice as many where they do not
constexpr int kSlots = 1;              // rows ahead of a warp (STREAM)
constexpr int kStreamWarps = 16;
constexpr int kNarrowThreads = 256;
constexpr int kStreamBytes = 200 * 1024;
constexpr int kVectors = 5;            // post weight and bias, branch factor, pre weight and bias
constexpr int kStreamVectors = 4;      // the branch factor folded into the first two

// A lane's eight elements of a chunk are two quads: quad h is columns
// h * 128 + 4 lane .. + 3 (VEC: whole or not there at all), or h * 128 + lane +
// 32 i where rows are not aligned.
template <bool VEC>
S3T_DEV int quad_col(int lane, int h, int i) {
    return h * kScaleBlock + (VEC ? lane * 4 + i : lane + 32 * i);
}

template <typename T>
S3T_DEV void widen4(const T* p, float2& a, float2& b) {
    if constexpr (sizeof(T) == 4) {
        const float4 v = *reinterpret_cast<const float4*>(p);
        a = make_float2(v.x, v.y);
        b = make_float2(v.z, v.w);
    } else {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        a = unpack2(v.x, T());
        b = unpack2(v.y, T());
    }
}

// A lane's elements of the chunk at p (columns c0 ..), zeros past dim.
template <bool VEC, typename T>
S3T_DEV void load_chunk(const T* p, int c0, int dim, int lane, float2 (&v)[4]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if constexpr (VEC) {
            const int c = c0 + quad_col<true>(lane, h, 0);
            if (c < dim) widen4(p + c, v[2 * h], v[2 * h + 1]);
            else v[2 * h] = v[2 * h + 1] = make_float2(0.f, 0.f);
        } else {
            float f[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = c0 + quad_col<false>(lane, h, i);
                f[i] = c < dim ? to_float(p[c]) : 0.f;
            }
            v[2 * h] = make_float2(f[0], f[1]);
            v[2 * h + 1] = make_float2(f[2], f[3]);
        }
    }
}

template <bool VEC, typename T>
S3T_DEV void store_chunk(T* p, int c0, int dim, int lane, const float2 (&v)[4]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const float2 a = v[2 * h], b = v[2 * h + 1];
        if constexpr (VEC) {
            const int c = c0 + quad_col<true>(lane, h, 0);
            if (c >= dim) continue;
            if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(p + c) = make_float4(a.x, a.y, b.x, b.y);
            else *reinterpret_cast<uint2*>(p + c) = make_uint2(pack2(a.x, a.y, T()), pack2(b.x, b.y, T()));
        } else {
            const float f[4] = {a.x, a.y, b.x, b.y};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = c0 + quad_col<false>(lane, h, i);
                if (c < dim) p[c] = from_float<T>(f[i]);
            }
        }
    }
}

// Element k of vector p: `otherwise` where there is none, 0 past the last
// column (so that columns past dim add nothing to x' and u).
template <bool VEC>
S3T_DEV void load_vector(const float* p, float otherwise, int c0, int dim, int lane, float2 (&v)[4]) {
    if (p) {
        load_chunk<VEC>(p, c0, dim, lane, v);
    } else {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                v[2 * h + i].x = c0 + quad_col<VEC>(lane, h, 2 * i) < dim ? otherwise : 0.f;
                v[2 * h + i].y = c0 + quad_col<VEC>(lane, h, 2 * i + 1) < dim ? otherwise : 0.f;
            }
    }
}

S3T_DEV float2 both(float v) { return make_float2(v, v); }

S3T_DEV float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

struct RowStats {
    float mean, rstd;
};

// How a row lies on the warps of its team: warp w holds the columns from
// w * CPW * kChunk on, all of them full but the last warp's.
struct Split {
    int lane, warp, warps, team;
    int last;                         // columns of the last warp
    float inv_dim, inv_last;
};

// Barrier of one team's warps (named barrier 1 + team; teams of more than one
// warp are at most eight a CTA).
S3T_DEV void team_sync(const Split& sp) {
    asm volatile("bar.sync %0, %1;" ::"r"(sp.team + 1), "r"(sp.warps * 32) : "memory");
}

// Mean (0 for RMSNorm) and 1 / sqrt(mean square or variance + eps) of a row of
// which this warp holds v, zeros past dim.
template <int CPW, bool VEC>
S3T_DEV RowStats row_stats(const float2 (&v)[CPW][4], int layer, int dim, float eps, const Split& sp, float2* exchange) {
    constexpr float kFull = float(CPW * kChunk);
    float sum = 0.f, mean = 0.f;
    if (layer) {
        float2 t = v[0][0];
#pragma unroll
        for (int j = 0; j < CPW; ++j)
#pragma unroll
            for (int i = j == 0 ? 1 : 0; i < 4; ++i) t = __fadd2_rn(t, v[j][i]);
        sum = warp_sum(t.x + t.y);
        mean = sum * (sp.warp + 1 == sp.warps ? sp.inv_last : 1.f / kFull);
    }
    float2 q = both(0.f);
    const float2 minus = both(-mean);
#pragma unroll
    for (int j = 0; j < CPW; ++j) {
        const int c0 = (sp.warp * CPW + j) * kChunk;
        if (!layer || c0 + kChunk <= dim) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 d = __fadd2_rn(v[j][i], minus);
                q = __ffma2_rn(d, d, q);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float2 d = __fadd2_rn(v[j][i], minus);
                if (c0 + quad_col<VEC>(sp.lane, i / 2, 2 * (i & 1)) >= dim) d.x = 0.f;
                if (c0 + quad_col<VEC>(sp.lane, i / 2, 2 * (i & 1) + 1) >= dim) d.y = 0.f;
                q = __ffma2_rn(d, d, q);
            }
        }
    }
    float m2 = warp_sum(q.x + q.y);
    if (sp.warps > 1) {
        if (sp.lane == 0) exchange[sp.warp] = make_float2(sum, m2);
        team_sync(sp);
        // Every warp merges all partials in the same order: the squares about
        // the row's mean are those about each warp's plus the means' spread.
        float total = 0.f;
        m2 = 0.f;
#pragma unroll 4
        for (int w = 0; w < sp.warps; ++w) {
            const float2 e = exchange[w];
            total += e.x;
            m2 += e.y;
        }
        if (layer) {
            mean = total * sp.inv_dim;
#pragma unroll 4
            for (int w = 0; w + 1 < sp.warps; ++w) {
                const float d = fmaf(exchange[w].x, 1.f / kFull, -mean);
                m2 = fmaf(d * kFull, d, m2);
            }
            const float d = fmaf(exchange[sp.warps - 1].x, sp.inv_last, -mean);
            m2 = fmaf(d * float(sp.last), d, m2);
        }
    }
    return {mean, rsqrtf(fmaf(m2, sp.inv_dim, eps))};
}

// v = (v - mean) rstd w + b
S3T_DEV void normalize(float2 (&v)[4], RowStats st, const float2 (&w)[4], const float2 (&b)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        v[i] = __ffma2_rn(__fmul2_rn(__fadd2_rn(v[i], both(-st.mean)), both(st.rstd)), w[i], b[i]);
}

S3T_DEV void apply_gate(float2 (&h)[4], float2 (&g)[4], int act) {
    if (act == kGateSigmoid) {
#pragma unroll
        for (int i = 0; i < 4; ++i) g[i] = make_float2(1.f / (1.f + expf(-g[i].x)), 1.f / (1.f + expf(-g[i].y)));
    } else if (act == kGateTanh) {
#pragma unroll
        for (int i = 0; i < 4; ++i) g[i] = make_float2(tanhf(g[i].x), tanhf(g[i].y));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __fmul2_rn(h[i], g[i]);
}

// u of this warp's chunks in 8 bits, with the scales of their groups.
template <int CPW, bool VEC>
S3T_DEV void store_eight(const NormResidualArgs& a, uint32_t row, int c0, int lane, float2 (&v)[CPW][4]) {
    // Columns past dim are zeros: their weights are.
    uint32_t peak[2 * CPW];
#pragma unroll
    for (int k = 0; k < 2 * CPW; ++k) {
        const float2 p = v[k / 2][2 * (k & 1)], q = v[k / 2][2 * (k & 1) + 1];
        // The bits of magnitudes order like them, NaN above all (and kept by absmax3_nan).
        peak[k] = __reduce_max_sync(0xffffffffu, abs_bits(absmax3_nan(absmax3_nan(p.x, p.y, q.x), q.y, q.y)));
    }
    // Lane 2 k divides for group k's scale, lane 2 k + 1 for its inverse.
    uint32_t pick = peak[0];
#pragma unroll
    for (int k = 1; k < 2 * CPW; ++k)
        if ((lane >> 1) == k) pick = peak[k];
    const float top = __uint_as_float(max(pick, kAmaxFloorBits));
    const bool odd = lane & 1;
    const float quotient = __fdiv_rn(odd ? kE4M3Max : top, odd ? top : kE4M3Max);
    uint8_t* q = static_cast<uint8_t*>(a.u) + int64_t(row) * a.u_stride;
#pragma unroll
    for (int k = 0; k < 2 * CPW; ++k) {
        const float2 inv = both(__shfl_sync(0xffffffffu, quotient, 2 * k + 1));
        const float2 s = __fmul2_rn(v[k / 2][2 * (k & 1)], inv), t = __fmul2_rn(v[k / 2][2 * (k & 1) + 1], inv);
        const uint32_t codes = pack_e4m3x4(s.x, s.y, t.x, t.y);
        const int base = c0 + (k / 2) * kChunk;
        if constexpr (VEC) {
            const int c = base + quad_col<true>(lane, k & 1, 0);
            if (c < a.dim) *reinterpret_cast<uint32_t*>(q + c) = codes;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = base + quad_col<false>(lane, k & 1, i);
                if (c < a.dim) q[c] = uint8_t(codes >> (8 * i));
            }
        }
    }
    const int g = c0 + (lane >> 1) * kScaleBlock;
    if (!odd && lane < 4 * CPW && g < a.dim) a.u_scale[int64_t(g / kScaleBlock) * a.u_scale_stride + row] = quotient;
}

// Few rows: a team of blockDim.x / 32 warps takes one row, blockDim.y teams a CTA.
// KEEP: the vectors fit registers and are asked for with the row.
template <typename T, typename R, int CPW, bool KEEP, bool VEC>
__global__ void __launch_bounds__(32 * (KEEP ? kMaxWarps : 2 * kMaxWarps)) norm_rows_kernel(const NormResidualArgs a) {
    __shared__ float2 exchange[4][2][2 * kMaxWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, team = threadIdx.y;
    const int dim = a.dim, last = dim - (warps - 1) * CPW * kChunk;
    const Split sp{lane, warp, warps, team, last, 1.f / float(dim), 1.f / float(last)};
    const uint32_t row = blockIdx.x * blockDim.y + team;
    if (row >= uint32_t(a.rows)) return;   // a whole team: no barrier is shared between teams
    const int c0 = warp * CPW * kChunk;
    float2 x[CPW][4], h[CPW][4], g[CPW][4], vec[kVectors][4];
    auto vectors = [&](int k, const float* p, float otherwise, int j) {
        load_vector<VEC>(p, otherwise, c0 + j * kChunk, dim, lane, vec[k]);
    };
#pragma unroll
    for (int j = 0; j < CPW; ++j) {
        load_chunk<VEC>(static_cast<const R*>(a.x) + int64_t(row) * a.x_stride, c0 + j * kChunk, dim, lane, x[j]);
        if (a.y) load_chunk<VEC>(static_cast<const T*>(a.y) + int64_t(row) * a.y_stride, c0 + j * kChunk, dim, lane, h[j]);
        if (KEEP && a.gate)
            load_chunk<VEC>(static_cast<const T*>(a.gate) + int64_t(row / uint32_t(a.gate_rows)) * a.gate_stride,
                            c0 + j * kChunk, dim, lane, g[j]);
    }
    if (KEEP) {
        vectors(0, a.post_weight, 1.f, 0);
        vectors(1, a.post_bias, 0.f, 0);
        vectors(2, a.channel, 1.f, 0);
        vectors(3, a.pre_weight, 1.f, 0);
        vectors(4, a.pre_bias, 0.f, 0);
    }
    RowStats st{0.f, 1.f};
    if (a.post) st = row_stats<CPW, VEC>(h, a.layer, dim, a.eps, sp, exchange[team][0]);
#pragma unroll
    for (int j = 0; j < CPW; ++j) {
        if (a.post) {
            if (!KEEP) {
                vectors(0, a.post_weight, 1.f, j);
                vectors(1, a.post_bias, 0.f, j);
            }
            normalize(h[j], st, vec[0], vec[1]);
        }
        if (a.gate) {
            if (!KEEP)
                load_chunk<VEC>(static_cast<const T*>(a.gate) + int64_t(row / uint32_t(a.gate_rows)) * a.gate_stride,
                                c0 + j * kChunk, dim, lane, g[j]);
            apply_gate(h[j], g[j], a.gate_act);
        }
        if (!KEEP) vectors(2, a.channel, 1.f, j);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[j][i] = __fmul2_rn(x[j][i], both(a.resid_scale));
            if (a.y) x[j][i] = __ffma2_rn(__fmul2_rn(vec[2][i], both(a.branch_scale)), h[j][i], x[j][i]);
        }
        if (a.x_out)
            store_chunk<VEC>(static_cast<R*>(a.x_out) + int64_t(row) * a.x_out_stride, c0 + j * kChunk, dim, lane, x[j]);
    }
    if (!a.u) return;
    st = row_stats<CPW, VEC>(x, a.layer, dim, a.eps, sp, exchange[team][1]);
#pragma unroll
    for (int j = 0; j < CPW; ++j) {
        if (!KEEP) {
            vectors(3, a.pre_weight, 1.f, j);
            vectors(4, a.pre_bias, 0.f, j);
        }
        normalize(x[j], st, vec[3], vec[4]);
        if (!a.u_eight)
            store_chunk<VEC>(static_cast<T*>(a.u) + int64_t(row) * a.u_stride, c0 + j * kChunk, dim, lane, x[j]);
    }
    if (a.u_eight) store_eight<CPW, VEC>(a, row, c0, lane, x);
}

// Shared memory of a streaming CTA: the vectors that the call has, each a row of
// floats padded to its team's columns; then per warp kSlots rows of its columns
// of x, y and gate, as far as there are; then the barriers.
template <typename T, typename R, int CPW>
struct StreamRow {
    static constexpr uint32_t COLS = CPW * kChunk;
    static constexpr uint32_t X = COLS * sizeof(R) + 16, Y = COLS * sizeof(T) + 16;   // and what lies around them
};
// Vector k: post weight and post bias with the branch's scales, pre weight, pre bias.
__host__ __device__ inline bool has_vector(const NormResidualArgs& a, int k) {
    return k == 0 ? a.y != nullptr : k == 1 ? a.post && a.post_bias : k == 2 ? a.u != nullptr : a.u && a.pre_bias;
}
template <typename Row>
__host__ __device__ uint32_t row_bytes(const NormResidualArgs& a) {
    return Row::X + (a.y ? Row::Y : 0) + (a.gate ? Row::Y : 0);
}

// The 16-byte units that hold `bytes` bytes from p on.
S3T_DEV uint32_t units_around(const void* p, uint32_t bytes) {
    return ((uint32_t(reinterpret_cast<uintptr_t>(p)) & 15) + bytes + 15) & ~15u;
}
S3T_DEV void bulk_load_around(uint8_t* to, const void* p, uint32_t bytes, uint64_t* bar) {
    bulk_load(to, reinterpret_cast<const void*>(reinterpret_cast<uintptr_t>(p) & ~uintptr_t(15)), units_around(p, bytes), bar);
}

// VEC: rows and columns in whole 16-byte units; else the units around a row
// come, and a lane picks its elements from where the row begins in them.
template <typename T, typename R, int CPW, bool VEC>
__global__ void __launch_bounds__(32 * kStreamWarps, 1) norm_stream_kernel(const NormResidualArgs a) {
    using Row = StreamRow<T, R, CPW>;
    // Two parities: a slot is written again two barriers after its last read.
    __shared__ float2 exchange[kStreamWarps][2][2][kStreamWarps];
    __shared__ uint64_t arrived[kStreamWarps][kSlots];
    extern __shared__ uint4 words[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, team = threadIdx.y;
    const int thread = threadIdx.y * blockDim.x + threadIdx.x, threads = blockDim.x * blockDim.y;
    const int dim = a.dim, last = dim - (warps - 1) * int(Row::COLS), padded = warps * int(Row::COLS);
    const Split sp{lane, warp, warps, team, last, 1.f / float(dim), 1.f / float(last)};
    const int c0 = warp * int(Row::COLS), cols = warp + 1 == warps ? last : int(Row::COLS);
    float* const vec0 = reinterpret_cast<float*>(words);
    float* const vec1 = vec0 + (has_vector(a, 0) ? padded : 0);
    float* const vec2 = vec1 + (has_vector(a, 1) ? padded : 0);
    float* const vec3 = vec2 + (has_vector(a, 2) ? padded : 0);
    uint8_t* const buffers = reinterpret_cast<uint8_t*>(vec3 + (has_vector(a, 3) ? padded : 0));
    for (int c = thread; c < padded; c += threads) {   // 0 past dim
        const bool in = c < dim;
        if (has_vector(a, 0)) {
            const float s = in ? a.branch_scale * (a.channel ? a.channel[c] : 1.f) : 0.f;
            vec0[c] = a.post && a.post_weight && in ? a.post_weight[c] * s : s;
            if (has_vector(a, 1)) vec1[c] = in ? a.post_bias[c] * s : 0.f;
        }
        if (has_vector(a, 2)) vec2[c] = in ? (a.pre_weight ? a.pre_weight[c] : 1.f) : 0.f;
        if (has_vector(a, 3)) vec3[c] = in ? a.pre_bias[c] : 0.f;
    }
    const uint32_t bytes = row_bytes<Row>(a);
    // VEC: columns past dim are never copied, they stay zeros.
    uint8_t* mine = buffers + (team * warps + warp) * kSlots * bytes;
    for (uint32_t i = lane; i < kSlots * bytes / 16; i += 32) reinterpret_cast<uint4*>(mine)[i] = make_uint4(0, 0, 0, 0);
    uint64_t* bar = arrived[team * warps + warp];
    if (lane == 0) {
        for (int i = 0; i < kSlots; ++i) mbar_init(bar + i, 1);
        fence_barrier_init();
    }
    fence_proxy_async_smem();
    __syncthreads();

    const uint32_t rows = uint32_t(a.rows), stride = gridDim.x * blockDim.y;
    uint32_t row = blockIdx.x * blockDim.y + team;
    const R* xp = static_cast<const R*>(a.x) + int64_t(row) * a.x_stride + c0;
    const T* yp = static_cast<const T*>(a.y) + int64_t(row) * a.y_stride + c0;
    R* xo = static_cast<R*>(a.x_out) + int64_t(row) * a.x_out_stride + c0;
    const int64_t x_step = int64_t(stride) * a.x_stride, y_step = int64_t(stride) * a.y_stride,
                  xo_step = int64_t(stride) * a.x_out_stride;
    uint32_t ahead = row;
    auto fetch = [&](int slot) {       // one lane
        if (ahead >= rows) return;
        uint8_t* to = mine + slot * bytes;
        const uint32_t xb = uint32_t(cols) * sizeof(R), tb = uint32_t(cols) * sizeof(T);
        const T* gp = static_cast<const T*>(a.gate);
        if (a.gate) gp += int64_t(ahead / uint32_t(a.gate_rows)) * a.gate_stride + c0;
        if constexpr (VEC) {
            mbar_arrive_expect_tx(bar + slot, xb + (a.y ? tb : 0) + (a.gate ? tb : 0));
            if (a.y) bulk_load(to + Row::X, yp, tb, bar + slot);
            bulk_load(to, xp, xb, bar + slot);
            if (a.gate) bulk_load(to + Row::X + Row::Y, gp, tb, bar + slot);
        } else {
            mbar_arrive_expect_tx(bar + slot, units_around(xp, xb) + (a.y ? units_around(yp, tb) : 0) +
                                                  (a.gate ? units_around(gp, tb) : 0));
            if (a.y) bulk_load_around(to + Row::X, yp, tb, bar + slot);
            bulk_load_around(to, xp, xb, bar + slot);
            if (a.gate) bulk_load_around(to + Row::X + Row::Y, gp, tb, bar + slot);
        }
        xp += x_step;
        yp += y_step;
        ahead = rows - ahead > stride ? ahead + stride : rows;
    };
    if (lane == 0)
        for (int i = 0; i < kSlots; ++i) fetch(i);
    const bool whole = c0 + int(Row::COLS) <= dim;      // no column of this warp lies past dim
    bool lost = false;
    for (uint32_t it = 0; row < rows; ++it) {
        const int slot = int(it % kSlots);
        // A row that never came is reported and no more are asked for; the loop
        // goes on without waiting, so that no warp of the team is left alone at a
        // barrier, and the copy has a second limit's time before the CTA may end.
        if (!lost && !mbar_wait(bar + slot, (it / kSlots) & 1, a.status, kErrTimeoutProducer, nullptr)) {
            lost = true;
            mbar_wait(bar + slot, (it / kSlots) & 1, a.status, kErrTimeoutDrain, nullptr);
        }
        const uint8_t* from = mine + slot * bytes;
        float2 x[CPW][4], h[CPW][4];
        auto vector = [&](const float* p, int j, float2(&v)[4]) { load_chunk<VEC>(p + c0 + j * kChunk, 0, kChunk, lane, v); };
        auto bias = [&](const float* p, bool there, int j, float2(&v)[4]) {
            if (there) {
                vector(p, j, v);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = both(0.f);
            }
        };
        // Chunk j of a row whose units lie at p and which begins where `at` says.
        auto chunk = [&](const uint8_t* p, auto* at, int j, float2(&v)[4]) {
            using E = typename std::remove_const<typename std::remove_pointer<decltype(at)>::type>::type;
            if constexpr (VEC) load_chunk<true>(reinterpret_cast<const E*>(p) + j * kChunk, 0, kChunk, lane, v);
            else load_chunk<false>(reinterpret_cast<const E*>(p + (reinterpret_cast<uintptr_t>(at) & 15)), j * kChunk, cols, lane, v);
        };
        if (a.y) {
#pragma unroll
            for (int j = 0; j < CPW; ++j)
                chunk(from + Row::X, static_cast<const T*>(a.y) + int64_t(row) * a.y_stride + c0, j, h[j]);
            if (a.post) {
                const RowStats st = row_stats<CPW, VEC>(h, a.layer, dim, a.eps, sp, exchange[team][it & 1][0]);
#pragma unroll
                for (int j = 0; j < CPW; ++j) {
                    float2 w[4], b[4];
                    vector(vec0, j, w);
                    bias(vec1, has_vector(a, 1), j, b);
                    normalize(h[j], st, w, b);
                }
            } else {
#pragma unroll
                for (int j = 0; j < CPW; ++j) {
                    float2 w[4];
                    vector(vec0, j, w);
#pragma unroll
                    for (int i = 0; i < 4; ++i) h[j][i] = __fmul2_rn(h[j][i], w[i]);
                }
            }
            if (a.gate) {
#pragma unroll
                for (int j = 0; j < CPW; ++j) {
                    float2 g[4];
                    chunk(from + Row::X + Row::Y,
                          static_cast<const T*>(a.gate) + int64_t(row / uint32_t(a.gate_rows)) * a.gate_stride + c0, j, g);
                    apply_gate(h[j], g, a.gate_act);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < CPW; ++j) {
            chunk(from, static_cast<const R*>(a.x) + int64_t(row) * a.x_stride + c0, j, x[j]);
            if (a.y) {
#pragma unroll
                for (int i = 0; i < 4; ++i) x[j][i] = __ffma2_rn(both(a.resid_scale), x[j][i], h[j][i]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) x[j][i] = __fmul2_rn(both(a.resid_scale), x[j][i]);
            }
        }
        __syncwarp();
        if (lane == 0 && !lost) fetch(slot);   // every lane has read the slot
        if (a.x_out) {
#pragma unroll
            for (int j = 0; j < CPW; ++j) {
                if (whole) store_chunk<VEC>(xo + j * kChunk, 0, kChunk, lane, x[j]);
                else store_chunk<VEC>(xo, j * kChunk, cols, lane, x[j]);
            }
        }
        if (a.u) {
            const RowStats st = row_stats<CPW, VEC>(x, a.layer, dim, a.eps, sp, exchange[team][it & 1][1]);
#pragma unroll
            for (int j = 0; j < CPW; ++j) {
                float2 w[4], b[4];
                vector(vec2, j, w);
                bias(vec3, has_vector(a, 3), j, b);
                normalize(x[j], st, w, b);
                if (!a.u_eight)
                    store_chunk<VEC>(static_cast<T*>(a.u) + int64_t(row) * a.u_stride, c0 + j * kChunk, dim, lane, x[j]);
            }
            if (a.u_eight) store_eight<CPW, VEC>(a, row, c0, lane, x);
        }
        xo += xo_step;
        row = rows - row > stride ? row + stride : rows;
    }
}

// ------------------------------------------------------- rows up to 256 ---

// Columns of element i of a lane's eight, LANES lanes a row; 16 lanes hold a
// group of 128.
template <int LANES, bool VEC>
S3T_DEV int narrow_col(int l, int i) {
    if constexpr (VEC) return l * 8 + i;
    else if constexpr (LANES <= 16) return l + LANES * i;
    else return (l / 16) * kScaleBlock + l % 16 + 16 * i;
}

// A lane's elements as they lie in memory: widened where they are used, since
// a conversion would wait for the load.
template <typename T>
struct alignas(16) NarrowRaw {
    T e[8];
};

template <int LANES, bool VEC, typename T>
S3T_DEV void narrow_load(const T* p, int dim, int l, bool there, NarrowRaw<T>& v) {
    if constexpr (VEC) {
        uint4 u[sizeof(T) / 2];
#pragma unroll
        for (int i = 0; i < int(sizeof(T)) / 2; ++i)
            u[i] = there && l * 8 < dim ? reinterpret_cast<const uint4*>(p + l * 8)[i] : make_uint4(0, 0, 0, 0);
        memcpy(v.e, u, sizeof(u));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int c = narrow_col<LANES, false>(l, i);
            v.e[i] = there && c < dim ? p[c] : from_float<T>(0.f);
        }
    }
}

template <typename T>
S3T_DEV void narrow_widen(const NarrowRaw<T>& r, float2 (&v)[4]) {
    widen4(r.e, v[0], v[1]);
    widen4(r.e + 4, v[2], v[3]);
}

template <int LANES, bool VEC, typename T>
S3T_DEV void narrow_store(T* p, int dim, int l, const float2 (&v)[4]) {
    if constexpr (VEC) {
        if (l * 8 >= dim) return;
        if constexpr (sizeof(T) == 4) {
            reinterpret_cast<float4*>(p + l * 8)[0] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
            reinterpret_cast<float4*>(p + l * 8)[1] = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
        } else {
            *reinterpret_cast<uint4*>(p + l * 8) = make_uint4(pack2(v[0].x, v[0].y, T()), pack2(v[1].x, v[1].y, T()),
                                                              pack2(v[2].x, v[2].y, T()), pack2(v[3].x, v[3].y, T()));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int c = narrow_col<LANES, false>(l, i);
            if (c < dim) p[c] = from_float<T>(i & 1 ? v[i / 2].y : v[i / 2].x);
        }
    }
}

template <int LANES>
S3T_DEV float lanes_sum(float v) {
#pragma unroll
    for (int o = LANES / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <int LANES, bool VEC>
S3T_DEV RowStats narrow_stats(const float2 (&v)[4], int layer, int dim, float inv_dim, float eps, int l) {
    float mean = 0.f;
    if (layer) {
        const float2 t = __fadd2_rn(__fadd2_rn(v[0], v[1]), __fadd2_rn(v[2], v[3]));
        mean = lanes_sum<LANES>(t.x + t.y) * inv_dim;
    }
    float2 q = both(0.f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float2 d = __fadd2_rn(v[i], both(-mean));
        if (narrow_col<LANES, VEC>(l, 2 * i) >= dim) d.x = 0.f;
        if (narrow_col<LANES, VEC>(l, 2 * i + 1) >= dim) d.y = 0.f;
        q = __ffma2_rn(d, d, q);
    }
    return {mean, rsqrtf(fmaf(lanes_sum<LANES>(q.x + q.y), inv_dim, eps))};
}

// A lane's elements of vector p: `otherwise` where there is none, 0 past dim.
template <int LANES, bool VEC>
S3T_DEV void narrow_vector(const float* p, float otherwise, int dim, int l, float2 (&v)[4]) {
    if (p) {
        NarrowRaw<float> raw;
        narrow_load<LANES, VEC>(p, dim, l, true, raw);
        narrow_widen(raw, v);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i].x = narrow_col<LANES, VEC>(l, 2 * i) < dim ? otherwise : 0.f;
            v[i].y = narrow_col<LANES, VEC>(l, 2 * i + 1) < dim ? otherwise : 0.f;
        }
    }
}

// Rows of up to 8 LANES columns (heads, mostly): LANES lanes a row, so that no
// lane idles, and the vectors in registers for all of a thread's rows.  82944
// rows, fp16, LayerNorm twice: 128 columns 24 us (a warp a row, streamed: 49
// us), 64 columns 14 us (48 us), 7 columns 6.3 us (58 us); 400000 x 128 86 us,
// 4.8 TB/s, with the next row on its way (119 us without, bound by the loads'
// latency at three CTAs an SM).
template <typename T, typename R, int LANES, bool VEC>
__global__ void __launch_bounds__(kNarrowThreads, 3) norm_narrow_kernel(const NormResidualArgs a) {
    const int l = threadIdx.x % LANES, dim = a.dim;
    const float inv_dim = 1.f / float(dim);
    const uint32_t rows = uint32_t(a.rows), stride = gridDim.x * (kNarrowThreads / LANES);
    const uint32_t in_warp = (threadIdx.x & 31) / LANES;
    NarrowRaw<R> raw_x;
    NarrowRaw<T> raw_y, raw_g;
    auto load_x = [&](uint32_t row) {
        narrow_load<LANES, VEC>(static_cast<const R*>(a.x) + int64_t(row) * a.x_stride, dim, l, row < rows, raw_x);
    };
    auto load_branch = [&](uint32_t row) {
        const bool there = row < rows;
        if (a.y) narrow_load<LANES, VEC>(static_cast<const T*>(a.y) + int64_t(row) * a.y_stride, dim, l, there, raw_y);
        if (a.gate)
            narrow_load<LANES, VEC>(static_cast<const T*>(a.gate) + int64_t(row / uint32_t(a.gate_rows)) * a.gate_stride, dim, l,
                                    there, raw_g);
    };
    // The loop's bound is the warp's, for the shuffles.  The first row is asked
    // for before the vectors: a call of a few rows is all latency.
    uint32_t first = blockIdx.x * (kNarrowThreads / LANES) + (threadIdx.x & ~31u) / LANES;
    load_branch(first + in_warp);
    load_x(first + in_warp);
    // As the streaming kernel's: the branch's scales folded in, 0 past dim.
    float2 post_w[4], post_b[4], pre_w[4], pre_b[4];
    {
        float2 ch[4];
        narrow_vector<LANES, VEC>(a.channel, 1.f, dim, l, ch);
        narrow_vector<LANES, VEC>(a.post ? a.post_weight : nullptr, 1.f, dim, l, post_w);
        narrow_vector<LANES, VEC>(a.post ? a.post_bias : nullptr, 0.f, dim, l, post_b);
        narrow_vector<LANES, VEC>(a.pre_weight, 1.f, dim, l, pre_w);
        narrow_vector<LANES, VEC>(a.pre_bias, 0.f, dim, l, pre_b);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            ch[i] = __fmul2_rn(ch[i], both(a.branch_scale));
            post_w[i] = __fmul2_rn(post_w[i], ch[i]);
            post_b[i] = __fmul2_rn(post_b[i], ch[i]);
        }
    }
    // The next row comes while this row's pre-norm runs.
    while (first < rows) {
        const uint32_t row = first + in_warp;
        const bool there = row < rows;
        first = rows - first > stride ? first + stride : rows;
        float2 x[4], h[4];
        if (a.y) {
            narrow_widen(raw_y, h);
            if (a.post) {
                normalize(h, narrow_stats<LANES, VEC>(h, a.layer, dim, inv_dim, a.eps, l), post_w, post_b);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) h[i] = __fmul2_rn(h[i], post_w[i]);
            }
            if (a.gate) {
                float2 g[4];
                narrow_widen(raw_g, g);
                apply_gate(h, g, a.gate_act);
            }
            narrow_widen(raw_x, x);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = __ffma2_rn(both(a.resid_scale), x[i], h[i]);
        } else {
            narrow_widen(raw_x, x);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = __fmul2_rn(both(a.resid_scale), x[i]);
        }
        if (first < rows) {
            load_branch(first + in_warp);
            load_x(first + in_warp);
        }
        if (a.x_out && there)
            narrow_store<LANES, VEC>(static_cast<R*>(a.x_out) + int64_t(row) * a.x_out_stride, dim, l, x);
        if (!a.u) continue;
        normalize(x, narrow_stats<LANES, VEC>(x, a.layer, dim, inv_dim, a.eps, l), pre_w, pre_b);
        if (!a.u_eight) {
            if (there) narrow_store<LANES, VEC>(static_cast<T*>(a.u) + int64_t(row) * a.u_stride, dim, l, x);
            continue;
        }
        // Columns past dim are zeros.
        constexpr int GROUP = LANES < 16 ? LANES : 16;       // lanes of a scale group
        uint32_t peak = abs_bits(absmax3_nan(absmax3_nan(absmax3_nan(x[0].x, x[0].y, x[1].x), x[1].y, x[2].x),
                                             absmax3_nan(x[2].y, x[3].x, x[3].y), 0.f));
#pragma unroll
        for (int o = GROUP / 2; o; o >>= 1) peak = max(peak, __shfl_xor_sync(0xffffffffu, peak, o));
        const float top = __uint_as_float(max(peak, kAmaxFloorBits));
        // Even lanes divide for the scale, odd ones for its inverse.
        const float quotient = __fdiv_rn(l & 1 ? kE4M3Max : top, l & 1 ? top : kE4M3Max);
        const float2 inv = both(__shfl_sync(0xffffffffu, quotient, 1, GROUP));
        float2 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __fmul2_rn(x[i], inv);
        const uint32_t lo = pack_e4m3x4(v[0].x, v[0].y, v[1].x, v[1].y), hi = pack_e4m3x4(v[2].x, v[2].y, v[3].x, v[3].y);
        if (!there) continue;
        uint8_t* q = static_cast<uint8_t*>(a.u) + int64_t(row) * a.u_stride;
        if constexpr (VEC) {
            if (l * 8 < dim) *reinterpret_cast<uint2*>(q + l * 8) = make_uint2(lo, hi);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int c = narrow_col<LANES, false>(l, i);
                if (c < dim) q[c] = uint8_t((i < 4 ? lo : hi) >> (8 * (i & 3)));
            }
        }
        if (l % GROUP == 0 && l * 8 < dim) a.u_scale[int64_t(l / 16) * a.u_scale_stride + row] = quotient;
    }
}

template <typename T, typename R, int LANES>
cudaError_t launch_narrow(const NormResidualArgs& a, int num_sms, cudaStream_t stream) {
    const int64_t ctas = (a.rows * LANES + kNarrowThreads - 1) / kNarrowThreads;
    const uint32_t grid = uint32_t(ctas < 3 * num_sms ? ctas : 3 * num_sms);
    if (a.vec) return launch_on(norm_narrow_kernel<T, R, LANES, true>, grid, kNarrowThreads, 0, stream, a);
    return launch_on(norm_narrow_kernel<T, R, LANES, false>, grid, kNarrowThreads, 0, stream, a);
}

template <typename T, typename R, int CPW, bool KEEP>
cudaError_t launch_few(const NormResidualArgs& a, cudaStream_t stream) {
    const int warps = (a.dim + CPW * kChunk - 1) / (CPW * kChunk);
    const int teams = warps == 1 ? 4 : 1;
    const int64_t ctas = (a.rows + teams - 1) / teams;
    const dim3 block(32 * warps, teams);
    if (a.vec) return launch_on(norm_rows_kernel<T, R, CPW, KEEP, true>, uint32_t(ctas), block, 0, stream, a);
    return launch_on(norm_rows_kernel<T, R, CPW, KEEP, false>, uint32_t(ctas), block, 0, stream, a);
}

// Rows a team from which the streaming kernel's set-up (the vectors' way into
// shared memory, 20 to 50 us for wide rows) is paid for.  Up to 4096 columns
// the other kernel keeps the vectors in registers and two rows do.  Above, it
// reads them again for every row, so two or three teams an SM win soon, a
// single one later, and later still with few vectors to read again or where
// five fp32 warps are all that hide a row's latency.  Measured where the two
// meet, post-norm and pre-norm, streamed / not, us:
//   2 teams, 4 vectors   f32 6144     at 2 rows 31 / 29, at 3 36 / 42
//   2 teams, 2 vectors   f32 8192     at 4 52 / 49, at 6 66 / 70; fp16 8192 at 3 38 / 33, at 6 48 / 60
//   1 team, 4 vectors    f32 7070     at 8 68 / 63, at 12 84 / 91; fp16 9024 at 8 65 / 60, at 12 79 / 87
//   1 team, 2 vectors    f32 9024     at 24 131 / 121, at 48 212 / 228
//                        fp16 10240   at 16 91 / 83, at 24 112 / 122; bf16 16384 at 12 92 / 91, at 16 106 / 119
//   5 warps of fp32      1 team, 4 vectors 5120 at 32 131 / 121, at 64 224 / 232; 3 teams, 2 vectors at 16
//                        117 / 114, at 32 212 / 219; 2 teams, 4 vectors 4352 at 5 33 / 31, at 15 73 / 90
template <typename T>
int stream_rounds(int teams, int warps, int vectors, int dim) {
    if (dim <= kMaxWarps * kChunk) return 2;
    const int rounds = teams > 1 ? (vectors > 2 ? 3 : 6) : vectors > 2 ? 10 : sizeof(T) == 4 ? 30 : 16;
    if (sizeof(T) == 2 || warps > 5) return rounds;
    return (teams > 1 && vectors > 2 ? 2 : 4) * rounds;
}

// The streaming kernel for rows of CPW chunks a warp; false: not for this call.
template <typename T, typename R, int CPW>
bool launch_stream(const NormResidualArgs& a, int num_sms, cudaStream_t stream, cudaError_t& e) {
    using Row = StreamRow<T, R, CPW>;
    const int warps = (a.dim + int(Row::COLS) - 1) / int(Row::COLS);
    int vectors = 0;
    for (int k = 0; k < kStreamVectors; ++k) vectors += has_vector(a, k);
    const int vector_bytes = vectors * warps * int(Row::COLS) * 4, team_bytes = warps * kSlots * int(row_bytes<Row>(a));
    int teams = vector_bytes < kStreamBytes ? (kStreamBytes - vector_bytes) / team_bytes : 0;
    if (teams > kStreamWarps / warps) teams = kStreamWarps / warps;
    if (teams == 0 || a.rows < int64_t(stream_rounds<T>(teams, warps, vectors, a.dim)) * num_sms * teams) return false;
    const dim3 block(32 * warps, teams);
    const uint32_t smem = uint32_t(vector_bytes + teams * team_bytes);
    e = a.vec ? launch_on(norm_stream_kernel<T, R, CPW, true>, num_sms, block, smem, stream, a)
              : launch_on(norm_stream_kernel<T, R, CPW, false>, num_sms, block, smem, stream, a);
    return true;
}

template <typename T, typename R>
cudaError_t launch_types(const NormResidualArgs& a, int num_sms, cudaStream_t stream) {
    if (a.dim <= 32) return launch_narrow<T, R, 4>(a, num_sms, stream);
    if (a.dim <= 64) return launch_narrow<T, R, 8>(a, num_sms, stream);
    if (a.dim <= 128) return launch_narrow<T, R, 16>(a, num_sms, stream);
    // A CTA of eight rows on every SM, a warp each: 82944 x 256 fp16 45 us, streamed
    // 55 us; with fewer rows one warp a row of the other kernel is as good (1000 x
    // 256 2.8 and 2.7 us).
    if (a.dim <= kChunk && a.rows >= 8 * num_sms) return launch_narrow<T, R, 32>(a, num_sms, stream);
    cudaError_t e = cudaSuccess;
    const bool streamed = a.dim <= kChunk       ? false
                          : a.dim <= 2 * kChunk ? launch_stream<T, R, 2>(a, num_sms, stream, e)
                                                : launch_stream<T, R, 4>(a, num_sms, stream, e);
    if (streamed) return e;
    if (a.dim <= kMaxWarps * kChunk) return launch_few<T, R, 1, true>(a, stream);
    if (a.dim <= 2 * kMaxWarps * kChunk) return launch_few<T, R, 1, false>(a, stream);
    return launch_few<T, R, 2, false>(a, stream);
}

template <typename T, typename R, int CPW>
cudaError_t prepare_stream() {
    const cudaError_t e =
        cudaFuncSetAttribute(norm_stream_kernel<T, R, CPW, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kStreamBytes);
    if (e != cudaSuccess) return e;
    return cudaFuncSetAttribute(norm_stream_kernel<T, R, CPW, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kStreamBytes);
}

template <typename T, typename R>
cudaError_t prepare_types() {
    cudaError_t e;
    if ((e = prepare_stream<T, R, 2>()) != cudaSuccess) return e;
    return prepare_stream<T, R, 4>();
}

}  // namespace

cudaError_t norm_prepare() {
    cudaError_t e;
    if ((e = prepare_types<float, float>()) != cudaSuccess) return e;
    if ((e = prepare_types<__half, float>()) != cudaSuccess) return e;
    if ((e = prepare_types<__half, __half>()) != cudaSuccess) return e;
    if ((e = prepare_types<__nv_bfloat16, float>()) != cudaSuccess) return e;
    return prepare_types<__nv_bfloat16, __nv_bfloat16>();
}

cudaError_t launch_norm_residual(const NormResidualArgs& a, int num_sms, cudaStream_t stream) {
    switch (a.kind) {
        case kF32: return launch_types<float, float>(a, num_sms, stream);
        case kF16:
            return a.resid_kind == kF32 ? launch_types<__half, float>(a, num_sms, stream)
                                        : launch_types<__half, __half>(a, num_sms, stream);
        case kBF16:
            return a.resid_kind == kF32 ? launch_types<__nv_bfloat16, float>(a, num_sms, stream)
                                        : launch_types<__nv_bfloat16, __nv_bfloat16>(a, num_sms, stream);
    }
    return cudaErrorInvalidValue;
}

}  // namespace s3t
