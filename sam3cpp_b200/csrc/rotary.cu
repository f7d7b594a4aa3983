// Rotary positions: the pairs of the first `rot` columns of every head turn by
// position * frequency,
//   (a, b) -> magnitude (a cos t - b sin t, a sin t + b cos t),
// where a pair is columns (2i, 2i + 1) (interleaved) or (i, i + rot / 2)
// (halves); the other columns pass through.
//
// The angle is taken in 64 bits as turns, position * frequency / 2 pi, and only
// its fraction goes to 32 bits: at position 10^6 an fp32 angle is off by up to
// 0.03 rad, this one by 2^-25 turns.  A CTA takes the tokens' cosines and sines
// into shared memory once for all their heads, so the trigonometry is rot / 2
// evaluations a token and the rest is a stream over the heads: bound by HBM,
// one read and one write of every element.
#include "elements.cuh"
#include "kernels.h"

namespace s3t {

namespace {

constexpr int kThreads = 256;
constexpr int kTableEntries = 2048;   // cos/sin pairs a CTA holds (16 KB)
constexpr int kMaxTokens = 64;        // tokens a CTA takes
constexpr int kAhead = 4;             // heads a thread has in flight

// Consecutive elements of one 16-byte access.
template <typename T>
constexpr int kVec = 16 / int(sizeof(T));

template <typename T, int V>
S3T_DEV void load_run(const T* p, float (&v)[V]) {
    if constexpr (V == 1) {
        v[0] = to_float(*p);
    } else if constexpr (V == 4) {
        const float4 f = *reinterpret_cast<const float4*>(p);
        v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
    } else {
        load8(p, v);
    }
}
template <typename T, int V>
S3T_DEV void store_run(T* p, const float (&v)[V]) {
    if constexpr (V == 1) {
        *p = from_float<T>(v[0]);
    } else if constexpr (V == 4) {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
        store8(p, v);
    }
}

S3T_DEV void turn(float& a, float& b, float2 cs) {
    const float ta = a * cs.x - b * cs.y, tb = a * cs.y + b * cs.x;
    a = ta;
    b = tb;
}

// A token's heads are walked in slots: `turned` slots of V pairs (halves: V
// columns of each half; interleaved: 2 V consecutive columns, or one run of V
// columns where V > 1) and then the slots of V columns that pass through.
template <typename T, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryArgs a, int tokens_per_cta, int turned, int slots) {
    __shared__ float2 table[kTableEntries];
    __shared__ int64_t position[kMaxTokens];
    const int64_t t0 = int64_t(blockIdx.x) * tokens_per_cta;
    const int tokens = int(min(int64_t(tokens_per_cta), a.tokens - t0));
    const int pairs = a.rot / 2;
    for (int i = threadIdx.x; i < tokens * pairs; i += kThreads) {
        const int t = i / pairs, p = i - t * pairs;
        const int64_t pos = a.positions[t0 + t];
        double turns = double(pos) * a.freq[p] * 0.15915494309189533577;   // 1 / (2 pi)
        turns -= rint(turns);
        float s, c;
        sincospif(2.f * float(turns), &s, &c);
        table[i] = make_float2(c * a.magnitude, (a.inverse ? -s : s) * a.magnitude);
    }
    if (threadIdx.x < tokens) position[threadIdx.x] = a.positions[t0 + threadIdx.x];
    __syncthreads();
    // A head's slots lie on consecutive threads, and a thread keeps its slot;
    // kAhead heads are on their way at a time.
    const int heads = a.part[0].heads + a.part[1].heads;
    const int lanes = min(slots, kThreads), at_once = kThreads / lanes;
    const int first = int(threadIdx.x) / lanes;
    if (first >= at_once) return;
    const int total = tokens * heads;
    for (int slot = int(threadIdx.x) - first * lanes; slot < slots; slot += lanes) {
        const bool turned_slot = slot < turned;
        // Columns of the slot's runs, and its first entry of a token's table.
        const bool pair_runs = turned_slot && !(INTERLEAVED && V > 1);
        int ca, cb, entry;
        if (!turned_slot) {
            ca = cb = a.rot + (slot - turned) * V;
            entry = 0;
        } else if (INTERLEAVED) {
            ca = V > 1 ? slot * V : 2 * slot;
            cb = ca + 1;
            entry = V > 1 ? slot * (V / 2) : slot;
        } else {
            ca = slot * V;
            cb = ca + pairs;
            entry = slot * V;
        }
        for (int r0 = first; r0 < total; r0 += kAhead * at_once) {
            T* to[kAhead];
            float va[kAhead][V], vb[kAhead][V];
            int token[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int r = r0 + k * at_once;
                const int t = r < total ? r / heads : 0;
                int h = r - t * heads;
                token[k] = t;
                to[k] = nullptr;
                if (r >= total || position[t] < 0) continue;
                const bool second = h >= a.part[0].heads;
                const RotaryPart& part = a.part[second];
                if (second) h -= a.part[0].heads;
                const T* x = static_cast<const T*>(part.x) + (t0 + t) * part.x_token + h * part.x_head;
                T* out = static_cast<T*>(part.out) + (t0 + t) * part.out_token + h * part.out_head;
                if (!turned_slot && x == out) continue;
                to[k] = out;
                load_run<T, V>(x + ca, va[k]);
                if (pair_runs) load_run<T, V>(x + cb, vb[k]);
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                if (!to[k]) continue;
                const float2* cs = table + token[k] * pairs + entry;
                if (pair_runs) {
#pragma unroll
                    for (int i = 0; i < V; ++i) turn(va[k][i], vb[k][i], cs[i]);
                    store_run<T, V>(to[k] + cb, vb[k]);
                } else if (turned_slot) {
#pragma unroll
                    for (int i = 0; i + 1 < V; i += 2) turn(va[k][i], va[k][i + 1], cs[i / 2]);
                }
                store_run<T, V>(to[k] + ca, va[k]);
            }
        }
    }
}

template <typename T, int V, bool INTERLEAVED>
cudaError_t launch(const RotaryArgs& a, cudaStream_t stream) {
    const int turned = INTERLEAVED && V > 1 ? a.rot / V : a.rot / (2 * V);
    const int slots = turned + (a.head_dim - a.rot) / V;
    const int heads = a.part[0].heads + a.part[1].heads;
    // About 16 slots a thread, within what the table holds; no more tokens
    // than leave every SM two CTAs.
    int64_t tpc = 16ll * kThreads / (int64_t(heads) * slots);
    tpc = min(tpc, int64_t(kTableEntries / (a.rot / 2)));
    tpc = min(tpc, a.tokens / 296);
    tpc = max(int64_t(1), min(tpc, int64_t(kMaxTokens)));
    const int64_t ctas = (a.tokens + tpc - 1) / tpc;
    if (ctas > 0x7fffffff) return cudaErrorInvalidValue;
    rotary_kernel<T, V, INTERLEAVED><<<uint32_t(ctas), kThreads, 0, stream>>>(a, int(tpc), turned, slots);
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch_type(const RotaryArgs& a, cudaStream_t stream) {
    if (a.interleaved)
        return a.vec ? launch<T, kVec<T>, true>(a, stream) : launch<T, 1, true>(a, stream);
    return a.vec ? launch<T, kVec<T>, false>(a, stream) : launch<T, 1, false>(a, stream);
}

}  // namespace

cudaError_t launch_rotary(const RotaryArgs& a, cudaStream_t stream) {
    switch (a.kind) {
        case kF32: return launch_type<float>(a, stream);
        case kF16: return launch_type<__half>(a, stream);
        case kBF16: return launch_type<__nv_bfloat16>(a, stream);
    }
    return cudaErrorInvalidValue;
}

}  // namespace s3t
