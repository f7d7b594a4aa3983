// Rotary positions: the pairs of the first `rot` columns of every head turn by
// position * frequency,
//   (a, b) -> magnitude (a cos t - b sin t, a sin t + b cos t),
// where a pair is columns (2i, 2i + 1) (interleaved) or (i, i + rot / 2)
// (halves); the other columns pass through.
//
// The angle is taken in 64 bits as turns, position * frequency / 2 pi, and its
// fraction goes to 32 bits in two parts: at position 10^6 an fp32 angle is off
// by up to 0.03 rad, this one's cosine and sine by two of their own roundings.
// (One part alone was off by 2^-27 turns: a third more error of fp32 heads, rms;
// the second costs nothing where heads are many, 17.3 -> 18.6 us for 65536
// tokens of one head of 128.)  A CTA takes the tokens' cosines and sines
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
constexpr int kRows = 512;            // heads whose places a CTA holds at a time

// Consecutive elements of one 16-byte access.
template <typename T>
constexpr int kVec = 16 / int(sizeof(T));

// V consecutive elements as they lie in memory, moved in one access: one, two,
// or 16 bytes of them.
template <int BYTES>
struct Word;
template <>
struct Word<2> { using W = uint16_t; };
template <>
struct Word<4> { using W = uint32_t; };
template <>
struct Word<8> { using W = uint2; };
template <>
struct Word<16> { using W = uint4; };
template <typename T, int V>
struct alignas(V * sizeof(T)) Run {
    T v[V];
};
template <typename T, int V>
S3T_DEV void load_run(const T* p, Run<T, V>& r) {
    using W = typename Word<V * int(sizeof(T))>::W;
    *reinterpret_cast<W*>(r.v) = *reinterpret_cast<const W*>(p);
}
template <typename T, int V>
S3T_DEV void store_run(T* p, const Run<T, V>& r) {
    using W = typename Word<V * int(sizeof(T))>::W;
    *reinterpret_cast<W*>(p) = *reinterpret_cast<const W*>(r.v);
}
template <typename T, int V>
S3T_DEV void widen(const Run<T, V>& r, float (&v)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = to_float(r.v[i]);
}
template <typename T, int V>
S3T_DEV void narrow(const float (&v)[V], Run<T, V>& r) {
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = from_float<T>(v[i]);
}

S3T_DEV void turn(float& a, float& b, float2 cs) {
    const float ta = a * cs.x - b * cs.y, tb = a * cs.y + b * cs.x;
    a = ta;
    b = tb;
}

// A token's heads are walked in slots: `turned` slots of V pairs (halves: V
// columns of each half; interleaved: 2 V consecutive columns, or one run of V
// columns where V > 1) and then the slots of V columns that pass through.  A
// head's slots lie on consecutive threads and a thread keeps its slot; its
// first head is on its way while the CTA makes the table.  65536 tokens of
// 20 heads of 128, 16-bit: 117 us in halves (5.7 TB/s), 123 us interleaved
// with 96 columns turned; two or four heads in flight a thread took 124 and
// 164 us, since fewer CTAs fit an SM.
template <typename T, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads, INTERLEAVED ? 8 : 6)
    rotary_kernel(const RotaryArgs a, int tokens_per_cta, int turned, int slots, int lanes) {
    __shared__ float2 table[kTableEntries];
    __shared__ int64_t position[kMaxTokens];
    __shared__ ulonglong2 row_at[kRows];      // x and out of a head
    __shared__ short row_token[kRows];
    const int64_t t0 = int64_t(blockIdx.x) * tokens_per_cta;
    const int tokens = int(min(int64_t(tokens_per_cta), a.tokens - t0));
    const int pairs = a.rot / 2;
    const int heads = a.part[0].heads + a.part[1].heads, total = tokens * heads;
    const int at_once = kThreads / lanes;
    const int first = int(threadIdx.x) / lanes;
    int slot = int(threadIdx.x) - first * lanes;

    // Columns of the slot's runs, and its first entry of a token's table.
    bool turned_slot, pair_runs;
    int ca, cb, entry;
    auto place = [&]() {
        turned_slot = slot < turned;
        pair_runs = turned_slot && !(INTERLEAVED && V > 1);
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
    };
    // Where rows base .. of the CTA's heads are: the divisions and 64-bit
    // products once a head, not once a slot.
    auto places = [&](int base) {
        for (int i = threadIdx.x; i < kRows && base + i < total; i += kThreads) {
            const int r = base + i, t = r / heads;
            int h = r - t * heads;
            const bool second = h >= a.part[0].heads;
            const RotaryPart& part = a.part[second];
            if (second) h -= a.part[0].heads;
            const T* x = static_cast<const T*>(part.x) + (t0 + t) * part.x_token + h * part.x_head;
            T* out = static_cast<T*>(part.out) + (t0 + t) * part.out_token + h * part.out_head;
            row_at[i] = make_ulonglong2(reinterpret_cast<unsigned long long>(x), reinterpret_cast<unsigned long long>(out));
            row_token[i] = short(t);
        }
    };
    T* to;
    Run<T, V> ra, rb;
    auto load = [&](int i) {   // row i of those whose places are known
        const ulonglong2 at = row_at[i];
        const T* x = reinterpret_cast<const T*>(at.x);
        to = reinterpret_cast<T*>(at.y);
        if (!turned_slot && x == to) {
            to = nullptr;
            return;
        }
        load_run(x + ca, ra);
        if (pair_runs) load_run(x + cb, rb);
    };
    const bool works = first < at_once;
    place();
    places(0);
    __syncthreads();
    if (works && first < total) load(first);   // first < at_once <= kRows

    for (int i = threadIdx.x; i < tokens * pairs; i += kThreads) {
        const int t = i / pairs, p = i - t * pairs;
        const int64_t pos = a.positions[t0 + t];
        double turns = double(pos) * a.freq[p] * 0.15915494309189533577;   // 1 / (2 pi)
        turns -= rint(turns);
        // What the fraction loses in 32 bits turns the pair a little further.
        const float near = float(turns), rest = float(turns - double(near)) * 6.283185307f;
        float s0, c0;
        sincospif(2.f * near, &s0, &c0);
        const float s = fmaf(c0, rest, s0), c = fmaf(-s0, rest, c0);
        table[i] = make_float2(c * a.magnitude, (a.inverse ? -s : s) * a.magnitude);
    }
    if (threadIdx.x < tokens) position[threadIdx.x] = a.positions[t0 + threadIdx.x];
    __syncthreads();
    for (int base = 0;;) {
        const int here = min(kRows, total - base);
        for (int s0 = 0; works && s0 + slot < slots; s0 += lanes) {   // again where a head has more slots than lanes
            if (s0) {
                slot += s0;
                place();
            }
            for (int i = first; i < here; i += at_once) {
                if (base || s0 || i != first) load(i);
                const int token = row_token[i];
                if (!to || position[token] < 0) continue;
                if (turned_slot) {
                    const float2* cs = table + token * pairs + entry;
                    float va[V];
                    widen(ra, va);
                    if (pair_runs) {
                        float vb[V];
                        widen(rb, vb);
#pragma unroll
                        for (int k = 0; k < V; ++k) turn(va[k], vb[k], cs[k]);
                        narrow(vb, rb);
                        store_run(to + cb, rb);
                    } else {
#pragma unroll
                        for (int k = 0; k + 1 < V; k += 2) turn(va[k], va[k + 1], cs[k / 2]);
                    }
                    narrow(va, ra);
                }
                store_run(to + ca, ra);
            }
            if (s0) {
                slot -= s0;
                place();
            }
        }
        base += kRows;
        if (base >= total) break;
        __syncthreads();
        places(base);
        __syncthreads();
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
    // Threads a head: of one to eight passes over its slots, the first that
    // leaves clearly fewer threads without one (152 slots: three passes of 51,
    // five heads at once, 52 us; in one pass, 104 threads idle, 72 us).
    int lanes = 0, best = 0;
    for (int passes = 1; passes <= 8; ++passes) {
        const int l = (slots + passes - 1) / passes, busy = l <= kThreads ? kThreads / l * slots / passes : 0;
        if (busy * 20 > best * 21) {
            best = busy;
            lanes = l;
        }
    }
    return launch_on(rotary_kernel<T, V, INTERLEAVED>, uint32_t(ctas), kThreads, 0, stream, a, int(tpc), turned, slots, lanes);
}

template <typename T, bool INTERLEAVED>
cudaError_t launch_run(const RotaryArgs& a, cudaStream_t stream) {
    if (a.run == kVec<T>) return launch<T, kVec<T>, INTERLEAVED>(a, stream);
    if (a.run == 2) return launch<T, 2, INTERLEAVED>(a, stream);
    return launch<T, 1, INTERLEAVED>(a, stream);
}

template <typename T>
cudaError_t launch_type(const RotaryArgs& a, cudaStream_t stream) {
    return a.interleaved ? launch_run<T, true>(a, stream) : launch_run<T, false>(a, stream);
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
