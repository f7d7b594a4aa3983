// C entry points of the 8-bit linear path and the operators around it:
// s3t_quantize_fp8, s3t_gemm_fp8, s3t_norm_residual, s3t_rotary_frequencies
// and s3t_rotary.  Each checks its arguments before it touches the device,
// launches one kernel on the caller's stream and leaves the current device as
// it was.
#include "s3t.h"
#include "kernels.h"

#include <cmath>
#include <exception>
#include <string>

using namespace s3t;

namespace {

int refuse(const char* op, const std::string& why) {
    return set_last_error((std::string(op) + ": " + why).c_str());
}

// ElementKind of an S3T_TYPE_* code, -1 for one the operators do not take.
int element_kind(int type) {
    switch (type) {
        case S3T_TYPE_F32: return kF32;
        case S3T_TYPE_F16: return kF16;
        case S3T_TYPE_BF16: return kBF16;
        case S3T_TYPE_E4M3: return kE4M3;
    }
    return -1;
}

// Keeps a size rounded up to whole tiles inside 32 bits.
constexpr int kMost = 1 << 30;

int element_bytes(int kind) { return kind == kF32 ? 4 : kind == kE4M3 ? 1 : 2; }

bool aligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % uintptr_t(bytes) == 0; }

// Rows that all start at a 16-byte boundary.
bool rows16(const void* p, int64_t stride, int kind) { return aligned(p, 16) && stride * element_bytes(kind) % 16 == 0; }

int64_t blocks(int64_t n) { return n / kScaleBlock + (n % kScaleBlock != 0); }

// An 8-bit matrix of rows x cols values with `scales` scales per group; null if it is one.
const char* bad_eight(const s3t_matrix* m, int64_t cols, int64_t scales) {
    if (!m || !m->data || !m->scale) return "an 8-bit matrix needs data and scale";
    if (!aligned(m->data, 16) || m->stride % 16 != 0) return "8-bit rows must start at multiples of 16 bytes";
    if (m->stride < cols) return "an 8-bit row stride is below its columns";
    if (!aligned(m->scale, 4)) return "scales must be 4-byte aligned";
    if (m->scale_stride < scales) return "a scale stride is below its count of rows or row blocks";
    return nullptr;
}

// Whether two of tokens x heads runs of `dim` elements, at t * token + h * head,
// share an element.  Strides are at least dim where there are two to a stride.
bool runs_overlap(int64_t tokens, int64_t token, int heads, int64_t head, int dim) {
    using Wide = __int128;
    if (tokens == 1 || heads == 1) return false;
    if (token >= Wide(heads - 1) * head + dim || head >= Wide(tokens - 1) * token + dim) return false;   // token- or head-major
    for (int h = 1; h < heads; ++h) {   // the tokens next to a head of token 0
        const Wide at = Wide(h) * head, t = at / token, past = at - t * token;
        if ((t < tokens && past < dim) || (t + 1 < tokens && token - past < dim)) return true;
    }
    return false;
}

template <typename Launch>
int run_on(const char* op, int device, Launch launch) {
    DeviceView dev;
    if (device_view(device, &dev)) return -1;
    const DeviceScope scope(device);
    const cudaError_t e = scope.error != cudaSuccess ? scope.error : launch(dev);
    if (e == cudaSuccess) return 0;
    cudaGetLastError();   // reported here: the caller's next check must not find it again
    return refuse(op, cudaGetErrorString(e));
}

#define S3T_CATCH(op)                                                    \
    catch (const std::exception& e) {                                    \
        return set_last_error(e.what());                                 \
    }                                                                    \
    catch (...) {                                                        \
        return set_last_error(op ": internal error");                    \
    }

}  // namespace

extern "C" {

int s3t_quantize_fp8(int device, int type, const void* x, int64_t rows, int64_t cols, int64_t x_stride, int block_rows,
                     const s3t_matrix* q, void* stream) {
    try {
        const char* op = "quantize_fp8";
        const int kind = element_kind(type);
        if (kind < 0 || kind == kE4M3) return refuse(op, "x must be F32, F16 or BF16");
        if (rows < 0 || cols < 0) return refuse(op, "rows and cols must not be negative");
        if (block_rows != 1 && block_rows != kScaleBlock) return refuse(op, "block_rows must be 1 or 128");
        if (rows == 0 || cols == 0) return 0;   // the arrays may be null: empty tensors are
        if (!x || !aligned(x, element_bytes(kind))) return refuse(op, "x must be a device pointer aligned to its type");
        if (x_stride < cols) return refuse(op, "x_stride is below cols");
        if (const char* why = bad_eight(q, cols, block_rows == 1 ? rows : blocks(rows))) return refuse(op, why);
        // Far beyond any GPU's memory; keeps every offset inside 64 bits.
        if (rows > (int64_t(1) << 40) || cols > (int64_t(1) << 40)) return refuse(op, "rows or cols too large");
        QuantizeArgs a{};
        a.x = x;
        a.rows = rows; a.cols = cols; a.x_stride = x_stride;
        a.kind = kind;
        a.block_rows = block_rows;
        a.vec = rows16(x, x_stride, kind);
        a.q = static_cast<uint8_t*>(q->data);
        a.q_stride = q->stride;
        a.scale = q->scale;
        a.scale_stride = q->scale_stride;
        return run_on(op, device, [&](const DeviceView&) { return launch_quantize_fp8(a, static_cast<cudaStream_t>(stream)); });
    } S3T_CATCH("quantize_fp8")
}

int s3t_gemm_fp8(int device, const s3t_matrix* x, const s3t_matrix* w, const float* bias, int M, int N, int K, int act,
                 int y_type, const s3t_matrix* y, void* stream) {
    try {
        const char* op = "gemm_fp8";
        const int kind = element_kind(y_type);
        if (kind < 0) return refuse(op, "y must be F32, F16, BF16 or E4M3");
        const bool empty = M == 0 || N == 0;   // then there may be no K either
        if (M < 0 || N < 0 || K < (empty ? 0 : 1)) return refuse(op, "needs M >= 0, N >= 0 and K >= 1");
        if (M > kMost || N > kMost || K > kMost) return refuse(op, "M, N and K must be at most 2^30");
        if (act != 0 && act != 1) return refuse(op, "act must be 0 (none) or 1 (GELU)");
        if (empty) return 0;
        if (const char* why = bad_eight(x, K, M)) return refuse(op, std::string("x: ") + why);
        if (const char* why = bad_eight(w, K, blocks(N))) return refuse(op, std::string("w: ") + why);
        if (!aligned(bias, 4)) return refuse(op, "bias must be 4-byte aligned");
        if (kind == kE4M3) {
            if (const char* why = bad_eight(y, N, M)) return refuse(op, std::string("y: ") + why);
        } else {
            if (!y || !y->data || !aligned(y->data, element_bytes(kind)))
                return refuse(op, "y must be a device pointer aligned to its type");
            if (y->stride < N) return refuse(op, "the row stride of y is below N");
        }
        GemmFp8Args a{};
        a.M = M; a.N = N; a.K = K;
        a.x = static_cast<const uint8_t*>(x->data);
        a.x_stride = x->stride;
        a.xs = x->scale;
        a.xs_stride = x->scale_stride;
        a.w = static_cast<const uint8_t*>(w->data);
        a.w_stride = w->stride;
        a.ws = w->scale;
        a.ws_stride = w->scale_stride;
        a.bias = bias;
        a.gelu = act == 1;
        a.out = kind;
        a.y = y->data;
        a.y_stride = y->stride;
        a.ys = y->scale;
        a.ys_stride = y->scale_stride;
        a.vec = rows16(y->data, y->stride, kind);
        return run_on(op, device, [&](const DeviceView& dev) {
            a.status = dev.status;
            return launch_gemm_fp8(a, dev.num_sms, static_cast<cudaStream_t>(stream));
        });
    } S3T_CATCH("gemm_fp8")
}

int s3t_norm_residual(int device, const s3t_norm_args* p, void* stream) {
    try {
        const char* op = "norm_residual";
        if (!p) return refuse(op, "no arguments");
        const int kind = element_kind(p->type), resid = element_kind(p->resid_type);
        if (kind < 0 || kind == kE4M3) return refuse(op, "type must be F32, F16 or BF16");
        if (resid != kF32 && resid != kind) return refuse(op, "resid_type must be F32 or type");
        if (p->rows < 0 || p->rows > 0x7fffffff) return refuse(op, "rows must be in [0, 2^31)");
        if (p->dim < 1 || p->dim > kNormMaxDim) return refuse(op, "dim must be in [1, 16384]");
        if (p->flags & ~(S3T_NORM_LAYER | S3T_NORM_POST | S3T_NORM_GATE_SIGMOID | S3T_NORM_GATE_TANH))
            return refuse(op, "unknown flags");
        const bool sigmoid = p->flags & S3T_NORM_GATE_SIGMOID, tanh = p->flags & S3T_NORM_GATE_TANH;
        if (sigmoid && tanh) return refuse(op, "a gate is a sigmoid or a tanh, not both");
        if (!(p->eps >= 0.f) || !std::isfinite(p->eps)) return refuse(op, "eps must be finite and not negative");
        if (p->rows == 0) return 0;
        if ((sigmoid || tanh) && !p->gate) return refuse(op, "a gate function needs the gate array");
        const int eb = element_bytes(kind), rb = element_bytes(resid), dim = p->dim;
        if (!p->x || !aligned(p->x, rb) || p->x_stride < dim) return refuse(op, "x must be an aligned device pointer with x_stride >= dim");
        if (!p->y && (p->gate || p->channel_scale || (p->flags & S3T_NORM_POST)))
            return refuse(op, "a post-norm, gate or channel scale needs y");
        if (p->y && (!aligned(p->y, eb) || p->y_stride < dim)) return refuse(op, "y must be aligned with y_stride >= dim");
        if (p->gate && (!aligned(p->gate, eb) || (p->gate_stride != 0 && p->gate_stride < dim)))
            return refuse(op, "gate must be aligned with gate_stride 0 or >= dim");
        if (p->gate && (p->gate_rows < 1 || p->gate_rows > 0x7fffffff)) return refuse(op, "gate_rows must be in [1, 2^31)");
        if (p->x_out && (!aligned(p->x_out, rb) || p->x_out_stride < dim))
            return refuse(op, "x_out must be aligned with x_out_stride >= dim");
        if (p->x_out == p->x && p->x_out_stride != p->x_stride) return refuse(op, "x_out in place needs x's stride");
        if (!p->x_out && !p->u.data) return refuse(op, "nothing to write: x_out and u are null");
        const float* const vectors[] = {p->post_weight, p->post_bias, p->channel_scale, p->pre_weight, p->pre_bias};
        bool vec = dim % 8 == 0 && rows16(p->x, p->x_stride, resid);
        for (const float* v : vectors) {
            if (!aligned(v, 4)) return refuse(op, "weights and scales must be 4-byte aligned");
            vec = vec && aligned(v, 16);
        }
        const int u_kind = element_kind(p->u_type);
        if (p->u.data) {
            if (u_kind != kind && u_kind != kE4M3) return refuse(op, "u_type must be type or E4M3");
            if (u_kind == kE4M3) {
                if (const char* why = bad_eight(&p->u, dim, p->rows)) return refuse(op, why);
            } else {
                if (!aligned(p->u.data, eb) || p->u.stride < dim) return refuse(op, "u must be aligned with a stride >= dim");
                vec = vec && rows16(p->u.data, p->u.stride, kind);
            }
        }
        vec = vec && (!p->y || rows16(p->y, p->y_stride, kind)) && (!p->gate || rows16(p->gate, p->gate_stride, kind)) &&
              (!p->x_out || rows16(p->x_out, p->x_out_stride, resid));
        NormResidualArgs a{};
        a.rows = p->rows; a.dim = dim;
        a.kind = kind; a.resid_kind = resid;
        a.u_eight = u_kind == kE4M3;
        a.layer = (p->flags & S3T_NORM_LAYER) != 0;
        a.post = (p->flags & S3T_NORM_POST) != 0;
        a.gate_act = sigmoid ? kGateSigmoid : tanh ? kGateTanh : kGatePlain;
        a.eps = p->eps; a.resid_scale = p->resid_scale; a.branch_scale = p->branch_scale;
        a.y = p->y; a.y_stride = p->y_stride;
        a.post_weight = p->post_weight; a.post_bias = p->post_bias;
        a.gate = p->gate; a.gate_stride = p->gate_stride;
        a.gate_rows = p->gate ? int(p->gate_rows) : 1;
        a.channel = p->channel_scale;
        a.x = p->x; a.x_stride = p->x_stride;
        a.x_out = p->x_out; a.x_out_stride = p->x_out_stride;
        a.pre_weight = p->pre_weight; a.pre_bias = p->pre_bias;
        a.u = p->u.data; a.u_stride = p->u.stride;
        a.u_scale = p->u.scale; a.u_scale_stride = p->u.scale_stride;
        a.vec = vec;
        return run_on(op, device, [&](const DeviceView& dev) {
            a.status = dev.status;
            return launch_norm_residual(a, dev.num_sms, static_cast<cudaStream_t>(stream));
        });
    } S3T_CATCH("norm_residual")
}

int s3t_rotary_frequencies(int rot_dim, double base, int scaling, double factor, double original_len, double fast,
                           double slow, double* freq, float* magnitude) {
    try {
        const char* op = "rotary_frequencies";
        if (!freq || !magnitude) return refuse(op, "freq and magnitude must not be null");
        if (rot_dim < 2 || rot_dim > kRotaryMaxDim || rot_dim % 2) return refuse(op, "rot_dim must be even and in [2, 1024]");
        if (!(base > 0) || !std::isfinite(base)) return refuse(op, "base must be positive");
        if (scaling < S3T_ROTARY_UNSCALED || scaling > S3T_ROTARY_BY_PARTS) return refuse(op, "unknown scaling");
        if (scaling != S3T_ROTARY_UNSCALED && (!(factor >= 1) || !std::isfinite(factor)))
            return refuse(op, "factor must be at least 1");
        if (scaling == S3T_ROTARY_BY_PARTS && (!(original_len > 0) || !std::isfinite(original_len) || !(slow >= 0) || !(fast > slow) ||
                                               !std::isfinite(fast)))
            return refuse(op, "scaling by parts needs original_len > 0 and fast > slow >= 0");
        const double two_pi = 6.283185307179586476925;
        // One pair has the frequency 1 at any base, so the base cannot scale it.
        if (scaling == S3T_ROTARY_BASE && rot_dim > 2) base *= std::pow(factor, rot_dim / double(rot_dim - 2));
        for (int i = 0; i < rot_dim / 2; ++i) {
            double f = std::pow(base, -2.0 * i / rot_dim);
            if (scaling == S3T_ROTARY_LINEAR) f /= factor;
            if (scaling == S3T_ROTARY_BY_PARTS) {
                double keep = (original_len * f / two_pi - slow) / (fast - slow);
                keep = keep < 0 ? 0 : keep > 1 ? 1 : keep;
                f = f * keep + f / factor * (1 - keep);
            }
            freq[i] = f;
        }
        *magnitude = scaling == S3T_ROTARY_BY_PARTS ? float(0.1 * std::log(factor) + 1.0) : 1.0f;
        return 0;
    } S3T_CATCH("rotary_frequencies")
}

int s3t_rotary(int device, const double* freq, int rot_dim, float magnitude, const int64_t* positions, int64_t tokens,
               int type, int head_dim, const s3t_rotary_view* q, const s3t_rotary_view* k, int flags, void* stream) {
    try {
        const char* op = "rotary";
        const int kind = element_kind(type);
        if (kind < 0 || kind == kE4M3) return refuse(op, "type must be F32, F16 or BF16");
        if (head_dim < 2 || head_dim > kRotaryMaxDim) return refuse(op, "head_dim must be in [2, 1024]");
        if (rot_dim < 2 || rot_dim > head_dim || rot_dim % 2) return refuse(op, "rot_dim must be even and in [2, head_dim]");
        if (flags & ~(S3T_ROTARY_INTERLEAVED | S3T_ROTARY_INVERSE)) return refuse(op, "unknown flags");
        if (tokens < 0 || tokens > (int64_t(1) << 31) - 1) return refuse(op, "tokens must be in [0, 2^31)");
        if (tokens == 0) return 0;
        if (!freq || !aligned(freq, 8)) return refuse(op, "freq must be an aligned device pointer");
        if (!positions || !aligned(positions, 8)) return refuse(op, "positions must be an aligned device pointer");
        if (!q) return refuse(op, "q must not be null");
        const int eb = element_bytes(kind);
        RotaryArgs a{};
        // Everything that a run of elements must divide: columns, strides and addresses.
        uint64_t marks = uint64_t(flags & S3T_ROTARY_INTERLEAVED ? rot_dim : rot_dim / 2) | uint64_t(head_dim - rot_dim);
        const s3t_rotary_view* const views[2] = {q, k};
        for (int i = 0; i < 2; ++i) {
            const s3t_rotary_view* s = views[i];
            if (!s) continue;
            if (s->heads < 1 || s->heads > 65536) return refuse(op, "heads must be in [1, 65536]");
            if (!s->x || !s->out || !aligned(s->x, eb) || !aligned(s->out, eb))
                return refuse(op, "x and out must be device pointers aligned to the type");
            if (s->x_token_stride < 0 || s->x_head_stride < 0) return refuse(op, "strides must not be negative");
            if ((tokens > 1 && s->out_token_stride < head_dim) || (s->heads > 1 && s->out_head_stride < head_dim))
                return refuse(op, "the strides of out must be at least head_dim");
            if (s->x == s->out && (s->x_token_stride != s->out_token_stride || s->x_head_stride != s->out_head_stride))
                return refuse(op, "in place needs the same strides of x and out");
            if (runs_overlap(tokens, s->out_token_stride, s->heads, s->out_head_stride, head_dim))
                return refuse(op, "heads of out overlap");
            RotaryPart& p = a.part[i];
            p.x = s->x;
            p.out = s->out;
            p.heads = s->heads;
            p.x_token = s->x_token_stride;
            p.x_head = s->x_head_stride;
            p.out_token = s->out_token_stride;
            p.out_head = s->out_head_stride;
            marks |= (reinterpret_cast<uintptr_t>(s->x) | reinterpret_cast<uintptr_t>(s->out)) / uintptr_t(eb);
            marks |= uint64_t(p.x_token) | uint64_t(p.x_head) | uint64_t(p.out_token) | uint64_t(p.out_head);
        }
        if (k && (q->out == k->out || q->out == k->x || k->out == q->x))
            return refuse(op, "q and k must not be written over one another");
        a.run = marks % uint64_t(16 / eb) == 0 ? 16 / eb : marks % 2 == 0 ? 2 : 1;
        a.freq = freq;
        a.rot = rot_dim;
        a.magnitude = magnitude;
        a.positions = positions;
        a.tokens = tokens;
        a.kind = kind;
        a.head_dim = head_dim;
        a.interleaved = (flags & S3T_ROTARY_INTERLEAVED) != 0;
        a.inverse = (flags & S3T_ROTARY_INVERSE) != 0;
        return run_on(op, device, [&](const DeviceView&) { return launch_rotary(a, static_cast<cudaStream_t>(stream)); });
    } S3T_CATCH("rotary")
}

}  // extern "C"
