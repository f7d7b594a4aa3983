/* s3t — SAM 3 ViT vision trunk on NVIDIA B200 (sm_100a): the C ABI.
 *
 * Drop-in for the reference's vision-trunk entry point
 *   sam3::VisionTrunk::run(image_nchw, shape_nchw)
 *   (include/sam3/vision_trunk.h:15-26, src/vision_trunk.cpp:297-488),
 * reading the same GGUF tensors (names resolved through the converter's
 * <file>.tensor_map.json sidecar like src/gguf_model.cpp:28-47,190-204) in the
 * same F32 / F16 / Q8_0 formats.
 *
 * Conventions follow the reference's C API (include/sam3/c_api.h,
 * src/c_api.cpp:19-23): functions return 0 on success and -1 on failure with
 * a thread-local message from s3t_last_error(); nothing throws across the ABI;
 * buffers passed in are borrowed, never freed.  One context is bound to one
 * GPU and is not safe for concurrent calls (like the reference's
 * VisionTrunk::run, which shares the backend's work buffer).
 */
#ifndef S3T_H
#define S3T_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ggml type codes of the weight formats (ggml/include/ggml.h GGML_TYPE_*). */
enum { S3T_TYPE_F32 = 0, S3T_TYPE_F16 = 1, S3T_TYPE_Q8_0 = 8 };
/* Element types of the operators that follow s3t_layernorm: F32, F16, BF16
 * (ggml's code) and 8-bit e4m3 (no ggml code). */
enum { S3T_TYPE_BF16 = 30, S3T_TYPE_E4M3 = 1000 };

/* s3t_trunk_run flags: where the image and output buffers live. */
enum {
    S3T_IMAGES_ON_DEVICE = 1, /* images_nchw is a device pointer on the context's GPU */
    S3T_OUTPUT_ON_DEVICE = 2, /* out_nchw is a device pointer on the context's GPU */
};

typedef struct s3t_ctx s3t_ctx;

/* Create a context on CUDA device `device`.  Replaces GgufModel::load's
 * backend selection (src/gguf_model.cpp:107-120) for the trunk.  NULL on error. */
s3t_ctx *s3t_create(int device);
void s3t_destroy(s3t_ctx *ctx);
const char *s3t_last_error(void);

/* Stage one trunk tensor (host bytes, ggml layout: ne[0] fastest).  `name`
 * is the original (unhashed) tensor name, e.g.
 * "backbone.vision_backbone.trunk.blocks.3.attn.qkv.weight".  Replaces the
 * per-tensor ggml_backend_tensor_set of src/gguf_model.cpp:150-153. */
int s3t_set_weight(s3t_ctx *ctx, const char *name, int ggml_type, const int64_t ne[4], const void *host_bytes,
                   size_t nbytes);

/* Read every trunk tensor of a GGUF file (GgufModel::load,
 * src/gguf_model.cpp:83-168).  tensor_map_path may be NULL, meaning
 * "<gguf_path>.tensor_map.json" if that file exists. */
int s3t_load_gguf(s3t_ctx *ctx, const char *gguf_path, const char *tensor_map_path);

/* Check a GGUF file as s3t_load_gguf reads it, without a GPU: header,
 * metadata, tensor records and every trunk tensor's type and byte range
 * against the file's length.  Outputs (may be NULL): the number of trunk
 * tensors and of transformer blocks found.  A truncated or corrupt file
 * returns -1 with a message, like GgufModel::load returning false
 * (src/gguf_model.cpp:83-94). */
int s3t_gguf_inspect(const char *gguf_path, const char *tensor_map_path, int *n_trunk_tensors, int *n_layers);

/* Validate shapes/types of the staged tensors, upload them and convert them
 * to the GEMM operand format (Q8_0 / F32 -> fp16 on the device, patch-embed
 * repacked).  Must be called once before the first run. */
int s3t_finalize_weights(s3t_ctx *ctx);

/* Number of transformer blocks found in the weights (32 for SAM 3). */
int s3t_num_layers(const s3t_ctx *ctx);

/* The trunk: images [batch][3][1008][1008] fp32 -> out [batch][1024][72][72]
 * fp32, both NCHW (VisionTrunk::run, src/vision_trunk.cpp:297-488, with the
 * batch of 1 generalised to `batch` independent images).  stream is a
 * cudaStream_t or NULL for the context's own stream.  With host buffers the
 * call returns after the output is in host memory; with both buffers on the
 * device it returns after enqueueing (check with s3t_sync). */
int s3t_trunk_run(s3t_ctx *ctx, const float *images_nchw, int batch, float *out_nchw, int flags, void *stream);

/* Same, stopping after the first n_layers blocks (0 = patch embed + pos +
 * ln_pre only).  Mirrors the per-stage dumps of the reference's
 * tools/export_vision_trunk_reference.py (.stem/.ln_pre/.layer_NN). */
int s3t_trunk_run_layers(s3t_ctx *ctx, const float *images_nchw, int batch, int n_layers, float *out_nchw, int flags,
                         void *stream);

/* One block of the trunk from a given residual: x_dev [batch*5184][1024]
 * fp32 token-major (token y*72 + x of each image, the input of block
 * `layer`) -> out_dev, the same layout, the block's output residual
 * (norm1, attention with its window partition, proj + residual, norm2, MLP
 * + residual: one iteration of the layer loop of src/vision_trunk.cpp:377-459).
 * Per-block parity entry, the counterpart of the per-layer dumps of the
 * reference's tools/export_vision_trunk_reference.py.  Device pointers on
 * the context's GPU; synchronous (returns after the block ran). */
int s3t_trunk_run_block(s3t_ctx *ctx, int layer, const float *x_dev, int batch, float *out_dev, void *stream);

/* The trunk from decoded 8-bit RGB: rgb [batch][height][width][3] uint8
 * (row-major HWC, what stbi_load returns; all images of a call share one
 * size) is resized and normalized on the device exactly as the reference's
 * load_image_rgb (src/pipeline.cpp:45-83; tools/sam3_vision_trunk.cpp:33-66
 * bilinear_resize_rgb) and then run through the trunk, replacing the host
 * preprocessing loop and the 12 MB fp32 image per request.  flags as for
 * s3t_trunk_run: S3T_IMAGES_ON_DEVICE means rgb is a device pointer.
 * 1 <= width, height <= 32768.  Image decoding (stbi_load) stays with the
 * caller. */
int s3t_trunk_run_rgb8(s3t_ctx *ctx, const uint8_t *rgb, int width, int height, int batch, float *out_nchw,
                       int flags, void *stream);

/* No counterpart in the reference: one eager (not graph-replayed) trunk run on
 * device buffers with a CUDA event after every launch, for measurement.
 * Returns per kernel class the summed device milliseconds and the launch
 * count, in this order: 0 stem (im2col + patch GEMM + ln_pre/norm1),
 * 1 QKV GEMM, 2 windowed attention, 3 global attention, 4 proj GEMM,
 * 5 LayerNorm, 6 fc1 GEMM, 7 fc2 GEMM.  kind_ms and kind_launches hold 8
 * entries each.  Synchronous. */
int s3t_trunk_profile(s3t_ctx *ctx, const float *images_dev, int batch, float *out_dev, void *stream,
                      double *kind_ms, int *kind_launches);

/* Wait for the context's queued work and report any device-side error. */
int s3t_sync(s3t_ctx *ctx, void *stream);

/* --- the vision neck's first operation, on the trunk's device output -------
 * The reference hands the trunk's output to sam3::VisionNeck::run as a host
 * vector (src/pipeline.cpp:159-163, src/vision_neck.cpp:203-206), a full D2H
 * and H2D in between.  These take the trunk's NCHW output where
 * s3t_trunk_run (S3T_OUTPUT_ON_DEVICE) left it and run the first operation of
 * one neck level (src/vision_neck.cpp:262-345) with the neck weights the same
 * GGUF file holds (backbone.vision_backbone.convs.*):
 *   level 0: 2x2 stride-2 transposed conv dconv_2x2_0 + bias, then GELU
 *            (the input of the second transposed conv) -> [B][512][144][144]
 *   level 1: 2x2 stride-2 transposed conv dconv_2x2 + bias -> [B][512][144][144]
 *   level 2: 1x1 conv conv_1x1 + bias                      -> [B][256][72][72]
 *   level 3: 2x2 max pool, then 1x1 conv conv_1x1 + bias   -> [B][256][36][36]
 * (channel counts as the file gives them; s3t_neck_first_shape reports them).
 * trunk_dev [batch][1024][72][72] and out_dev are fp32 device memory of the
 * context's GPU; enqueued on `stream` (NULL: the context's own stream).  The
 * operands are fp16 with fp32 accumulation and the result passes through
 * fp16.  The transposed conv multiplies the values in the order the
 * reference's graph reads them (its ggml_permute(x, 2, 0, 1, 3) on [W, H, C],
 * :96-105).  Uses the context's workspace: not concurrently with a trunk run
 * on the same context. */
int s3t_neck_first(s3t_ctx *ctx, int level, const float *trunk_dev, int batch, float *out_dev, void *stream);

/* Shape [1][C][H][W] of s3t_neck_first's output for one image, or -1 if the
 * file holds no weights for that level. */
int s3t_neck_first_shape(const s3t_ctx *ctx, int level, int64_t shape[4]);

/* --- several GPUs of one node -------------------------------------------
 * No counterpart in the reference, which runs the trunk on one backend device
 * (src/gguf_model.cpp:107-120).  The trunk is per image, so a batch is split
 * into contiguous shards of ceil(batch / n_devices) images, one per GPU; each
 * GPU holds its own copy of the weights and is driven by its own host thread.
 * The only exchange is moving images in and feature maps out (peer copies,
 * no collective inside the trunk).  A handle is not safe for concurrent calls. */
typedef struct s3t_multi s3t_multi;

/* Load the trunk of gguf_path onto every listed device (distinct device
 * indices; devices[0] is the "first GPU" below).  NULL on error. */
s3t_multi *s3t_multi_create(const int *devices, int n_devices, const char *gguf_path, const char *tensor_map_path);
void s3t_multi_destroy(s3t_multi *m);
int s3t_multi_num_devices(const s3t_multi *m);

/* images [batch][3][1008][1008] -> out [batch][1024][72][72] fp32 NCHW.  Host
 * buffers (flags 0): every GPU copies its own slices in and out; returns when
 * the output is in host memory.  With S3T_IMAGES_ON_DEVICE /
 * S3T_OUTPUT_ON_DEVICE the buffers are memory of devices[0]: the other GPUs
 * peer-copy their images in and their features out (the gather to the first
 * GPU), chunk by chunk so the copies overlap their compute.  `stream` is a
 * stream of devices[0] (NULL: its context's own stream); with device buffers
 * the call returns after enqueueing, and that stream waits for every GPU's
 * work (check with s3t_multi_sync). */
int s3t_multi_run(s3t_multi *m, const float *images_nchw, int batch, float *out_nchw, int flags, void *stream);

/* Wait for every GPU's queued work of the handle and report device errors. */
int s3t_multi_sync(s3t_multi *m, void *stream);

/* --- op-level entry points (parity tests, microbenchmarks) --------------- */

/* Dequantize GGUF weight bytes on the device to fp32: F16 and Q8_0
 * (dequantize_row_q8_0, ggml/src/ggml-quants.c:436-450).  Device pointers. */
int s3t_dequantize(int ggml_type, const void *src_dev, int64_t n, float *dst_dev, void *stream);

/* The fp16 GEMM operand that s3t_finalize_weights makes of a linear weight,
 * with the same conversion: Q8_0 -> fp16(q * d) (the exact product of
 * dequantize_row_q8_0, ggml/src/ggml-quants.c:436-450, rounded to nearest
 * even fp16), F32 -> fp16 (round to nearest even), F16 -> unchanged.
 * Device pointers; dst16 holds n fp16 values. */
int s3t_weight_operand(int ggml_type, const void *src_dev, int64_t n, void *dst16_dev, void *stream);

/* y16[M][N] = fp16(act(x16[M][K] * w16[N][K]^T + bias)) — the trunk's GEMM
 * (ggml_mul_mat + bias, src/vision_trunk.cpp:50-62).  act: 0 none, 1 GELU-erf.
 * q8: apply the Q8_0 activation rounding to the output.  Device pointers. */
int s3t_gemm_f16(int device, const void *x16, const void *w16, const float *bias, int M, int N, int K, int act,
                 int q8, void *y16, void *stream);

/* Flash attention on grouped, already-rotated q/k/v [groups*16][L][64]
 * (fp16 or bf16), output token-major [images*5184][1024] in natural token
 * order (windowed: 9 groups per image).  Device pointers. */
int s3t_attention(int device, const void *q, const void *k, const void *v, int groups, int L, int windowed, int bf16,
                  void *out, void *stream);

/* Multi-head attention of the encoder fusion, 8 heads of 32 (model width
 * 256): replaces mha() of src/encoder_fusion.cpp:63-88, the
 * ggml_flash_attn_ext call with prec F32 and scale 1/sqrt(32) that the
 * encoder's self attention (:266, no mask) and image-to-prompt cross
 * attention (:299, prompt mask) run.  `batch` independent sequences (the
 * reference runs one image per call; batch 1 is that call): q_dev
 * [batch][q_len][256], k_dev/v_dev [batch][kv_len][256] token-major fp16
 * (flags & S3T_MHA_BF16: bf16), head h in columns [32h, 32h+32).
 * key_mask_dev: null, or [batch][kv_len] fp32 added to every query row's
 * scaled scores; a key whose entry is -inf takes no part (the reference
 * builds its prompt mask as 0 / -inf rows of this vector, :120-133), and a
 * row whose keys are all masked gives 0, as ggml's CPU kernel does.  out_dev
 * [batch][q_len][256] fp32, or the operand type with S3T_MHA_OUT_F16.
 * Device pointers, 16-byte aligned, on `device`, enqueued on `stream`.
 * Returns 0, or -1 with s3t_last_error(). */
#define S3T_MHA_BF16 1
#define S3T_MHA_OUT_F16 2
/* With S3T_MHA_BIAS, key_mask_dev is a full additive bias [batch][8][q_len]
 * [kv_len] fp32 (one row per sequence, head and query): the decoder's image
 * cross attention with its box relative-position bias (mha() of
 * src/decoder.cpp:95-127 over image_bias_t, :401-418, :457-465).  The
 * decoder's other two attentions are the plain call: self attention over its
 * 201 queries (:430, no mask) and the text cross attention with the prompt
 * mask row (:443).  The decoder computes softmax explicitly (ggml_soft_max_ext):
 * the result is the same, except that a row with every key at -inf is NaN
 * there and 0 here.
 * Scratch: when the query tiles cannot fill the GPU and there are 16 or more
 * blocks of 64 keys (the decoder's 201 queries against 5184 image tokens),
 * each tile's keys are split into ranges computed in parallel and merged;
 * the call then allocates a stream-ordered scratch buffer of about
 * batch * ceil(q_len / 128) * 128 * 8 heads * splits * 34 floats
 * (cudaMallocAsync on `stream`, freed with cudaFreeAsync on the same stream;
 * 5.3 MB for that decoder call, split 19 ways).  Every other call allocates
 * nothing. */
#define S3T_MHA_BIAS 4
int s3t_mha_d32(int device, const void *q_dev, const void *k_dev, const void *v_dev, int batch, int q_len,
                int kv_len, const float *key_mask_dev, void *out_dev, int flags, void *stream);

/* The preprocessing of s3t_trunk_run_rgb8 alone: rgb_dev [batch][height]
 * [width][3] uint8 -> out_dev [batch][3][1008][1008] fp32, bit-exact with
 * the reference's bilinear_resize_rgb (tools/sam3_vision_trunk.cpp:33-66).
 * Device pointers on `device`, enqueued on `stream`. */
int s3t_preprocess_rgb8(int device, const uint8_t *rgb_dev, int width, int height, int batch, float *out_dev,
                        void *stream);

/* Axial RoPE in place on grouped q or k (layout as above). */
int s3t_rope(int device, void *x, int groups, int L, int windowed, int bf16, void *stream);

/* LayerNorm over 1024 columns (eps 1e-5), fp32 in -> fp16 out (q8: Q8_0
 * activation rounding of the output).  Device pointers. */
int s3t_layernorm(int device, const float *x, int rows, const float *gamma, const float *beta, void *y16, int q8,
                  void *stream);

/* --- 8-bit products and the operators around them ------------------------
 * No counterpart in the reference, whose 8-bit path is Q8_0 weights on a CPU.
 * s3t_quantize_fp8 makes 8-bit operands, s3t_gemm_fp8 multiplies them,
 * s3t_norm_residual is the step between two blocks and can write the next
 * product's operand, and s3t_rotary turns the heads that a product returned.
 * Shared rules: device pointers on `device`, work enqueued on `stream` (a
 * cudaStream_t, NULL: the default stream) in one kernel, no allocation and no
 * workspace, so calls may overlap on several streams and be captured.  The
 * first call of any entry point on a device prepares that device (allocates):
 * make it before a capture.  The caller's current device is left as it was.
 * Strides count elements.  Inputs are read in whole 16-byte units that hold one
 * of their bytes.  Outputs overlap no input, except where in place is allowed
 * below.  A call with no rows or tokens (or no columns) writes nothing
 * and succeeds, whatever its pointers and strides. */

/* Rows of a matrix in device memory.  scale and scale_stride belong to e4m3
 * matrices: the scale of column group g (128 columns; the last may be
 * narrower) of row block i is scale[g * scale_stride + i].  A row block is one
 * row of an activation and 128 rows of a weight; a value stands for its e4m3
 * number times its block's scale.  e4m3 data is 16-byte aligned and its stride
 * a multiple of 16; bytes between the columns and the stride are not read and
 * not written. */
typedef struct s3t_matrix {
    void *data;
    int64_t stride;
    float *scale;
    int64_t scale_stride;
} s3t_matrix;

/* x [rows][x_stride] (F32, F16 or BF16; `cols` columns) -> q: e4m3 values with
 * a scale per 128 columns and block_rows rows (1: an activation, 128: a
 * weight).  With a = max(largest magnitude of the block, 2^-100): scale =
 * a / 448, value = e4m3(x * (448 / a)), every operation in fp32 to nearest
 * even.  A block that holds an infinity or a NaN gets that as its scale and
 * stands for NaN as a whole. */
int s3t_quantize_fp8(int device, int type, const void *x_dev, int64_t rows, int64_t cols, int64_t x_stride,
                     int block_rows, const s3t_matrix *q, void *stream);

/* y[M][N] = act(x[M][K] * w[N][K]^T + bias) of an e4m3 activation x (row
 * blocks of 1) and an e4m3 weight w (row blocks of 128): the products of a
 * group of 128 columns are summed in fp32 and scaled by both scales, the
 * groups are summed in fp32.  bias: [N] fp32 or NULL.  act: 0 none, 1 GELU-erf,
 * computed in fp32 to within 1.9e-7 |x| and, for x >= -6, 2.4e-4 of GELU(x)
 * itself (below, where |GELU| < 6e-9, it falls to 0 sooner than GELU).  y_type:
 * F32, F16, BF16, or E4M3, which holds what s3t_quantize_fp8 with block_rows 1
 * makes of the F32 result (y->scale for [ceil(N / 128)][scale_stride >= M]),
 * ready to be the next product's x.  Any M, N >= 0 and K >= 1 (without rows or
 * columns of y K >= 0), up to 2^30 each.  The result does not depend on what
 * else runs; the order of a row's fp32 sums does depend on M, N and K, so that
 * with another M the same row may differ by a few of their roundings (an 8-bit
 * result by a code at a boundary).  A wait that runs out inside the kernel is
 * reported by s3t_device_status. */
int s3t_gemm_fp8(int device, const s3t_matrix *x, const s3t_matrix *w, const float *bias_dev, int M, int N, int K,
                 int act, int y_type, const s3t_matrix *y, void *stream);

/* The step between two transformer blocks, per row of `dim` columns:
 *   h    = post-norm(y) with S3T_NORM_POST, else y
 *   x'   = resid_scale * x + branch_scale * channel_scale * f(gate) * h
 *   u    = pre-norm(x')
 * Norms are RMSNorm, v / sqrt(mean(v^2) + eps) * weight + bias, or with
 * S3T_NORM_LAYER LayerNorm, (v - mean) / sqrt(var + eps) * weight + bias.  f
 * is the identity, or a sigmoid or tanh by flag.  Everything is computed in
 * fp32; u is taken from x' before its rounding to resid_type.  The order of a
 * row's sums and products depends on the count of rows, dim and alignment, so
 * that among other rows it may differ by a few fp32 roundings.  A wait that runs
 * out inside the kernel is reported by s3t_device_status. */
enum {
    S3T_NORM_LAYER = 1,
    S3T_NORM_POST = 2,
    S3T_NORM_GATE_SIGMOID = 4,
    S3T_NORM_GATE_TANH = 8,
};
typedef struct s3t_norm_args {
    int64_t rows;               /* [0, 2^31) */
    int32_t dim;                /* [1, 16384] */
    int32_t type;               /* of y and gate: F32, F16 or BF16 */
    int32_t resid_type;         /* of x and x_out: F32 or `type` */
    int32_t u_type;             /* of u: `type`, or E4M3 (quantized like s3t_quantize_fp8, block_rows 1) */
    int32_t flags;
    float eps;
    float resid_scale;
    float branch_scale;
    const void *y;              /* the block's output, or NULL: x' = resid_scale * x */
    int64_t y_stride;
    const float *post_weight;   /* [dim] each, or NULL: 1 and 0 */
    const float *post_bias;
    const void *gate;           /* row r uses gate row r / gate_rows (gate_rows 1: one per token; the tokens of a
                                 * sequence: one per sequence); NULL: 1 */
    int64_t gate_stride;        /* 0: one gate row for all */
    int64_t gate_rows;
    const float *channel_scale; /* [dim], or NULL: 1 */
    const void *x;              /* the residual */
    int64_t x_stride;
    void *x_out;                /* x' (may be x itself, with its stride), or NULL: not written */
    int64_t x_out_stride;
    const float *pre_weight;    /* [dim] each, or NULL: 1 and 0 */
    const float *pre_bias;
    s3t_matrix u;               /* the next block's input, or data NULL: no pre-norm */
} s3t_norm_args;
int s3t_norm_residual(int device, const s3t_norm_args *args, void *stream);

/* Radians per position of each of the rot_dim / 2 pairs of rotary positions,
 * freq[i] = base^(-2 i / rot_dim), and the magnitude to multiply by, scaled
 * for contexts `factor` (>= 1) times the trained one:
 *   LINEAR    freq / factor (position interpolation)
 *   BASE      base * factor^(rot_dim / (rot_dim - 2))
 *   BY_PARTS  pairs with more than `fast` full turns within original_len keep
 *             their frequency, pairs with fewer than `slow` get freq / factor,
 *             linear in the turns between; magnitude 0.1 ln(factor) + 1 (YaRN,
 *             Peng et al. 2023, the ramp as the paper has it; programs that ramp
 *             over the index of the pair between two rounded limits have other
 *             frequencies there: s3t_rotary takes any that the caller computes)
 * Host only: freq is host memory, to be copied to the device once. */
enum { S3T_ROTARY_UNSCALED = 0, S3T_ROTARY_LINEAR = 1, S3T_ROTARY_BASE = 2, S3T_ROTARY_BY_PARTS = 3 };
int s3t_rotary_frequencies(int rot_dim, double base, int scaling, double factor, double original_len, double fast,
                           double slow, double *freq, float *magnitude);

/* The heads of one tensor: token t, head h, column c is
 * x[t * x_token_stride + h * x_head_stride + c], so token-major, head-major
 * and packed projections (a pointer to the first head) are all views.  out may
 * be x itself, with the same strides.  Heads of x may overlap (a stride of 0
 * turns one head by every position); heads of out must not, neither with one
 * another nor with the other tensor's. */
typedef struct s3t_rotary_view {
    const void *x;
    void *out;
    int32_t heads;
    int64_t x_token_stride, x_head_stride, out_token_stride, out_head_stride;
} s3t_rotary_view;

/* Turns the first rot_dim columns of every head of q and (unless NULL) k by
 * positions[t] * freq[i]: pair i is columns (i, i + rot_dim / 2), or (2 i,
 * 2 i + 1) with S3T_ROTARY_INTERLEAVED; S3T_ROTARY_INVERSE turns back (the
 * magnitude still multiplies).  The other columns are copied.  The angle is
 * taken in 64 bits: for positions up to 2^27 and frequencies up to 1 it is exact
 * to 2^-27 turns, and cosine and sine to 1.5 fp32 steps besides.  The heads of a
 * token whose position is negative (padding) are not written. */
enum { S3T_ROTARY_INTERLEAVED = 1, S3T_ROTARY_INVERSE = 2 };
int s3t_rotary(int device, const double *freq_dev, int rot_dim, float magnitude, const int64_t *positions_dev,
               int64_t tokens, int type, int head_dim, const s3t_rotary_view *q, const s3t_rotary_view *k, int flags,
               void *stream);

/* No counterpart in the reference: failure-detection self-test.  One device
 * thread waits, for limit_ms (1..2000), on an mbarrier that nothing arrives
 * at; the bounded wait gives up, records a timeout in the device status word
 * and the kernel returns.  Returns 0 when the wait gave up as designed; the
 * next s3t_device_status(device) then reports (and clears) the timeout, and
 * the device stays usable. */
int s3t_selftest_wait_timeout(int device, int limit_ms);

/* Synchronize `device` and report (then clear) the device status word that
 * the op-level entry points write when a bounded in-kernel wait times out. */
int s3t_device_status(int device);

/* Allocation-free stem (no counterpart in the reference): patch embedding +
 * tiled position embedding + ln_pre for one image, the same values as
 * s3t_trunk_run_layers(ctx, ..., n_layers = 0, ...) but token-major:
 * images_dev [batch][3][1008][1008] fp32 -> out_tokens_dev [batch*5184][1024]
 * fp32, both device pointers on the context's GPU and 16-byte aligned,
 * enqueued on `stream` (NULL = the context's own stream, as for every other
 * entry point that takes a context).  For callers that cannot call
 * cudaMalloc (plugins whose host application owns all device memory, loops
 * with a fixed memory budget): it allocates nothing; its one scratch buffer
 * is a static device array inside the library sized for batch <= 1
 * (6,635,520 bytes, held by every GPU that loads the library until exit).
 * Larger batches are rejected with an error.  The first call on a device
 * looks up that array's device address; make that first call before any
 * stream capture.  Calls whose work overlaps on the same GPU race on the
 * shared array. */
int s3t_stem_noalloc(s3t_ctx *ctx, const float *images_dev, int batch, float *out_tokens_dev, void *stream);

#ifdef __cplusplus
}
#endif
#endif
