/*
 * ttrl_b200.h -- C ABI of the B200 (sm_100a) learner-update kernels.
 *
 * Every entry point:
 *   - takes raw device pointers, element counts and hyper-parameters only,
 *   - enqueues work on the caller's CUDA stream (`stream` is a cudaStream_t)
 *     and never synchronises, allocates device memory or reads device memory
 *     back to the host, so every call can be captured into a CUDA graph,
 *   - returns TTRL_OK (0) or an error code; ttrl_last_error() gives the
 *     message of the most recent failure on the calling thread.
 *
 * Device-side waits are bounded. A kernel that gives up on a wait writes a
 * non-zero code into the optional `status` word (a device int the caller
 * owns and zeroes) instead of hanging.
 *
 * Layout conventions follow the reference engine (scaleresearch/tt-rl,
 * ttrl/engine):
 *   - activations of a convolution are flattened NHWC rows, [N*H*W, C]
 *     (ttrl/engine/layers.py:158-200, ttrl/engine/conv/forward.py:160-205);
 *   - a Linear weight is stored (in_features, out_features)
 *     (ttrl/engine/layers.py:43-47);
 *   - a Conv2d weight is held here as [Cout][KH][KW][Cin] ("KRSC"), the
 *     order in which one output row of the implicit GEMM walks the input;
 *     the logical OIHW form is a host-side permutation
 *     (ttrl/engine/conv/module.py:131-219 keeps a device-specific prepared
 *     layout for the same reason).
 */
#ifndef TTRL_B200_H
#define TTRL_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef void* ttrl_stream_t; /* a cudaStream_t */

enum {
  TTRL_OK = 0,
  TTRL_EINVAL = 1,       /* bad argument (shape, alignment, null pointer) */
  TTRL_ECUDA = 2,        /* a CUDA runtime call failed */
  TTRL_EWORKSPACE = 3,   /* caller workspace too small */
  TTRL_EUNSUPPORTED = 4  /* valid but not implemented for this shape */
};

/* Precision of the tensor-core contractions. */
enum {
  TTRL_PREC_TF32X3 = 0, /* split-TF32: a_hi*b_hi + a_hi*b_lo + a_lo*b_hi, fp32-faithful */
  TTRL_PREC_TF32 = 1    /* single TF32 pass (operands truncated to 10 mantissa bits) */
};

/* ------------------------------------------------------------------ misc */

/* Message of the last failed call on this thread (never NULL). */
const char* ttrl_last_error(void);

/* ABI version of this library. */
int ttrl_version(void);

/* Number of kernels this library has enqueued in this process (launches
 * recorded into a CUDA graph count once, at capture). */
unsigned long long ttrl_launch_count(void);

/* One-time per-device set-up (kernel attributes, driver entry points).
 * Call once per device, outside any stream capture, before other calls. */
int ttrl_init(int device);

/* ------------------------------------------------------------------ GEMM */

/* How an operand tile is gathered. A GEMM computes
 *   D[r][c] = sum_k A[r][k] * B[c][k]
 * and each operand describes its own [rows][k] view of memory. */
enum {
  TTRL_OPND_DENSE = 0,      /* element (r,k) at ptr[r*rs + k*ks] */
  TTRL_OPND_CONV_FPROP = 1, /* im2col of an NHWC activation: r=(n,oy,ox), k=(ky,kx,c) */
  TTRL_OPND_CONV_WGRAD = 2  /* transposed im2col: r=(ky,kx,c), k=(n,oy,ox) */
};

/* Operand flag: every value is exactly representable in tf32 (e.g. raw
 * 0..255 pixel values), so the split-TF32 path needs no low part for it. */
#define TTRL_OPND_EXACT_TF32 1

typedef struct {
  const void* ptr;
  int32_t kind;
  int32_t rows;   /* extent along the tile-row dimension */
  int32_t kdim;   /* extent along the reduction dimension */
  int32_t flags;  /* TTRL_OPND_* flags */
  int64_t rs, ks; /* DENSE: element strides */
  /* conv geometry (CONV_* kinds): input [n][h][w][c], kernel kh x kw,
   * stride, symmetric zero padding, output oh x ow */
  int32_t n, h, w, c, kh, kw, stride, pad, oh, ow;
} ttrl_operand;

enum { TTRL_BIAS_NONE = 0, TTRL_BIAS_ROW = 1, TTRL_BIAS_COL = 2 };

/* Epilogue applied to the fp32 accumulator, in this order:
 *   v = alpha * acc; v += bias; v = mask > 0 ? v : 0; v = relu ? max(v,0) : v;
 *   out = accumulate ? out + v : v                                     */
typedef struct {
  float* out;
  int64_t ors, ocs; /* out[r*ors + c*ocs] */
  float alpha;
  int32_t bias_mode;
  const float* bias;
  const float* mask; /* optional; same (r,c) -> mask[r*mrs + c*mcs] */
  int64_t mrs, mcs;
  int32_t relu;
  int32_t accumulate;
} ttrl_epilogue;

typedef struct {
  int32_t m, n, k;
  int32_t precision; /* TTRL_PREC_* */
  int32_t splits;    /* 0 = choose; >1 splits K across CTAs (needs workspace) */
  int32_t pad0;
  ttrl_operand a, b;
  ttrl_epilogue ep;
} ttrl_gemm_desc;

/* Bytes of workspace ttrl_gemm needs for this descriptor (0 when the
 * chosen schedule does not split K). */
size_t ttrl_gemm_workspace_bytes(const ttrl_gemm_desc* d);

/* General tcgen05 GEMM with fused epilogue. Replaces the ttnn.matmul calls
 * of ttrl/engine/ops/matmul.py:42-45,79-84 and the ttnn.conv2d /
 * conv_transpose2d / strided-slice-matmul calls of
 * ttrl/engine/conv/{weights.py:89-108, transform.py:103-129,
 * backward.py:45-78}. Split-K partial sums are reduced in a fixed order,
 * so results are bit-identical from run to run. */
int ttrl_gemm(const ttrl_gemm_desc* d, float* workspace, size_t workspace_bytes, int* status,
              ttrl_stream_t stream);

/* ---------------------------------------------------------------- Linear */

/* y[M,N] = x[M,K] @ W[K,N] (+ b[N]) (then ReLU if relu).
 * Replaces Linear.forward (ttrl/engine/layers.py:57-61) with the following
 * ReLU (ttrl/engine/ops/unary.py:25-37) fused into the epilogue. */
int ttrl_linear_fwd(const float* x, const float* w, const float* b, float* y, int m, int k,
                    int n, int relu, int precision, float* workspace, size_t workspace_bytes,
                    int* status, ttrl_stream_t stream);

/* Fixed scratch size of ttrl_linear_fwd_noalloc: 64 KB of split-K counters
 * plus partial sums. */
#define TTRL_NOALLOC_SCRATCH_BYTES (4u << 20)

/* ttrl_linear_fwd without a workspace argument, for callers that cannot
 * allocate device memory (a C host that owns no memory pool, or a loop that
 * must not let cudaMalloc synchronise the device). It has no counterpart in
 * the reference. Its split-K scratch is a fixed array of
 * TTRL_NOALLOC_SCRATCH_BYTES inside this library, one per device, and it
 * calls no allocating routine. Shapes whose split-K scratch exceeds that
 * size are refused with TTRL_EWORKSPACE before anything is enqueued. The
 * array is shared by every call on the device: calls issued to one stream
 * are safe, calls whose GPU work overlaps race and may give wrong results.
 * Output is bit-identical to ttrl_linear_fwd on the same inputs. Uses the
 * current device. */
int ttrl_linear_fwd_noalloc(const float* x, const float* w, const float* b, float* y, int m,
                            int k, int n, int relu, int precision, int* status,
                            ttrl_stream_t stream);

/* dx[M,K] (=|+=) (g[M,N] @ W[K,N]^T) masked by (mask > 0) when mask != NULL.
 * Replaces matmul's dA = g @ b^T (ttrl/engine/ops/matmul.py:79-81) and the
 * relu_bw of the layer below it. */
int ttrl_linear_dgrad(const float* g, const float* w, const float* mask, float* dx, int m,
                      int k, int n, int accumulate, int precision, float* workspace,
                      size_t workspace_bytes, int* status, ttrl_stream_t stream);

/* dw[K,N] (=|+=) x[M,K]^T @ g[M,N] and, when db != NULL,
 * db[N] (=|+=) sum_m g[m][:] (an extra row of ones in the same GEMM).
 * The workspace size comes from ttrl_linear_wgrad_workspace_bytes. Replaces matmul's dB = a^T @ g (ttrl/engine/ops/matmul.py:82-84)
 * and the bias-add backward (ttrl/engine/ops/elementwise.py:36-41 with
 * ttrl/engine/ops/broadcast.py:11-30). */
int ttrl_linear_wgrad(const float* x, const float* g, float* dw, float* db, int m, int k, int n,
                      int accumulate, int accumulate_db, int precision, float* workspace,
                      size_t workspace_bytes, int* status, ttrl_stream_t stream);

/* Workspace bytes ttrl_linear_wgrad needs for these extents (the weight
 * GEMM's split-K partials). */
size_t ttrl_linear_wgrad_workspace_bytes(int m, int k, int n);

/* ------------------------------------------------------------------ Conv */

/* Conv flag: the input activation holds values exactly representable in
 * tf32 (the raw 0..255 frames a first layer reads; its 1/255 is `alpha`). */
#define TTRL_CONV_INPUT_EXACT 1

typedef struct {
  int32_t n, h, w, c;      /* input, NHWC */
  int32_t cout, kh, kw;    /* kernel */
  int32_t stride, pad;
  int32_t oh, ow;          /* output extent (validated) */
  int32_t flags;           /* TTRL_CONV_* flags */
} ttrl_conv_geom;

/* y[N*OH*OW, Cout] = alpha * conv(x, W) (+ b) (then ReLU if relu).
 * W is [Cout][KH][KW][Cin]. alpha is the folded input scale of
 * ttrl/engine/conv/forward.py:160-182 (conv(s*x, W) == s*conv(x, W)).
 * Replaces ttnn.conv2d (ttrl/engine/conv/weights.py:89-108) plus the bias
 * add (ttrl/engine/conv/module.py:257-263) and the following ReLU. */
int ttrl_conv_fprop(const float* x, const float* w, const float* b, float* y,
                    const ttrl_conv_geom* g, float alpha, int relu, int precision,
                    float* workspace, size_t workspace_bytes, int* status,
                    ttrl_stream_t stream);

/* dx[N*H*W, Cin] (=|+=) conv_transpose(dy, W) masked by (mask > 0).
 * Replaces input_grad (ttrl/engine/conv/backward.py:33-42) and the relu_bw
 * of the layer below. Needs workspace of ttrl_conv_dgrad_workspace_bytes. */
int ttrl_conv_dgrad(const float* dy, const float* w, const float* mask, float* dx,
                    const ttrl_conv_geom* g, int accumulate, int precision, float* workspace,
                    size_t workspace_bytes, int* status, ttrl_stream_t stream);
size_t ttrl_conv_dgrad_workspace_bytes(const ttrl_conv_geom* g);

/* The same data gradient in two steps, for a caller that prepares the
 * weights off its critical path (they change only at optimizer steps).
 * Applies to unpadded convolutions whose stride divides the kernel and whose
 * windows cover the input exactly; other geometries return TTRL_EUNSUPPORTED
 * (and ttrl_conv_dgrad_weights_bytes returns 0). out receives the s^2
 * stacked, flipped sub-kernels ((s*s*Cin) x (kb*kb*Cout), kb = KH / s) of
 * w[Cout][KH][KW][Cin]; ttrl_conv_dgrad_prepared then computes dx from dy and
 * them as one sub-pixel GEMM, with ttrl_conv_dgrad's mask and accumulate
 * semantics. Replace input_grad (ttrl/engine/conv/backward.py:33-42) and
 * the weight transform inside it (ttrl/engine/conv/transform.py:71-129). */
size_t ttrl_conv_dgrad_weights_bytes(const ttrl_conv_geom* g);
int ttrl_conv_dgrad_weights(const float* w, float* out, const ttrl_conv_geom* g,
                            ttrl_stream_t stream);
int ttrl_conv_dgrad_prepared(const float* dy, const float* wt, const float* mask, float* dx,
                             const ttrl_conv_geom* g, int accumulate, int precision,
                             float* workspace, size_t workspace_bytes, int* status,
                             ttrl_stream_t stream);
size_t ttrl_conv_dgrad_prepared_workspace_bytes(const ttrl_conv_geom* g);

/* dw[Cout][KH][KW][Cin] (=|+=) alpha * sum_m dy[m][o] * x_col[m][(ky,kx,c)]
 * and, when db != NULL, db[Cout] (=|+=) sum_m dy[m][o].
 * Replaces weight_grad (ttrl/engine/conv/backward.py:45-78) and the bias
 * gradient of ttrl/engine/ops/broadcast.py:11-30. */
int ttrl_conv_wgrad(const float* x, const float* dy, float* dw, float* db,
                    const ttrl_conv_geom* g, float alpha, int accumulate, int accumulate_db,
                    int precision, float* workspace, size_t workspace_bytes, int* status,
                    ttrl_stream_t stream);
size_t ttrl_conv_wgrad_workspace_bytes(const ttrl_conv_geom* g);

/* uint8 frames [N][C][H][W] -> fp32 NHWC rows [N*H*W][C], times `scale`.
 * Optional `index` (int32, length N) gathers frames: out image i reads
 * in image index[i]. Replaces the host cast+transpose of
 * ttrl/nets/obs.py:56-75. */
int ttrl_u8_nchw_to_f32_nhwc(const uint8_t* in, const int32_t* index, float* out, int n, int c,
                             int h, int w, float scale, ttrl_stream_t stream);

/* The same frames converted straight into space-to-depth rows for a first
 * convolution whose stride `fold` divides its kernel and the frame size:
 * out[(img, Y, X)][(dy*fold + dx)*c + ch] = in[index ? index[img] : img][ch]
 *   [Y*fold + dy][X*fold + dx] * scale, rows [n*(h/fold)*(w/fold)][fold*fold*c].
 * That convolution is then a stride-1 convolution with kernel k/fold over
 * fold*fold*c channels: the same products, whose operand gathers read
 * contiguous channel runs. Plays the part of ttrl/nets/obs.py:73-75 and the
 * reference's space-to-depth fold (ttrl/engine/conv/packing.py) for the
 * Nature-CNN's first layer. */
int ttrl_u8_nchw_to_f32_s2d(const uint8_t* in, const int32_t* index, float* out, int n, int c,
                            int h, int w, int fold, float scale, ttrl_stream_t stream);

/* ------------------------------------------------------------------ Adam */

/* One parameter tensor of a multi-tensor Adam launch. */
typedef struct {
  float* param;
  const float* grad;
  float* s;    /* S = m / (1 - b1), the reference's stored first moment */
  float* v;    /* V = v / (1 - b2), the reference's stored second moment */
  int64_t numel;
  int32_t step_index; /* index into the device step-counter array */
  int32_t lr_index;   /* index into lr_device (0 when one rate serves all) */
} ttrl_adam_tensor;

/* Multi-tensor fused Adam step in the reference's S/V form
 * (ttrl/engine/optim/adam.py:93-134, scalars from
 * ttrl/engine/optim/scalars.py:13-27):
 *   t = steps[i] + 1;  V = g^2 + b2*V;  S = g + b1*S;
 *   p -= alpha_t * S / (sqrt(V) + eps_t)
 * with alpha_t = lr(1-b1)/(1-b1^t)/c, eps_t = eps/c, c = sqrt((1-b2)/(1-b2^t)),
 * evaluated on the device in double precision.
 * `steps` (int32, device) holds each tensor's update count; the launch
 * increments it, so the call can be replayed from a CUDA graph. `ticket` is
 * one device int32 owned by the caller, zero before the first call (the
 * kernel leaves it zero). `grad_scale` (device float, may be NULL)
 * multiplies every gradient first (the clip factor of
 * ttrl/algos/grads.py:29-43); weight_decay adds wd*p to g next
 * (adam.py:110-113). `lr_device` (device doubles, may be NULL) overrides
 * `lr` at execution time, tensor i reading lr_device[tensors[i].lr_index],
 * so a replayed graph follows a learning-rate schedule
 * (ttrl/algos/ppo/learn.py:54-56) and one launch can step the parameters of
 * several optimizers (SAC's policy and temperature, ttrl/algos/sac/
 * agent.py:218-238) that share betas, eps and weight decay but keep their
 * own rates and counters. `bias_table` (device doubles, may be NULL) holds
 * the bias terms of steps t = 1..bias_steps as pairs (1 - b1^t, c_t), the
 * host's own pow() results; a step beyond the table reads its last pair,
 * which must be the converged one (1, 1), so the table is finite. NULL: the
 * kernel evaluates pow() itself. Up to TTRL_ADAM_MAX_TENSORS tensors per
 * call. */
#define TTRL_ADAM_MAX_TENSORS 64
int ttrl_adam_step(const ttrl_adam_tensor* tensors, int count, int32_t* steps, int32_t* ticket,
                   const float* grad_scale, const double* lr_device, double lr, double b1,
                   double b2, double eps, double weight_decay, const double* bias_table,
                   int64_t bias_steps, ttrl_stream_t stream);

/* One tensor of a multi-tensor AdamW launch. bits 32: m and v are fp32 like
 * param. bits 8: m holds int8 and v uint8 codes, padded to whole blocks of
 * TTRL_ADAMW_BLOCK elements on a 4-byte boundary, and m_scale, v_scale one
 * fp32 a block (all zero for zero moments):
 *   m = m_scale * sign(c) (c / 127)^2,   v = v_scale * (c / 255)^4. */
#define TTRL_ADAMW_BLOCK 256
#define TTRL_ADAMW_MAX_TENSORS 384
typedef struct {
  float* param;
  const float* grad;
  void* m;
  void* v;
  float* m_scale; /* bits 8 */
  float* v_scale;
  int64_t numel;
  int32_t step_index; /* into the device step counters; every tensor its own, or shared
                         by tensors of one call */
  int32_t bits;       /* 32 or 8 */
} ttrl_adamw_tensor;

/* AdamW (decoupled weight decay) over up to TTRL_ADAMW_MAX_TENSORS tensors in
 * one launch:
 *   t = steps[i] + 1;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2;
 *   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
 * The step uses the new moments before they are rounded to codes. steps,
 * ticket, grad_scale and bias_table are ttrl_adam_step's; lr_device (one
 * device double, may be NULL) overrides lr at execution time. eps is at least
 * 2^-126, as the quotient is a float's. A value that is
 * not finite makes its block's 8-bit moments NaN. No reference counterpart
 * (its Adam adds the decay to the gradient, ttrl/engine/optim/adam.py:110-113). */
int ttrl_adamw_step(const ttrl_adamw_tensor* tensors, int count, int32_t* steps, int32_t* ticket,
                    const float* grad_scale, const double* lr_device, double lr, double b1,
                    double b2, double eps, double weight_decay, const double* bias_table,
                    int64_t bias_steps, ttrl_stream_t stream);

/* 8-bit moments to fp32 (pack 0) or fp32 moments to codes and scales (pack
 * 1), rounded as the step rounds them: what a checkpoint reads and writes. */
typedef struct {
  float* m32;
  float* v32;
  void* m8;
  void* v8;
  float* m_scale;
  float* v_scale;
  int64_t numel;
} ttrl_adamw_state;
int ttrl_adamw_state_convert(const ttrl_adamw_state* tensors, int count, int pack,
                             ttrl_stream_t stream);

/* out[0] = sum over tensors of sum(g^2), accumulated in double and reduced
 * in a fixed order (ttrl/algos/grads.py:13-26 grad_norm's float64 sum,
 * grad_sq_device at :46-61). When max_norm > 0 also writes
 * out[1] = max_norm/(norm+1e-6) if norm > max_norm else 1, the clip factor
 * of clip_grad_norm (ttrl/algos/grads.py:29-43). `grads`/`numels` are host
 * arrays of device pointers and counts, of any length (a launch for every
 * TTRL_ADAM_MAX_TENSORS); `out` is a device float[2];
 * `workspace` needs ttrl_grad_sqnorm_workspace_bytes and must start zeroed
 * (the kernel leaves its ticket zero). */
int ttrl_grad_sqnorm(const float* const* grads, const int64_t* numels, int count, float* out,
                     float max_norm, void* workspace, size_t workspace_bytes,
                     ttrl_stream_t stream);
size_t ttrl_grad_sqnorm_workspace_bytes(const int64_t* numels, int count);

/* ------------------------------------------------------- tape primitives */

/* Elementwise op codes of ttrl_ew. Binary ops read a and b; *_S ops combine
 * a with `scalar`; unary ops read a only. */
enum {
  TTRL_EW_ADD = 0, TTRL_EW_SUB = 1, TTRL_EW_MUL = 2, TTRL_EW_DIV = 3,
  TTRL_EW_ADD_S = 4, TTRL_EW_SUB_S = 5, TTRL_EW_RSUB_S = 6, TTRL_EW_MUL_S = 7,
  TTRL_EW_DIV_S = 8, TTRL_EW_RELU = 9, TTRL_EW_RELU_BW = 10, TTRL_EW_ABS = 11,
  TTRL_EW_SIGN = 12, TTRL_EW_NEG = 13, TTRL_EW_EXP = 14, TTRL_EW_LOG = 15,
  TTRL_EW_TANH = 16, TTRL_EW_SIGMOID = 17, TTRL_EW_SQRT = 18, TTRL_EW_SQUARE = 19,
  TTRL_EW_EQZ = 20, TTRL_EW_FILL = 21, TTRL_EW_COPY = 22, TTRL_EW_GT_S = 23,
  TTRL_EW_EQ = 24
};

/* out[i] = op(a[i], b[i], scalar) over a contiguous output of rank <= 4;
 * a and b are read through their own element strides (0 = broadcast).
 * One launch per tape op of ttrl/engine/ops/{elementwise,unary}.py
 * (add/sub/mul/div, relu/relu_bw, abs, sign, exp, log, tanh, sigmoid,
 * sqrt, square, eqz, full_like). */
int ttrl_ew(int op, const float* a, const int64_t* a_strides, const float* b,
            const int64_t* b_strides, float* out, const int64_t* shape, int ndim, float scalar,
            ttrl_stream_t stream);

enum { TTRL_RED_SUM = 0, TTRL_RED_MAX = 1, TTRL_RED_ARGMAX = 2 };

/* Reduce the middle axis of in viewed as [outer][n][inner] into
 * out[outer][inner] (argmax as an fp32 index, first maximum wins).
 * Sequential or fixed-tree order: deterministic. Replaces ttnn.sum /
 * ttnn.max / ttnn.argmax of ttrl/engine/ops/reduce.py:11-99. */
int ttrl_reduce(int op, const float* in, float* out, int64_t outer, int64_t n, int64_t inner,
                ttrl_stream_t stream);

/* dst (=|+=) src over a rank <= 4 box, both read through element strides.
 * Backs concat / split / slice (ttrl/engine/ops/shape.py). */
int ttrl_copy_strided(float* dst, const int64_t* dst_strides, const float* src,
                      const int64_t* src_strides, const int64_t* shape, int ndim, int accumulate,
                      ttrl_stream_t stream);

/* Self-check of the bounded waits every kernel uses: a wait on a barrier
 * that nothing completes gives up after about a second and records
 * the code 1001 in status[0]; the context stays usable.
 * No reference counterpart (ttnn ops do not time out). */
int ttrl_wait_probe(int* status, ttrl_stream_t stream);

/* dst = (1 - tau) * dst + tau * src, elementwise, in that operation order
 * (ttrl/algos/sac/targets.py:55-61, the Polyak blend). */
int ttrl_polyak(float* dst, const float* src, int64_t n, float tau, ttrl_stream_t stream);

/* Multi-tensor target-network update over `count` (dst, src, n) pairs in
 * one launch (a network's parameters need not be contiguous):
 *   TTRL_BLEND_COPY:   dst = src, bit for bit -- the DQN hard target copy
 *     (ttrl/algos/dqn/agent.py:205-208 -> ttrl/engine/nn/module.py:164-189,
 *     one ttnn.add(src, 0) per parameter in ttrl/engine/tensor/arena.py:35-47);
 *   TTRL_BLEND_POLYAK: dst = (1 - tau) * dst + tau * src, in the operation
 *     order of ttrl/algos/sac/targets.py:55-61 (PolyakSync._blend).
 * Pairs must not overlap one another. */
enum { TTRL_BLEND_COPY = 0, TTRL_BLEND_POLYAK = 1 };
typedef struct {
  float* dst;
  const float* src;
  int64_t n;
} ttrl_blend_pair;
int ttrl_blend_multi(const ttrl_blend_pair* pairs, int count, int mode, float tau,
                     ttrl_stream_t stream);

/* dst[i][:] = src[idx[i]][:] for n rows of `row` 4-byte words (fp32 or
 * int32 payloads): the minibatch gather of
 * ttrl/buffers/rollout.py:271-282, done on the device. */
int ttrl_gather_rows(const void* src, const int32_t* idx, void* dst, int n, int row,
                     ttrl_stream_t stream);

/* The same gather for up to TTRL_GATHER_MAX_JOBS arrays that share one
 * index list (a minibatch's actions, old log-probs, values, returns and
 * advantages), in one launch. */
#define TTRL_GATHER_MAX_JOBS 8
typedef struct {
  const void* src;
  void* dst;
  int32_t row;  /* 4-byte words per row */
  int32_t pad0;
} ttrl_gather_job;
int ttrl_gather_rows_multi(const ttrl_gather_job* jobs, int count, const int32_t* idx, int n,
                           ttrl_stream_t stream);

/* ------------------------------------------------------------------ losses */

/* One DQN update's loss head, fused: the online Q(s,a) gather, the
 * (double-)DQN bootstrap target (argmax of `q_sel` with the optional
 * action-mask penalty, value read from `q_tgt`, done mask, per-sample
 * discount), the Huber loss (optionally importance-weighted), its mean,
 * mean Q, optional |TD|, and dq = d loss / d q.
 * ttrl/algos/dqn/losses.py:77-140 with ttrl/engine/ops/functional.py:56-69,
 * ttrl/algos/mask.py:113-121. Vectors are [batch]; matrices [batch][actions]. */
int ttrl_dqn_loss(const float* q, const float* q_sel, const float* q_tgt, const float* onehot,
                  const float* rewards, const float* dones, const float* discounts,
                  const float* next_mask, const float* is_weights, float* loss, float* mean_q,
                  float* td_abs, float* dq, int batch, int actions, float delta, int accumulate,
                  ttrl_stream_t stream);

/* PPO's objective and its gradient, fused: log-softmax, new log-prob of the
 * taken actions, clipped surrogate, clipped value loss (x0.5), entropy
 * bonus, reduced by the mean (valid == NULL) or the masked mean over
 * `valid`; metrics[4] = {loss, policy_loss, value_loss, entropy};
 * dlogits = d loss / d logits, dvalue = d loss / d value.
 * ttrl/algos/ppo/loss.py:27-83 with ttrl/algos/ppo/policy.py:64-76 and
 * ttrl/engine/ops/functional.py:160-178. */
int ttrl_ppo_loss(const float* logits, const float* value, const int32_t* actions,
                  const float* old_logp, const float* adv, const float* returns,
                  const float* old_values, const float* valid, float* metrics, float* new_logp,
                  float* dlogits, float* dvalue, int batch, int actions_n, float clip_eps,
                  float value_clip_eps, float value_coef, float entropy_coef,
                  ttrl_stream_t stream);

/* SAC's heads, fused (each call is one launch; results equal the reference's
 * composed tape ops, rounding for rounding where the order of a sum allows).
 *
 * ttrl_sac_sample: the tanh-squashed Gaussian of ttrl/algos/sac/policy.py:
 * 30-40 with the log-density of ttrl/algos/gaussian.py:55-90 and the action
 * box of gaussian.py:150-165. log_std = clamp(log_std_raw, min, max) by the
 * relu identities of ttrl/engine/ops/select.py:54-63; u = mean +
 * exp(log_std) * noise; logp[b] = normal_logp(u) - sum(log(1 - tanh(u)^2))
 * - log_det; the env action tanh(u) * scale + centre lands in columns
 * [obs_dim, obs_dim + action_dim) of `joint` ([batch][obs_dim +
 * action_dim]), whose first obs_dim columns receive `obs` -- the critic's
 * concat(obs, action) input (ttrl/nets/fusion.py) built in the same launch.
 * With pack_joint != NULL the launch also writes [pack_obs | pack_act] rows
 * into pack_joint (the replayed batch's critic input). */
#define TTRL_SAC_MAX_CRITICS 8
int ttrl_sac_sample(const float* mean, const float* log_std_raw, const float* noise,
                    const float* scale, const float* centre, const float* obs, float* joint,
                    float* logp, int batch, int action_dim, int obs_dim, float log_std_min,
                    float log_std_max, float log_det, const float* pack_obs,
                    const float* pack_act, float* pack_joint, ttrl_stream_t stream);

/* Backward of ttrl_sac_sample: d_mean and d_log_std_raw (each written, or
 * added to when its accumulate flag is set) from d_action (element (b, d)
 * at d_action[b * d_action_ld + d]; NULL: zero) and d_logp ([batch]; NULL:
 * zero). The forward is recomputed from the same inputs. */
int ttrl_sac_sample_backward(const float* mean, const float* log_std_raw, const float* noise,
                             const float* scale, const float* d_action, int64_t d_action_ld,
                             const float* d_logp, float* d_mean, float* d_log_std_raw,
                             int accumulate_mean, int accumulate_log_std, int batch,
                             int action_dim, float log_std_min, float log_std_max,
                             ttrl_stream_t stream);

/* The twin-critic loss of ttrl/algos/sac/losses.py:46-76: alpha =
 * exp(*log_alpha); y = r + (1 - done) * discount * (min_i q_target[i] -
 * alpha * next_logp) (min by the relu identity); loss = 0.5 * sum_i
 * mean(w * (q[i] - y)^2) (w = is_weights, or 1 when NULL); dq[i] = d loss /
 * d q[i]; target = y; td_abs (NULL: skipped) = mean_i |q[i] - y|
 * (losses.py:30-43). All vectors [batch]; q, q_target, dq are host arrays of
 * n_critics device pointers. batch * n_critics * 4 bytes must fit 200 KB. */
int ttrl_sac_critic_loss(const float* const* q, const float* const* q_target, int n_critics,
                         const float* next_logp, const float* log_alpha, const float* rewards,
                         const float* dones, const float* discounts, const float* is_weights,
                         float* loss, float* alpha, float* target, float* const* dq,
                         float* td_abs, int batch, ttrl_stream_t stream);

/* The actor loss mean(alpha * logp - min_i q[i]) of ttrl/algos/sac/losses.py:
 * 79-84 with dq[i] and d_logp, and (alpha_loss != NULL) the temperature loss
 * -mean(log_alpha * (logp + target_entropy)) of losses.py:87-95 with its
 * gradient d_log_alpha. batch * 12 bytes must fit 200 KB. */
int ttrl_sac_actor_loss(const float* const* q, int n_critics, const float* logp,
                        const float* log_alpha, float target_entropy, float* loss,
                        float* const* dq, float* d_logp, float* alpha_loss,
                        float* d_log_alpha, int batch, ttrl_stream_t stream);

/* ------------------------------------------------------------------ acting */

/* The DQN acting choice over q[batch][n_actions]: greedy = the first maximum
 * over the columns with mask > 0.5 (mask == NULL: all columns), then
 * actions[b] = draws[b] < *eps ? alt_actions[b] : greedy. draws (uniform in
 * [0, 1), double) and alt_actions (exploring actions) are drawn by the caller
 * in the reference's order; draws == NULL acts greedily. eps is a device
 * double so a captured acting graph replays with the current epsilon.
 * Replaces the argmax_dim_detached + host np.where of
 * ttrl/algos/dqn/agent.py:97-119 and ttrl/algos/mask.py:95-110. */
int ttrl_epsilon_greedy(const float* q, const float* mask, const double* draws,
                        const int32_t* alt_actions, const double* eps, int32_t* actions, int batch,
                        int n_actions, ttrl_stream_t stream);

/* The PPO acting draw over logits[batch][n_actions]: log-softmax with the
 * operations of ttrl_ppo_loss, then the first maximum (uniforms == NULL) or
 * the inverse-CDF draw against uniforms[b] (probs = exp(logp) normalised,
 * action = number of cumulative probabilities below the uniform, clipped to
 * n_actions - 1); logp[b] (may be NULL) receives the chosen action's
 * log-prob. Replaces CategoricalPolicy.sample (ttrl/algos/ppo/policy.py:36-62)
 * after its device log_softmax. */
int ttrl_categorical_sample(const float* logits, const double* uniforms, int32_t* actions,
                            float* logp, int batch, int n_actions, ttrl_stream_t stream);

/* ------------------------------------------------------- prioritized replay */

/* Write back one batch's priorities into the float64 table [lanes][columns]
 * of (p + eps)^alpha: table[lanes[b]][cols[b]] = (|td_abs[b]| + eps)^alpha,
 * a pair drawn twice taking its last value, and *max_priority = max(
 * *max_priority, max |td_abs|). from_max != 0 writes (*max_priority +
 * eps)^alpha instead (a freshly written column; td_abs unused). A non-finite
 * |td| writes 1003 into `status` and leaves the table unchanged. td_abs is the
 * device output of ttrl_dqn_loss, so nothing is read back to the host.
 * Replaces PrioritySampler.update / on_write (ttrl/buffers/sampling.py:131-203)
 * behind write_back_priorities (ttrl/algos/offpolicy.py:136-145). */
int ttrl_per_update(double* table, int columns, const int32_t* lanes, const int32_t* cols,
                    const float* td_abs, int batch, double alpha, double eps,
                    double* max_priority, int from_max, int* status, ttrl_stream_t stream);

/* Each lane's run (positions p = 0 .. counts[l]-1, oldest first, column
 * (start[l] + p) % columns) summed in order into cdf[l][p] (float64, numpy's
 * cumsum order); totals[l] = the lane's sum. */
int ttrl_per_cdf(const double* table, int n_lanes, int columns, const int32_t* counts,
                 const int32_t* start, double* cdf, double* totals, ttrl_stream_t stream);

/* One draw per sample b within lane lane_of[b]: the first position whose cdf
 * exceeds uniforms[b] * (the lane's total), clipped to the run
 * (ttrl/buffers/sampling.py:221-227); writes the position, its column and its
 * table value (for the importance-sampling weight). */
int ttrl_per_draw(const double* cdf, const double* table, int columns, const int32_t* counts,
                  const int32_t* start, const int32_t* lane_of, const double* uniforms, int batch,
                  int32_t* positions, int32_t* cols, double* picked, ttrl_stream_t stream);

/* ----------------------------------------------------------------- rollout */

/* GAE-lambda over a [n_steps][n_envs] rollout, one lane per thread walking
 * t = n_steps-1 .. 0 in the reference's float32 operation order (bit-exact
 * with ttrl/buffers/rollout.py:195-227): delta = r + gamma*next*(1-done) - v;
 * gae = (delta + gamma_lam*(1-done)*gae) * valid (valid == NULL: 1);
 * advantages = gae, returns = gae + v, next = v; `next` starts at
 * last_values[n_envs]. gamma_lam is float32(gamma * lambda) as the reference
 * rounds it. */
int ttrl_gae(const float* rewards, const float* values, const float* dones, const float* valid,
             const float* last_values, float* advantages, float* returns, int n_steps,
             int n_envs, float gamma, float gamma_lam, ttrl_stream_t stream);

/* out = (adv - mean) / (std + 1e-8) with mean and (population) std over the
 * slots whose valid > 0 (valid == NULL: all), applied to every slot
 * (ttrl/buffers/rollout.py:269-270, ttrl/buffers/seqbatch.py:86-101). The
 * statistics accumulate in double in a fixed order; a rollout with no valid
 * slot writes 1002 into `status` and leaves `out` untouched. */
int ttrl_normalize_advantages(const float* advantages, const float* valid, float* out,
                              long long n, int* status, ttrl_stream_t stream);

/* --------------------------------------------------------------- recurrent */

/* One GRU step after its recurrent GEMM: with gi = x_t @ W_ih + b_ih and
 * gh = hm @ W_hh + b_hh (rows [batch][3*hidden], gate columns reset | update |
 * candidate), r = sigmoid(gi_r + gh_r), z = sigmoid(gi_z + gh_z),
 * n = tanh(gi_n + r * gh_n), out = (1 - z) * n + z * hm. gates[batch][3*hidden]
 * receives (r, z, n) for the backward; when hm_next != NULL it receives
 * out * (1 - start_next[b]) (start_next == NULL: out), the masked state
 * entering the next step. Each operation rounds as the op-by-op composition
 * of ttrl/engine/recurrent.py:86-94 does, so equal gi, gh give equal bits.
 * Replaces the split / sigmoid / tanh / mul / add / sub launches of
 * GRUCell.forward (ttrl/engine/recurrent.py:88-94) and the
 * apply_done_mask of GRU.forward (:164-165). */
int ttrl_gru_gates_fwd(const float* gi, const float* gh, const float* hm, const float* start_next,
                       float* out, float* gates, float* hm_next, int batch, int hidden,
                       ttrl_stream_t stream);

/* The backward of one step. dh = dout (NULL: 0) plus, when carry != 0,
 * dhm * (1 - start_next[b]) (the gradient reaching this step's output
 * through the next step's masked state). Writes d gi and d gh
 * ([batch][3*hidden]) and overwrites dhm with dh * z, the direct part of
 * d hm; the caller accumulates d gh @ W_hh^T onto it (ttrl_linear_dgrad with
 * accumulate = 1). Replaces the tape backward of the ops in
 * ttrl/engine/recurrent.py:88-94 and :164-165. */
int ttrl_gru_gates_bwd(const float* dout, float* dhm, const float* start_next, int carry,
                       const float* gates, const float* gh, const float* hm, float* dgi,
                       float* dgh, int batch, int hidden, ttrl_stream_t stream);

/* Nonzero when the sequence kernels below take this batch and hidden width
 * (hidden a multiple of 4, shared-memory slices that fit). Uses the current
 * device (after ttrl_init). */
int ttrl_gru_sequence_supported(int batch, int hidden);

/* The recurrent half of a whole GRU unroll in one launch of thread-block
 * clusters: for t = 0 .. steps-1, hm[t] = (t ? out[t-1] : h0) * (1 -
 * starts[t]) (starts == NULL: no mask), gh[t] = hm[t] @ W_hh + b_hh, the
 * gates of ttrl_gru_gates_fwd from gi[t] and gh[t], out[t] = the new state.
 * gi, gh, gates are [steps][batch][3*hidden]; hm, out [steps][batch][hidden];
 * starts [steps][batch]; w_hh [hidden][3*hidden]; b_hh [3*hidden]. gh is
 * summed in fp32 on the CUDA cores. Replaces the T-step loop of GRU.forward
 * (ttrl/engine/recurrent.py:160-168) after the input projection. */
int ttrl_gru_sequence_fwd(const float* gi, const float* h0, const float* starts,
                          const float* w_hh, const float* b_hh, float* gh, float* gates, float* hm,
                          float* out, int steps, int batch, int hidden, ttrl_stream_t stream);

/* Its backward through time in one launch: from dout [steps][batch][hidden]
 * (NULL: zero) and the forward's saved gates, gh and hm, writes d gi and d gh
 * ([steps][batch][3*hidden]) and, when dh0 != NULL, d h0. The weight
 * gradients are one GEMM each over all steps (ttrl_linear_wgrad of hm against
 * d gh, and of x against d gi). Replaces the tape backward of the T-step loop
 * (ttrl/engine/recurrent.py:160-168). */
int ttrl_gru_sequence_bwd(const float* dout, const float* starts, const float* w_hh,
                          const float* gates, const float* gh, const float* hm, float* dgi,
                          float* dgh, float* dh0, int steps, int batch, int hidden,
                          ttrl_stream_t stream);

/* out[b][:] = h[b][:] * (1 - start[b]) (start == NULL: a copy): the done mask
 * of ttrl/engine/ops/functional.py:40-46 (apply_done_mask) on a [batch][hidden]
 * state, used for the state entering step 0 and for d h0. */
int ttrl_gru_mask(const float* h, const float* start, float* out, int batch, int hidden,
                  ttrl_stream_t stream);

/* -------------------------------------------------------------- group norm */

/* Activations fused behind the norm. */
enum { TTRL_ACT_NONE = 0, TTRL_ACT_RELU = 1, TTRL_ACT_SILU = 2 };

/* y = act(hat * weight + bias) over `images` blocks of [spatial][channels]
 * channels-last rows (the rows ttrl_conv_fprop writes; spatial = 1: one row
 * an image; up to 65535 * 256 channels), hat = (x - mean) / sqrt(var + eps) with mean and (biased)
 * variance over the spatial * channels / groups elements of an image's group.
 * weight, bias: [channels], NULL for 1 and 0. stats ([images][groups][2]:
 * mean, 1 / sqrt(var + eps)) is what the backward reads; NULL: not written.
 * y may be x, and overlaps nothing else. `workspace` (ttrl_group_norm_workspace_bytes) is laid out as
 * the GEMM's: 64 KB of counters, zero before and after, then scratch, so one
 * buffer serves both. No reference counterpart (ttrl has no group norm; its
 * LayerNorm is ttrl/engine/layers.py:64-115). */
int ttrl_group_norm_fwd(const float* x, const float* weight, const float* bias, float* y,
                        float* stats, int images, int spatial, int channels, int groups, float eps,
                        int act, void* workspace, size_t workspace_bytes,
                        ttrl_stream_t stream);

/* Its backward from dy and the forward's x and stats: dx (may be dy), and
 * dweight, dbias ([channels], NULL: skipped; added to with their accumulate
 * flag), none over another operand. z is recomputed from x, so a ReLU's gate is the forward's. */
int ttrl_group_norm_bwd(const float* dy, const float* x, const float* weight, const float* bias,
                        const float* stats, float* dx, float* dweight, float* dbias, int images,
                        int spatial, int channels, int groups, int act, int accumulate_weight,
                        int accumulate_bias, void* workspace, size_t workspace_bytes,
                        ttrl_stream_t stream);
size_t ttrl_group_norm_workspace_bytes(int images, int spatial, int channels, int groups,
                                       int backward);

/* ------------------------------------------------------- linear attention */

/* Linear attention with a decay for each head, the memory whose unroll is
 * parallel in time:
 *   S_t = decay[h] (1 - starts[t]) S_{t-1} + k_t v_t^T,  out_t = scale q_t S_t
 * over time-major rows, as the GRU's: qkv is [steps][batch] rows of
 * [q: heads x key_dim | k: heads x key_dim | v: heads x value_dim], out
 * [steps][batch][heads * value_dim]. state (NULL: zero) and new_state (NULL:
 * not written) are [batch][heads][key_dim][value_dim]. starts
 * ([steps][batch], NULL: none): where it is not 0 the state is dropped before
 * the token, whatever it holds. A token's error is a few 2^-22 of the sum of
 * decay^n |q| |k| |v| that its output is made of (2-norms; in a column of v of
 * that column), whatever the size of other tokens, episodes and columns (a
 * chunk whose columns differ by more than about 2^17 is done in fp32, at ten
 * times its time). decay: [heads] floats in [0, 1]. key_dim,
 * value_dim up to 128. No result may overlap an operand. `workspace` is laid out as the GEMM's (64 KB of
 * counters, left as they are, then scratch). No reference counterpart (its
 * only memory is the GRU, ttrl/engine/recurrent.py:45-168). */
int ttrl_linear_attention_fwd(const float* qkv, const float* state, const float* starts,
                              const float* decay, float* out, float* new_state, int steps,
                              int batch, int heads, int key_dim, int value_dim, float scale,
                              void* workspace, size_t workspace_bytes, ttrl_stream_t stream);

/* Its backward: dqkv (like qkv, all of it) and dstate (NULL: not wanted) from
 * dout and dnew_state (NULL: zero); the decay has no gradient. No result may
 * overlap an operand. */
int ttrl_linear_attention_bwd(const float* dout, const float* dnew_state, const float* qkv,
                              const float* state, const float* starts, const float* decay,
                              float* dqkv, float* dstate, int steps, int batch, int heads,
                              int key_dim, int value_dim, float scale, void* workspace,
                              size_t workspace_bytes, ttrl_stream_t stream);
size_t ttrl_linear_attention_workspace_bytes(int steps, int batch, int heads, int key_dim,
                                             int value_dim);

/* The recurrent form, one token a lane: qkv [batch] rows, starts [batch], out
 * [batch][heads * value_dim]; new_state may be state. */
int ttrl_linear_attention_step(const float* qkv, const float* state, const float* starts,
                               const float* decay, float* out, float* new_state, int batch,
                               int heads, int key_dim, int value_dim, float scale,
                               ttrl_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* TTRL_B200_H */
