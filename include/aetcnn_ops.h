/*
 * aetcnn_ops.h -- C-ABI of the MI355X (gfx950) HIP kernels for one CNN
 * training step of aet-cnn.  Plain pointers and sizes only; every pointer
 * argument named like a tensor is DEVICE memory unless stated otherwise.
 *
 * Each entry point replaces one operation of the reference's CPU path
 * (paths relative to /root/reference/src/com/ai/dnn/) with CPU-path
 * semantics; the reference's own GPU ("mtcs") path differs from its CPU path
 * (biased BN variance, other eps, 0.99 rolling momentum, beta gradient) and
 * is NOT what these functions compute.
 *
 * Conventions
 *  - tensors are fp32 NCHW, batch outermost: ((b*C + c)*H + h)*W + w
 *  - `stream` is a hipStream_t passed as void*; NULL = the null stream
 *  - functions return 0 on success or a negative ACH_E* code; nothing is
 *    synchronised unless the name says so
 *  - functions that need scratch take (ws, ws_bytes) and have a matching
 *    *_workspace() query; kernels never allocate
 */
#ifndef AETCNN_OPS_H
#define AETCNN_OPS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define ACH_OK 0
#define ACH_EINVAL (-1)     /* bad argument / shape                        */
#define ACH_EWORKSPACE (-2) /* workspace missing or too small               */
#define ACH_EHIP (-3)       /* HIP runtime error (ach_last_hip_error())     */
#define ACH_EUNSUPPORTED (-4)
#define ACH_ENAN (-5)       /* a NaN where the reference's CPU path exits    */

/* Activation ids = the reference's ActivationType order (Activation.h). */
#define ACH_LOGISTIC 0
#define ACH_RELU 1
#define ACH_LINEAR 3
#define ACH_LEAKY 7

typedef void *ach_stream_t;

/* ---- runtime plumbing (the reference's MtcsMem / MtcsStream roles:
 *      mtcs/MtcsTool.c:22-30, mtcs/MtcsData.c:20-28) ----------------------- */
const char *ach_version(void);
int ach_device_count(void);
int ach_set_device(int dev);
const char *ach_last_hip_error(void);
int ach_malloc(void **ptr, size_t bytes);
int ach_free(void *ptr);
int ach_host_alloc(void **ptr, size_t bytes); /* pinned host memory */
int ach_host_free(void *ptr);
int ach_memcpy_h2d(void *dst, const void *src, size_t bytes, ach_stream_t stream);
int ach_memcpy_d2h(void *dst, const void *src, size_t bytes, ach_stream_t stream);
int ach_memcpy_d2d(void *dst, const void *src, size_t bytes, ach_stream_t stream);
/* enqueue only (no synchronisation); truly asynchronous from pinned memory */
int ach_memcpy_h2d_async(void *dst, const void *src, size_t bytes, ach_stream_t stream);
int ach_stream_create(ach_stream_t *stream);
int ach_stream_destroy(ach_stream_t stream);
int ach_stream_sync(ach_stream_t stream);
int ach_device_sync(void);
/* events for timing (hipEvent_t as void*) */
int ach_event_create(void **ev);
int ach_event_destroy(void *ev);
int ach_event_record(void *ev, ach_stream_t stream);
int ach_event_elapsed_ms(void *start, void *stop, float *ms); /* syncs stop */
int ach_event_sync(void *ev);                         /* host waits for ev */
int ach_stream_wait_event(ach_stream_t stream, void *ev); /* stream waits for ev */

/* ---- BLAS-1 helpers (mtcs/MtcsTool.c:33-132; NData.setZero NData.c:232) */
int ach_fill(float *x, size_t n, float value, ach_stream_t stream);
int ach_axpy(size_t n, float alpha, const float *x, float *y, ach_stream_t stream);
int ach_scal(size_t n, float alpha, float *x, ach_stream_t stream);

/* ---- GEMM (Gemm.gemm, Gemm.c:116-144; Gemm.h:12-16) --------------------
 * Row-major C = ALPHA*op(A)*op(B) + BETA*C on fp32 MFMA.                  */
int ach_gemm(int TA, int TB, int M, int N, int K, float ALPHA,
             const float *A, int lda, const float *B, int ldb,
             float BETA, float *C, int ldc, ach_stream_t stream);

/* ---- im2col / col2im for one image (Im2Col.c:65-103, 155-192; the
 * signatures of Im2Col.h:10-15, 24-28, dilation included: window taps at
 * k*dilation, output size (in + 2*pad - (dilation*(k-1)+1))/stride + 1).
 * Dilation below 1 returns ACH_EINVAL.  (The conv entry points below take
 * no dilation: the cfg parser rejects dilated convolutions.)              */
int ach_im2col(const float *im, int channels, int height, int width,
               int kh, int kw, int ph, int pw, int sh, int sw,
               int dilation_h, int dilation_w, float *col, ach_stream_t stream);
/* col2im zeroes `im` first, as the reference does (Im2Col.c:162)          */
int ach_col2im(const float *col, int channels, int height, int width,
               int kh, int kw, int ph, int pw, int sh, int sw,
               int dilation_h, int dilation_w, float *im, ach_stream_t stream);

/* ---- convolution (ConvolutionalLayer.c:684-803, 906-947) ----------------
 * stride is the width stride (the layer's stride_x, ConvolutionalLayer.c:
 * 77-79) and stride_y the height stride, 0 meaning the same as stride; the
 * output is ((h + 2*pad - size)/stride_y + 1) x ((w + 2*pad - size)/stride
 * + 1) (ConvolutionalLayer.c:337-344).  With unequal strides every entry
 * point below runs the reference's per-image passes on the device -- the
 * forward im2col + GEMM (ConvolutionalLayer.c:790-803), the weight
 * gradient im2col + GEMM added into dw and the input gradient GEMM +
 * col2im (:913-945) -- with one image's column buffer as workspace, except
 * for a fully connected geometry (one output position, which no stride
 * moves), and ach_conv_bwd_data_prepared returns ACH_EUNSUPPORTED.       */
typedef struct {
    int batch, c, h, w;   /* input  [batch][c][h][w]                     */
    int n;                /* filters (output channels)                   */
    int size, stride, pad;/* square kernel, stride, padding (groups = 1) */
    int stride_y;         /* height stride; 0: the same as stride        */
} ach_conv_desc;

int ach_conv_out_h(const ach_conv_desc *d);
int ach_conv_out_w(const ach_conv_desc *d);
/* y = W * im2col(x), overwriting y        (ConvolutionalLayer.c:689,716-803) */
size_t ach_conv_fwd_workspace(const ach_conv_desc *d);
int ach_conv_fwd(const ach_conv_desc *d, const float *x, const float *w, float *y,
                 void *ws, size_t ws_bytes, ach_stream_t stream);
/* dx = col2im(W^T * dy), overwriting dx   (ConvolutionalLayer.c:933-945)   */
size_t ach_conv_bwd_data_workspace(const ach_conv_desc *d);
int ach_conv_bwd_data(const ach_conv_desc *d, const float *dy, const float *w, float *dx,
                      void *ws, size_t ws_bytes, ach_stream_t stream);
/* dw += sum_b dy_b * im2col(x_b)^T        (ConvolutionalLayer.c:913-929)   */
size_t ach_conv_bwd_filter_workspace(const ach_conv_desc *d);
int ach_conv_bwd_filter(const ach_conv_desc *d, const float *x, const float *dy, float *dw,
                        void *ws, size_t ws_bytes, ach_stream_t stream);
/* ach_conv_bwd_filter, then the weights' step of ConvolutionalLayer.update
 * (ConvolutionalLayer.c:959-980) on (w, dw): dw += decay_coef*w;
 * w += lr_coef*dw; dw *= momentum -- the results of ach_conv_bwd_filter
 * followed by ach_sgd_update(F*C*k*k, w, dw, ...), bit for bit, with the
 * update done in the pass that finishes dw (no pass of its own).  The
 * caller orders it after every reader of w: ach_conv_bwd_data_reads_w(d)
 * tells whether this layer's _prepared input gradient is one.  Same
 * workspace as ach_conv_bwd_filter.                                       */
int ach_conv_bwd_filter_sgd(const ach_conv_desc *d, const float *x, const float *dy, float *w,
                            float *dw, float decay_coef, float lr_coef, float momentum, void *ws,
                            size_t ws_bytes, ach_stream_t stream);
/* 1 if ach_conv_bwd_data_prepared (or ach_conv_bwd_data) reads w, 0 if it
 * reads only the flipped copy wft (stride 1, filters wider than 1x1, more
 * than 4 input channels)                                                   */
int ach_conv_bwd_data_reads_w(const ach_conv_desc *d);

/* ---- prepared filters -------------------------------------------------------
 * The conv GEMMs read the filter k-major (Wt[C*k*k][n]) and, for the stride-1
 * input gradient, flipped k-major (Wft[(f*k*k + t)*C + c] = W[f][c][k*k-1-t]).
 * ach_conv_fwd / ach_conv_bwd_data build these in the workspace on every
 * call; a caller that keeps them (the network refreshes all of them with one
 * ach_conv_prepare_filters launch per step) calls the _prepared variants.
 * wft may be NULL when not needed: stride > 1, or a 1x1 filter (including a
 * kernel covering the whole unpadded input), whose flipped copy is W itself.
 * A fully connected geometry (ach_conv_is_fully_connected: a kernel covering
 * the whole unpadded input, or a 1x1 filter on a 1x1 input) needs no copy at
 * all: ach_conv_prepare_filters leaves its wt untouched and the _prepared
 * forward reads its wt argument as the filter itself, so pass w there.
 * No counterpart in the reference, which has no such layouts.              */
typedef struct {
    ach_conv_desc desc;
    const float *w;   /* [n][c][size][size] */
    float *wt;        /* n*c*size*size floats */
    float *wft;       /* n*c*size*size floats or NULL */
} ach_filter_job;
int ach_conv_prepare_filters(int njobs, const ach_filter_job *jobs, ach_stream_t stream);
/* 1 for a fully connected geometry (see above), else 0                    */
int ach_conv_is_fully_connected(const ach_conv_desc *d);
/* workspace: ach_conv_fwd_workspace(d) / ach_conv_bwd_data_workspace(d)
 * bytes suffice (the _prepared calls use only the split-K part of it)      */
int ach_conv_fwd_prepared(const ach_conv_desc *d, const float *x, const float *wt, float *y,
                          void *ws, size_t ws_bytes, ach_stream_t stream);
/* The forward of a convolutional layer without batch-norm in one pass:
 * y = act(conv(x) + bias), the output-side steps of ConvolutionalLayer.
 * forward (ConvolutionalLayer.c:684-716, then IOData.addBias IOData.c:43-55
 * and activate IOData.c:60-72) applied to each sum in the GEMM epilogue
 * (or the split-K reduction) with the same fp32 arithmetic: the results
 * are those of ach_conv_fwd_prepared + ach_add_bias + ach_activate, bit for
 * bit.  bias may be NULL (no bias); activation is ACH_LOGISTIC, ACH_RELU,
 * ACH_LINEAR or ACH_LEAKY (else ACH_EUNSUPPORTED); the logistic activation
 * (a double exp per element) and, for 256-row tiles without a K split,
 * bias and activation run as separate passes inside the call.             */
int ach_conv_fwd_bias_act_prepared(const ach_conv_desc *d, const float *x, const float *wt,
                                   const float *bias, int activation, float *y, void *ws,
                                   size_t ws_bytes, ach_stream_t stream);
/* The same for a training step's forward: every sum on the fp32 matrix
 * instructions, so that a step's sums -- whose last bits decide branches of
 * activations and argmaxes of pools, which later steps amplify -- do not
 * depend on the rounding of the faster forms the other forward calls may
 * take.  bias NULL and ACH_LINEAR: ach_conv_fwd_prepared's form.           */
int ach_conv_fwd_train_prepared(const ach_conv_desc *d, const float *x, const float *wt,
                                const float *bias, int activation, float *y, void *ws,
                                size_t ws_bytes, ach_stream_t stream);
/* stride-1 only (ACH_EUNSUPPORTED otherwise); w is read for 1x1 filters,
 * wft otherwise                                                             */
int ach_conv_bwd_data_prepared(const ach_conv_desc *d, const float *dy, const float *w,
                               const float *wft, float *dx, void *ws, size_t ws_bytes,
                               ach_stream_t stream);

/* ---- bias (IOData.addBias IOData.c:43-55; BiasData.calcGrad BiasData.c:40-57) */
int ach_add_bias(float *out, const float *biases, int batch, int n, int spatial,
                 ach_stream_t stream);
/* bias_updates[c] += sum of delta over images and positions; the workspace
 * (ach_bias_grad_workspace bytes) holds double partial sums per image chunk */
size_t ach_bias_grad_workspace(int batch, int n, int spatial);
int ach_bias_grad(float *bias_updates, const float *delta, int batch, int n, int spatial,
                  void *ws, size_t ws_bytes, ach_stream_t stream);
/* The same gradient in two halves, for a pass that already writes the delta
 * (the activation gradient below, or a max-pool's input gradient): that
 * pass stores plane_sums[b][c] = sum over positions of delta[b][c][:]
 * (double [batch][n]: DnnUtils.sum of each image's plane, BiasData.c:
 * 52-56), and this call adds bias_updates[c] += sum over b ascending of
 * plane_sums[b][c] (in double, rounded once).                             */
int ach_bias_grad_planes(float *bias_updates, const double *plane_sums, int batch, int n,
                         ach_stream_t stream);

/* ---- batch-norm, training mode ------------------------------------------
 * Forward (forwardNormCPU NLayer.c:141-162 = NormData.calcVarianceAndMean
 * NormData.c:141-186, scalAxpyRollMeanAndRollVariance :224-229, normalize
 * :244-282).  `out` holds the conv output on entry; on return x = copy of it,
 * x_norm (optional, may be NULL) = (x-mean)/(sqrt(var)+1e-6), and
 * out = act(x_norm*scales + biases) where act is ACH_LINEAR for the plain op
 * or ACH_LEAKY / ACH_RELU to fuse the layer's activation (Activation.c:160).
 * mean/variance (unbiased) and rolling_mean/rolling_variance (.9/.1) are
 * updated.  `x` may equal NULL only if x_norm is also NULL and the caller
 * keeps the pre-BN tensor itself (pass it as `out` != x is required).        */
size_t ach_bn_workspace(int batch, int c, int spatial);
int ach_bn_train_fwd(float *out, int batch, int c, int spatial,
                     const float *scales, const float *biases,
                     float *mean, float *variance,
                     float *rolling_mean, float *rolling_variance,
                     float *x, float *x_norm, int activation,
                     void *ws, size_t ws_bytes, ach_stream_t stream);
/* Same, reading the pre-BN tensor from `x` and writing only `out`
 * (x is not copied): the layout the network driver uses.                   */
int ach_bn_train_fwd_from_x(const float *x, float *out, int batch, int c, int spatial,
                            const float *scales, const float *biases,
                            float *mean, float *variance,
                            float *rolling_mean, float *rolling_variance,
                            int activation, void *ws, size_t ws_bytes,
                            ach_stream_t stream);
/* Allocation-free variant of ach_bn_train_fwd_from_x.  No counterpart in
 * the reference: it is for callers that cannot allocate or pass scratch
 * memory (work recorded into a HIP graph, tight serving loops, harnesses
 * that forbid hipMalloc).  The per-(channel, image chunk) partial sums go to
 * a fixed device array of ACH_BN_NOALLOC_SCRATCH_BYTES that the library
 * holds on each device it runs on until the process ends; the call makes no
 * allocation of any kind.  Same arguments and results as
 * ach_bn_train_fwd_from_x without (ws, ws_bytes).  Limit: the partial sums
 * (ach_bn_workspace(batch, c, spatial) bytes) must fit the array, which
 * holds every shape with c <= 10922 channels; larger shapes return
 * ACH_EWORKSPACE with a message in ach_last_hip_error().  Every call on one
 * device shares that device's array: calls that overlap in time on one
 * device (e.g. on two streams) race and must be ordered by the caller.    */
#define ACH_BN_NOALLOC_SCRATCH_BYTES (256u * 1024u)
int ach_bn_train_fwd_from_x_noalloc(const float *x, float *out, int batch, int c, int spatial,
                                    const float *scales, const float *biases,
                                    float *mean, float *variance,
                                    float *rolling_mean, float *rolling_variance,
                                    int activation, ach_stream_t stream);
/* Inference (forwardNormCPU test branch, NLayer.c:155-160 ->
 * NormData.normalizeByRoll, NormData.c:291-326): out = act(((x - rolling_mean)
 * * inv) * scales + biases), inv = 1/(sqrt(rolling_variance) + 1e-6) in
 * double; statistics are not updated.  x may equal out.                    */
int ach_bn_infer(const float *x, float *out, int batch, int c, int spatial,
                 const float *scales, const float *biases, const float *rolling_mean,
                 const float *rolling_variance, int activation, ach_stream_t stream);
/* Conv-BN folding for inference (ConvolutionalLayer.fuseConvBatchnorm,
 * ConvolutionalLayer.c:983-1003): per filter f, r = sqrt((double)
 * rolling_variance[f] + 1e-5); biases[f] -= scales[f]*rolling_mean[f]/r and
 * weights[f][0..fsize) *= scales[f]/r, in double, rounded once to float.
 * weights is [filters][fsize] (fsize = C*k*k), updated in place.           */
int ach_conv_bn_fold(int filters, int fsize, float *weights, float *biases,
                     const float *scales, const float *rolling_mean,
                     const float *rolling_variance, ach_stream_t stream);
/* Backward (backwardNormCPU NLayer.c:246-278): scale_updates += sum(d*x_norm);
 * d *= scales; mean_delta, variance_delta; d <- normalize_delta.  No beta
 * gradient (the CPU path computes none).  If activation is ACH_LEAKY/RELU the
 * activation gradient (ConvolutionalLayer.c:898, Activation.c:233-239) is
 * applied to `delta` first, its sign taken from the recomputed BN output.
 * x_norm may be NULL (recomputed from x).  mean_delta/variance_delta may be
 * NULL.                                                                     */
int ach_bn_bwd(float *delta, int batch, int c, int spatial,
               const float *x, const float *x_norm,
               const float *mean, const float *variance,
               const float *scales, const float *biases, float *scale_updates,
               float *mean_delta, float *variance_delta, int activation,
               void *ws, size_t ws_bytes, ach_stream_t stream);

/* ---- activations (Activation.c:160-179 activate, :233-239 gradientArray) */
int ach_activate(float *x, size_t n, int activation, ach_stream_t stream);
int ach_gradient(const float *y, size_t n, int activation, float *delta,
                 ach_stream_t stream);
/* ach_gradient of a [batch][n][spatial] tensor (the same products, ACH_LINEAR
 * included: delta unchanged) that also stores the bias gradient's
 * plane_sums[b][c] of the result (ach_bias_grad_planes)                    */
int ach_gradient_planes(const float *y, int batch, int n, int spatial, int activation,
                        float *delta, double *plane_sums, ach_stream_t stream);

/* ---- max-pool (MaxPoolLayer.c:237-272 forward, :318-331 backward) --------
 * out size = (in + padding - size)/stride + 1, window offset -padding/2,
 * -FLT_MAX init, strict '>' (first max in row-major scan wins); indexes are
 * global flat input indices.  Backward adds into delta_in in ascending
 * output order, bit-identical to the reference's scatter loop.  With
 * accumulate = 0 the sums start from +0 instead of delta_in's contents (the
 * reference's delta is zeroed in forward, NNetwork.c:388-391), so a caller
 * whose delta_in is all zeros may skip that zeroing; delta_in is then only
 * written.                                                                 */
int ach_maxpool_out(int in, int size, int stride, int padding);
int ach_maxpool_fwd(const float *in, int batch, int c, int h, int w,
                    int size, int stride, int padding,
                    float *out, int32_t *indexes, ach_stream_t stream);
int ach_maxpool_bwd(const float *delta_out, const int32_t *indexes,
                    int batch, int c, int h, int w, int size, int stride, int padding,
                    float *delta_in, int accumulate, ach_stream_t stream);
/* The same pool with a width stride stride_x and a height stride stride_y
 * (MaxPoolLayer.c:40-41, 255-256: out w = (w + padding - size)/stride_x + 1,
 * h likewise with stride_y); equal strides take the calls above.           */
int ach_maxpool_fwd_xy(const float *in, int batch, int c, int h, int w, int size, int stride_x,
                       int stride_y, int padding, float *out, int32_t *indexes,
                       ach_stream_t stream);
int ach_maxpool_bwd_xy(const float *delta_out, const int32_t *indexes, int batch, int c, int h,
                       int w, int size, int stride_x, int stride_y, int padding, float *delta_in,
                       int accumulate, ach_stream_t stream);
/* A dropout layer that follows the max-pool and shares its output
 * (DropoutLayer.c:55-86, NetworkFactory.c:644-650), applied by the pool:
 * the forward writes the masked output (ach_maxpool_fwd + ach_dropout_fwd on
 * out), the backward masks delta_out as it reads it (ach_dropout_bwd on
 * delta_out + ach_maxpool_bwd; delta_out itself may be left unmasked) --
 * the same values bit for bit.  Fused into the 2x2 / stride
 * 2 kernels; other windows run the two steps inside the call.  (The network
 * loops of aetcnn_net.h run pool and dropout as separate layers, as the
 * reference does, so the shared delta is masked in place.)                */
int ach_maxpool_fwd_dropout(const float *in, int batch, int c, int h, int w,
                            int size, int stride, int padding, float *out, int32_t *indexes,
                            float probability, uint64_t seed, uint32_t iter, uint32_t layer,
                            ach_stream_t stream);
int ach_maxpool_bwd_dropout(float *delta_out, const int32_t *indexes,
                            int batch, int c, int h, int w, int size, int stride, int padding,
                            float *delta_in, int accumulate, float probability, uint64_t seed,
                            uint32_t iter, uint32_t layer, ach_stream_t stream);
/* ach_maxpool_bwd, then delta_in *= f'(y_in) with the previous layer's
 * output y_in and activation act_in (Activation.gradientArray,
 * Activation.c:233-239, the first step of that layer's backward,
 * ConvolutionalLayer.c:863-948) in the same pass: the same values, bit for
 * bit, as ach_maxpool_bwd + ach_gradient.  Used when the pool's input
 * gradient is that layer's whole delta.                                   */
int ach_maxpool_bwd_act(const float *delta_out, const int32_t *indexes,
                        int batch, int c, int h, int w, int size, int stride, int padding,
                        float *delta_in, int accumulate, const float *y_in, int act_in,
                        ach_stream_t stream);
/* ach_maxpool_bwd_act with accumulate = 0 (y_in may be NULL: no gradient)
 * that also stores the bias gradient's plane_sums[b][c] of the delta_in it
 * writes (ach_bias_grad_planes; double [batch][c]).  For pools whose output
 * planes are staged in LDS with at most 8 planes per workgroup (input
 * planes of 128+ pixels, output planes of at most 4096): ACH_EUNSUPPORTED
 * otherwise, with nothing launched.                                       */
int ach_maxpool_bwd_act_planes(const float *delta_out, const int32_t *indexes, int batch, int c,
                               int h, int w, int size, int stride, int padding, float *delta_in,
                               const float *y_in, int act_in, double *plane_sums,
                               ach_stream_t stream);
/* ach_maxpool_bwd_act_planes (plane_sums may be NULL here) for a relu or
 * leaky layer below, with the activation gradient taken from the pool's
 * own forward output `pooled` instead of the layer's output: a pixel that
 * receives a sum is the argmax of its windows and the window's output is
 * its value, so the results equal ach_maxpool_bwd_act_planes' bit for bit
 * while reading the pooled tensor instead of the pool's input.  `pooled`
 * must hold what ach_maxpool_fwd wrote (not masked in place since).
 * ACH_EINVAL for another activation; ACH_EUNSUPPORTED, with nothing
 * launched, for pools the plane-staged kernel does not take (as above).   */
int ach_maxpool_bwd_act_pooled(const float *delta_out, const int32_t *indexes, int batch, int c,
                               int h, int w, int size, int stride, int padding, float *delta_in,
                               const float *pooled, int act_in, double *plane_sums,
                               ach_stream_t stream);

/* ---- global average pool (AvgPoolLayer.c:29-46, 73-88) ----------------- */
int ach_avgpool_fwd(const float *in, int batch, int c, int spatial, float *out,
                    ach_stream_t stream);
int ach_avgpool_bwd(const float *delta_out, int batch, int c, int spatial,
                    float *delta_in, ach_stream_t stream);

/* ---- softmax + cross-entropy (SoftMaxLayer.c:47-119) ---------------------
 * output = softmax(in/temperature) per (image, group); if truth != NULL:
 * error = t ? -log(p) : 0, delta = t - p, *cost (device float) = sum(error).
 * Backward is ach_axpy(n, 1, delta, delta_prev) (SoftMaxLayer.c:313).      */
size_t ach_softmax_workspace(int batch, int groups);
int ach_softmax_xent(const float *in, int batch, int inputs, int groups,
                     float temperature, const float *truth,
                     float *output, float *delta, float *error, float *cost,
                     void *ws, size_t ws_bytes, ach_stream_t stream);

/* ---- operators on logits: log probabilities, distillation -----------------
 * No counterpart in the reference, whose softmax layer (SoftMaxLayer.c:
 * 47-119) knows one-hot truth and whose answers are probabilities and a top-k
 * taken on the host (DnnUtils.c:463-477).
 *
 * `logits` holds `rows` rows of `classes` values of `type`, row r at element
 * r*stride (stride 0: classes; else >= classes; what lies between the rows is
 * neither read nor written).  Any element address will do; rows may be 0.
 * z = x/temperature (positive, 1e-6 to 1e6).  Everything is computed in 32
 * bits or more and rounded once, to nearest even, where an output has fewer;
 * results do not depend on the run (no float atomics).
 *  - a logit of -inf is a masked class: its probability is 0
 *  - a row whose logits are all -inf has no distribution: log probabilities
 *    are -inf, ranks 0, the entropy, losses and gradients 0
 *  - a row with a NaN or a +inf gives NaN, and ranks and top ids of -1 (but
 *    for the rows that are said below to be set to 0)
 *  - a class id outside [0, classes) stands for "none" (padding)
 * Workspaces are aligned to 16 bytes and belong to one call at a time: calls
 * that may overlap, on two streams, need one each.  Outputs overlap neither
 * one another nor the inputs, but for what is said below.                  */
#define ACH_F32 0
#define ACH_BF16 1
#define ACH_F16 2
#define ACH_TOP_MAX 128 /* most alternatives, or teacher entries, of a row  */
typedef struct {
    int rows, classes;
    int type;             /* ACH_F32, ACH_BF16 or ACH_F16                    */
    float temperature;
    int64_t stride;       /* elements from one row to the next; 0: classes   */
} ach_logits_desc;
/* Any of the outputs may be NULL (top_ids and top_logprobs only with k 0):
 *   logprobs[r]   log softmax(z)[ids[r]]; 0 where ids[r] is none
 *   ranks[r]      number of classes with a larger logit than ids[r]'s; -1
 *                 where it is none
 *   entropy[r]    -sum p log p
 *   stats[r][2]   {max of x, log sum exp((x - max)/temperature)}, which
 *                 ach_logprobs_bwd reads
 *   top_ids[r][k], top_logprobs[r][k]
 *                 the k (at most ACH_TOP_MAX and classes) largest logits,
 *                 largest first, equal ones by ascending id
 * ids may be NULL if logprobs and ranks are.                               */
size_t ach_logprobs_workspace(const ach_logits_desc *d, int k);
int ach_logprobs_fwd(const ach_logits_desc *d, const void *logits, const int32_t *ids, int k,
                     float *logprobs, int32_t *ranks, float *entropy, float *stats,
                     int32_t *top_ids, float *top_logprobs, void *ws, size_t ws_bytes,
                     ach_stream_t stream);
/* dlogits[r][j] = 1/temperature * (dlogprobs[r]*([j == ids[r]] - p_j)
 *                                  - dentropy[r]*p_j*(log p_j + entropy[r]))
 * from the stats and (with dentropy) the entropy of ach_logprobs_fwd.
 * dlogprobs (with ids) or dentropy may be NULL, not both.  dlogits has the
 * logits' type and rows dstride apart (0: classes); it may be `logits`
 * itself with the same stride.  Rows whose ids[r] is none take no gradient
 * from dlogprobs[r]; rows with no gradient to take (that and/or zeros) are
 * set to 0 without reading their logits, whatever these hold.              */
int ach_logprobs_bwd(const ach_logits_desc *d, const void *logits, const int32_t *ids,
                     const float *stats, const float *entropy, const float *dlogprobs,
                     const float *dentropy, void *dlogits, int64_t dstride, ach_stream_t stream);
/* Distillation.  The teacher of row r is k entries (teacher_ids[r][k],
 * teacher_values[r][k] of teacher_type); entries whose id is none or repeats
 * an earlier one of the row are dropped.  With q = softmax(z):
 *   ACH_DISTILL_RENORM  values are logits, or log probabilities at
 *       temperature 1: p = softmax(values/temperature) over the row's
 *       entries; KD = sum p_i (log p_i - log q_i), 0 where no entry is left
 *   ACH_DISTILL_TAIL    values are log probabilities at this temperature
 *       (top_logprobs of ach_logprobs_fwd): p = exp(values), and all other
 *       classes form one more entry, of p_rest = max(0, 1 - sum p) against
 *       q_rest = their sum of q; KD = sum p_i (log p_i - log q_i)
 *       + p_rest (log p_rest - log q_rest), without the last term where q_rest
 *       has no class of finite logit
 *   loss[r] = row_weights[r] * (soft*temperature^2*KD
 *                               - hard*log softmax(x)[labels[r]])
 *   delta[r][j] = -d loss[r] / d x[r][j]   (the sign of ach_softmax_xent)
 *   *cost = sum of loss[r] (in double, rounded once)
 * Either term is left out where its factor is 0 (soft: the teacher may then
 * be NULL and k 0; hard: labels may be NULL); a label that is none has no
 * second term.  row_weights NULL: 1.  Rows of weight 0, and rows that are left
 * with neither an entry nor a label, have loss and delta 0, whatever their
 * logits hold; in other rows a NaN or a +inf makes both NaN.  delta (of the
 * logits' type, rows delta_stride apart, 0: classes; it may be `logits` itself
 * with the same stride), loss and cost may be NULL, not all three; cost and
 * delta need no loss array.                                                */
#define ACH_DISTILL_RENORM 0
#define ACH_DISTILL_TAIL 1
typedef struct {
    int k;                /* teacher entries per row, up to ACH_TOP_MAX      */
    int mode;
    int teacher_type;     /* of teacher_values                               */
    float soft, hard;
} ach_distill_desc;
size_t ach_distill_workspace(const ach_logits_desc *d, const ach_distill_desc *t);
int ach_distill_xent(const ach_logits_desc *d, const ach_distill_desc *t, const void *logits,
                     const int32_t *teacher_ids, const void *teacher_values,
                     const int32_t *labels, const float *row_weights, float *loss, void *delta,
                     int64_t delta_stride, float *cost, void *ws, size_t ws_bytes,
                     ach_stream_t stream);

/* ---- activation checkpoints in 8 bits --------------------------------------
 * No counterpart in the reference, whose layers keep every activation that
 * their backward reads in 32 bits.
 *
 * `rows` (0 to 2^30) rows of `features` (1 to 2^30) values of `type` (ACH_F32, ACH_BF16
 * or ACH_F16), row r at element r*stride (0: features; else >= features; what
 * lies between the rows is neither read nor written), at any element address,
 * are kept as one buffer of ach_checkpoint_bytes(), at an address that is a
 * multiple of 16:
 *   int8_t  codes[rows][F]      F: features rounded up to a multiple of 32
 *   uint8_t steps[rows][F/32]   one for each block of 32 codes
 * A value is code * 2^(step - 133): MXINT8 blocks of the OCP Microscaling
 * Formats, without code -128 and steps below 7.  For a block whose largest
 * magnitude is a, step is the smallest, from 7 to 254, with
 * rint(a * 2^(133 - step)) <= 127, and the codes are the values rounded to
 * nearest even, at most 2^(step - 134) off, that is a/127, and exact where a is
 * 0.  (Codes end at 127 where a is above 127.5*2^121; values below 2^-127
 * are 0.)  A block that holds a NaN or an infinity has step 255 and stands
 * for NaN throughout.  Codes behind a row's last value are 0.
 * ach_checkpoint_unpack writes the values, rounded to nearest even where the
 * type is narrower than they are and no further than its largest finite value.
 * A checkpoint overlaps neither x nor another tensor.                        */
typedef struct {
    int rows, features;
    int type;             /* of x                                            */
    int64_t stride;       /* elements from one row of x to the next          */
} ach_checkpoint_desc;
/* 0 for rows or features outside these ranges                              */
size_t ach_checkpoint_bytes(int rows, int features);
int ach_checkpoint_pack(const ach_checkpoint_desc *d, const void *x, void *checkpoint,
                        ach_stream_t stream);
int ach_checkpoint_unpack(const ach_checkpoint_desc *d, const void *checkpoint, void *x,
                          ach_stream_t stream);

/* ---- layer norm -------------------------------------------------------------
 * No counterpart in the reference, which normalises over the batch only (the
 * entry points above); the same roles: scales and biases per feature, the
 * scales' and biases' gradients added into *_updates.
 *
 * Rows as of a checkpoint: an image's (or a token's) features, normalised
 * among themselves.  eps from 1e-12 to 1.  Everything is computed in 32 bits
 * or more and rounded once where an output has fewer; results do not depend
 * on the run (no float atomics).  A row that holds a NaN or an infinity gives
 * NaN in all its outputs, statistics that are not finite, and NaN in
 * scale_updates (bias_updates are sums of delta alone); other rows are not
 * touched by it.  Workspaces are aligned to 16 bytes and belong to one call at
 * a time.  Outputs overlap neither one another nor the inputs, but for what is
 * said below.                                                              */
typedef struct {
    int rows, features;
    int type;             /* of x, y, delta and dx                           */
    float eps;
    int64_t stride;       /* elements from one row of x to the next          */
} ach_layernorm_desc;
/* mean = sum x / n, rstd = 1/sqrt(sum (x - mean)^2 / n + eps),
 * x_norm = (x - mean)*rstd, y = x_norm*scales + biases (float [features];
 * NULL: 1 and 0).  y has rows y_stride apart (0: features) and may be x itself
 * with the same stride.  Either of y, stats (float [rows][2], mean and rstd)
 * and checkpoint (x_norm in 8 bits, from the unrounded values) may be NULL,
 * not all three.                                                           */
size_t ach_layernorm_fwd_workspace(const ach_layernorm_desc *d);
int ach_layernorm_fwd(const ach_layernorm_desc *d, const void *x, const float *scales,
                      const float *biases, void *y, int64_t y_stride, float *stats,
                      void *checkpoint, void *ws, size_t ws_bytes, ach_stream_t stream);
/* From the stats and either x or the checkpoint of x_norm (the other NULL):
 *   g = delta*scales;  dx = rstd*(g - sum g / n - x_norm * sum(g*x_norm) / n)
 *   scale_updates[j] (+)= sum_r delta*x_norm;  bias_updates[j] (+)= sum_r delta
 * added to what is there with accumulate 1 (as ach_bn_bwd's), or replacing it
 * with accumulate 0 (rows 0 then gives zeros).  delta and dx have rows
 * delta_stride and dx_stride apart (0: features); dx may be delta itself with
 * the same stride.  dx, scale_updates and bias_updates may be NULL, not all
 * three; scales NULL: 1.  For dx alone, rows of up to 16384 values need no
 * workspace (ws NULL).                                                     */
size_t ach_layernorm_bwd_workspace(const ach_layernorm_desc *d);
int ach_layernorm_bwd(const ach_layernorm_desc *d, const void *delta, int64_t delta_stride,
                      const void *x, const void *checkpoint, const float *stats,
                      const float *scales, void *dx, int64_t dx_stride, float *scale_updates,
                      float *bias_updates, int accumulate, void *ws, size_t ws_bytes,
                      ach_stream_t stream);

/* ---- a fully connected layer's weight gradient from its input's checkpoint --
 * ach_conv_bwd_filter of a fully connected geometry with the input kept in 8
 * bits: dw[o][i] (+)= sum_r delta[r][o]*x[r][i], dw float [outputs][inputs]
 * without gaps, x the checkpoint of rows x inputs, delta rows of `outputs` values
 * of `type`, `stride` elements apart (0: outputs), at any element address; rows 0
 * to 2^30, inputs, outputs and stride up to 2^23.  accumulate as above (rows 0 and
 * accumulate 0: zeros).  Every product is exact and the sums are in 32 bits: an
 * fp32 delta is taken as three bf16 pieces (fp16: two), down to the last bit of
 * the smallest.  What an infinity or a NaN in delta, or a block of NaN in x, is
 * summed into is not finite; results do not depend on the run.  fp32 deltas or
 * sums near 2^111 and above, infinities and NaN cost time: what they are summed
 * into is done again without the matrix instructions.                      */
typedef struct {
    int rows, inputs, outputs;
    int type;             /* of delta                                        */
    int64_t stride;       /* elements from one row of delta to the next      */
} ach_fc_desc;
size_t ach_fc_bwd_filter_checkpoint_workspace(const ach_fc_desc *d);
int ach_fc_bwd_filter_checkpoint(const ach_fc_desc *d, const void *checkpoint, const void *delta,
                                 float *dw, int accumulate, void *ws, size_t ws_bytes,
                                 ach_stream_t stream);

/* ---- dropout (DropoutLayer.c:55-86) ---------------------------------------
 * r = u(seed, iter, layer, i) from a counter-based generator (SplitMix64
 * finaliser, top 24 bits); r < p -> 0 else x * 1/(1-p).  Same mask forward
 * and backward; nothing is stored.                                          */
float ach_dropout_uniform(uint64_t seed, uint32_t iter, uint32_t layer, uint32_t i);
int ach_dropout_fwd(float *x, size_t n, float probability, uint64_t seed,
                    uint32_t iter, uint32_t layer, ach_stream_t stream);
int ach_dropout_bwd(float *delta, size_t n, float probability, uint64_t seed,
                    uint32_t iter, uint32_t layer, ach_stream_t stream);

/* ---- NaN scan (the reference's isnan checks: NormData.normalize exits on a
 * NaN normalized value, NormData.c:273-276; ScaleData.addUpdatesToScale and
 * scaleUpdates abort on a NaN scale or scale update, ScaleData.c:51-54,
 * 67-70).  spans (device memory) lists nspans arrays; for every array that
 * holds a NaN, *flag = min(*flag, its tag), so with tags in checking order
 * *flag names the first offending array.  One launch for all the arrays;
 * the caller initialises *flag (e.g. to INT32_MAX) and reads it later.     */
typedef struct ach_nan_span {
    const float *p;
    uint64_t n;
    int32_t tag;
    int32_t reserved;
} ach_nan_span;
int ach_nan_scan(const ach_nan_span *spans, int nspans, int32_t *flag, ach_stream_t stream);

/* ---- SGD momentum / weight-decay update ----------------------------------
 * ConvolutionalLayer.update (ConvolutionalLayer.c:959-980):
 *   dW += -decay*batch*W; W += (lr/batch)*dW; dW *= momentum;
 *   b  += (lr/batch)*db;  db *= momentum;  (scales likewise, no decay)
 * scales/scale_updates may be NULL.                                        */
int ach_conv_update(size_t nweights, float *weights, float *weight_updates,
                    size_t n, float *biases, float *bias_updates,
                    float *scales, float *scale_updates,
                    int batch, float learning_rate, float momentum, float decay,
                    ach_stream_t stream);
/* One flat buffer: v += decay_coef*w; w += lr_coef*v; v *= momentum, with
 * decay_coef = -decay*batch (0 for no decay), lr_coef = lr/batch.          */
int ach_sgd_update(size_t n, float *w, float *v, float decay_coef, float lr_coef,
                   float momentum, ach_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif
