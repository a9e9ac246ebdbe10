/*
 * alpha_dense.h — C ABI of the dense operators that stand around the convolutions of alpha_conv.h in a training step:
 * the matrix product with its epilogue (a fully connected layer, or a 1x1 stride-1 convolution on the N*OH*OW rows of an
 * NHWC tensor) and its backward, the gated pair of projections of a feed-forward block and its backward, and clipping of
 * all gradients by their global norm.
 *
 * Conventions:
 *   - Element types: ALPHA_DENSE_F32, ALPHA_DENSE_BF16; every tensor of a call has the call's type (gradClip: one type per
 *     tensor). Sums are held in fp32 (the norm's in fp64 from the sums of 16 bytes' squares on) and rounded once, to the output's
 *     type; bf16 backward rounds deltaZ (deltaG, deltaU) to bf16, the matrix pipe's operand, before its products, deltaB is summed
 *     from the unrounded values.
 *   - Matrices are row-major, X[N,IC], W[OC,IC] (a filter W[OC,1,1,IC]), Y[N,OC]; `*_stride` is the distance of two rows
 *     in elements (>= the row's length, <= 2^22). N < 2^30, IC, OC <= 2^22 (OC of a gated pair <= 2^21); N * IC, 2 * N * OC and
 *     OC * IC, with IC and OC rounded up to 8, below 2^34. Any other size, any stride, pointers aligned to their element.
 *     Large bf16 products copy operands whose row length or stride is no multiple of 8 elements, or whose address is no
 *     multiple of 16 bytes, and a pair of filters of two strides may be copied, into the workspace; all others are read in
 *     place. A bf16 element is read with the 4-byte word it lies in.
 *   - N, IC and OC may be 0: an empty sum is 0 (IC = 0: Z = Bias; N = 0: deltaW and deltaB are zeros).
 *   - All pointers are DEVICE pointers, borrowed for the duration of the enqueued work. Nothing is allocated, freed or
 *     synchronised; scratch is supplied by the caller: alpha_*_workspace gives its bytes for a call's type and sizes (0 to 2^63-1,
 *     or -1 for sizes the call refuses), `workspace` is 256-byte aligned and may be NULL where that is 0. Kernels that
 *     share a workspace must not overlap on the device: one workspace per stream, one per captured graph that may run
 *     beside another.
 *   - `streams`, `length`: as in alpha_conv.h; everything is enqueued on streams[0], which belongs to the current device,
 *     as does the memory. Calls may be captured into a graph. Results are bit-identical from run to run.
 *   - Outputs must not overlap inputs, the workspace or each other, except where said.
 *   - Large fp32 products run on the bf16 matrix pipe as sums of three-part splits: six of the nine partial products, the
 *     left-out ones together below 2^-23 of a product. The split keeps all 24 bits of an operand of 2^-110 and more; of a
 *     smaller one, whose last parts would be below bf16's last subnormal, it keeps what is above 2^-134. Others are plain
 *     fp32. Infinities and NaN come out as in plain fp32 either way; what is not finite is computed again, so a product that is
 *     full of them takes three to four times as long.
 *
 * Return value: 0 on success, a hipError_t value, or ALPHA_DENSE_EINVAL; alpha_dense_last_error() has the thread's message.
 */
#ifndef ALPHA_DENSE_H
#define ALPHA_DENSE_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define ALPHA_DENSE_EINVAL 10001

#define ALPHA_DENSE_F32 0
#define ALPHA_DENSE_BF16 1

/* act(z): z; z > 0 ? z : k z; z (1 + erf(z / sqrt 2)) / 2; z / (1 + exp(-z)); 1 / (1 + exp(-z)). `k` is the leaky ReLU's
 * slope (k = 0: ReLU), ignored by the others. */
#define ALPHA_DENSE_ACT_NONE 0
#define ALPHA_DENSE_ACT_LEAKY_RELU 1
#define ALPHA_DENSE_ACT_GELU 2
#define ALPHA_DENSE_ACT_SILU 3
#define ALPHA_DENSE_ACT_SIGMOID 4

const char *alpha_dense_last_error(void);

/* Z = X W^T + Bias,  Y = act(Z) + R.
 * Bias[OC], R[N,OC] and Z[N,OC] may be NULL (Z is written where the backward will want it). Y may be R (same stride). */
int64_t alpha_matMul_fused_workspace(int type, int N, int IC, int OC);
int alpha_matMul_fused(const int64_t *streams, int length, int type,
                       const void *X, int64_t X_stride, const void *W, int64_t W_stride, const void *Bias,
                       int act, float k, const void *R, int64_t R_stride,
                       void *Z, int64_t Z_stride, void *Y, int64_t Y_stride,
                       int N, int IC, int OC, void *workspace, int64_t workspace_bytes);

/* Its backward: deltaZ = deltaY * act'(Z),
 *     deltaX = deltaZ W,  deltaW = deltaZ^T X,  deltaB[c] = sum_n deltaZ[n, c]   (the gradient of R is deltaY itself).
 * deltaX, deltaW, deltaB may be NULL (not wanted); X may be NULL without deltaW, W without deltaX, Z with
 * ALPHA_DENSE_ACT_NONE. The derivative of the leaky ReLU at 0 is k. */
int64_t alpha_dmatMul_fused_workspace(int type, int N, int IC, int OC);
int alpha_dmatMul_fused(const int64_t *streams, int length, int type,
                        const void *deltaY, int64_t deltaY_stride, const void *Z, int64_t Z_stride, int act, float k,
                        const void *X, int64_t X_stride, const void *W, int64_t W_stride,
                        void *deltaX, int64_t deltaX_stride, void *deltaW, int64_t deltaW_stride, void *deltaB,
                        int N, int IC, int OC, void *workspace, int64_t workspace_bytes);

/* G = X Wg^T + Bg,  U = X Wu^T + Bu,  H = act(G) * U: both projections, the activation and the product in one kernel.
 * Bg, Bu and the kept pre-activations G, U may be NULL (each for itself). */
int64_t alpha_gatedMatMul_workspace(int type, int N, int IC, int OC);
int alpha_gatedMatMul(const int64_t *streams, int length, int type,
                      const void *X, int64_t X_stride, const void *Wg, int64_t Wg_stride, const void *Bg,
                      const void *Wu, int64_t Wu_stride, const void *Bu, int act, float k,
                      void *G, int64_t G_stride, void *U, int64_t U_stride, void *H, int64_t H_stride,
                      int N, int IC, int OC, void *workspace, int64_t workspace_bytes);

/* Its backward: deltaG = deltaH * U * act'(G), deltaU = deltaH * act(G),
 *     deltaX = deltaG Wg + deltaU Wu,  deltaWg = deltaG^T X,  deltaWu = deltaU^T X,  deltaBg, deltaBu their column sums.
 * Outputs may be NULL (not wanted); X may be NULL without deltaWg and deltaWu, Wg and Wu without deltaX. */
int64_t alpha_dgatedMatMul_workspace(int type, int N, int IC, int OC);
int alpha_dgatedMatMul(const int64_t *streams, int length, int type,
                       const void *deltaH, int64_t deltaH_stride, const void *G, int64_t G_stride, const void *U, int64_t U_stride,
                       int act, float k, const void *X, int64_t X_stride,
                       const void *Wg, int64_t Wg_stride, const void *Wu, int64_t Wu_stride,
                       void *deltaX, int64_t deltaX_stride, void *deltaWg, int64_t deltaWg_stride,
                       void *deltaWu, int64_t deltaWu_stride, void *deltaBg, void *deltaBu,
                       int N, int IC, int OC, void *workspace, int64_t workspace_bytes);

/* The global norm of `count` gradients and clipping by it:
 *     norm = sqrt(sum over all tensors and elements of g^2),  c = min(1, max_norm / (norm + eps)),  dst = g * c.
 * types[i], lengths[i] (elements, >= 0), src[i], dst[i]: HOST arrays, read during the call; the tensors are dense device
 * memory aligned to their element, dst[i] of src[i]'s type, and dst[i] may be src[i] (in place) but no other src or dst: the
 * same gradient twice is refused where it would be scaled twice. dst may be NULL: only the norm. norm_c: two device floats,
 * {norm, c}, written; NaN and infinities follow the formula (a NaN makes c NaN; an infinite norm makes c 0 and the infinite
 * elements NaN), so a caller sees them in norm_c[0]. max_norm and eps are finite and >= 0, max_norm + eps > 0. */
int64_t alpha_gradClip_workspace(int count, const int64_t *lengths);
int alpha_gradClip(const int64_t *streams, int length, int count, const int *types, const int64_t *lengths,
                   const void *const *src, void *const *dst, float max_norm, float eps, float *norm_c,
                   void *workspace, int64_t workspace_bytes);

#ifdef __cplusplus
}
#endif
#endif /* ALPHA_DENSE_H */
