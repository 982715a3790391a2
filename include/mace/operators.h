/* Dense layer and layer norm, forward and backward, on device arrays (B200 build addition; no
 * counterpart in the reference, whose radial networks and node linears run only inside its
 * calculator).  They are the building blocks of the MH1 radial networks -- Linear, LayerNorm
 * (biased variance), SiLU -- as calls of their own, for networks that are trained or served
 * beside the model.
 *
 * Arrays are row major with the last index contiguous; ld* is the distance of two rows in
 * elements, at least the row's length.  All arrays of a call have one type and are device
 * memory of the current device; statistics (mean, rstd) are float.  Sums are accumulated in
 * float, and a result is rounded once, when it is written.  Every reduction has a fixed order:
 * equal calls give equal bits.
 *
 * Calls return 0, or -1 with the message in mace_last_error (same thread) and nothing launched.
 * They run asynchronously on `stream` (NULL: the default stream) without waiting, allocate
 * nothing and may be captured into a CUDA graph; the first call on a device sets that device
 * up and should come before any capture.  `workspace` is 16-byte aligned device memory of at
 * least the size that the matching *_workspace call gives for the same arguments; it may be
 * NULL where that is 0, its contents do not matter, and it is free again when the call's work
 * on the stream is done.  Calls that may run at the same time need workspaces of their own.
 * Outputs do not overlap inputs, the workspace or each other, with the exceptions named below.
 * rows may be 0.  Waits inside the kernels are bounded; one that ran out would show as NaN. */
#pragma once
#include <mace/export.h>
#ifdef __cplusplus
extern "C" {
#endif
enum { MACE_F32 = 0, MACE_BF16 = 1, MACE_F16 = 2 };
/* silu z / (1 + exp(-z)); gelu z Phi(z) (by the error function, not by tanh); relu max(z, 0) with
 * slope 0 at 0. */
enum { MACE_ACT_NONE = 0, MACE_ACT_SILU = 1, MACE_ACT_GELU = 2, MACE_ACT_RELU = 3 };

/* y = act(z) + residual with z = x weight^T + bias, for x [rows][inputs], weight
 * [outputs][inputs], bias [outputs] (or NULL), residual, y and z [rows][outputs] (residual or
 * z NULL: left out).  z, kept for mace_dense_backward, is written before the activation.
 * residual may be y itself (same address and ld).
 * float products run on the tensor cores as split fp16 pairs (but for up to 8 rows or outputs, few
 * inputs, and some unaligned rows: plain float arithmetic): per row and 64 consecutive inputs the largest magnitude sets
 * the scale, values down to 2^-29 of it keep 22 bits, and smaller ones are held to 2^-52 of it.
 * Infinities and NaN give what the sum gives (such results are summed again, which is slow where
 * there are many). */
MACE_EXPORT int mace_dense(int type, long long rows, long long inputs, long long outputs, const void *x,
                           long long ldx, const void *weight, long long ldw, const void *bias, int activation,
                           const void *residual, long long ldr, void *y, long long ldy, void *z, long long ldz,
                           void *workspace, long long workspace_bytes, void *stream);
/* Workspace bytes of mace_dense, or -1. */
MACE_EXPORT long long mace_dense_workspace(int type, long long rows, long long inputs, long long outputs,
                                           const void *x, long long ldx, const void *weight, long long ldw);
/* Gradients of mace_dense for the output gradient dy [rows][outputs]: with dz = dy act'(z),
 *   dx [rows][inputs] = dz weight, dweight [outputs][inputs] = dz^T x, dbias [outputs] = the
 * column sums of dz; each of dx, dweight and dbias may be NULL and is then not computed (x is
 * read for dweight only, weight for dx only).  z may be NULL where activation is none.  The
 * residual's gradient is dy.  With rows = 0, dweight and dbias are zero.  In 16-bit types, dz is
 * rounded to the type before the products of layers that run on the tensor cores, as a tensor
 * between two layers would be; dbias sums the float values. */
MACE_EXPORT int mace_dense_backward(int type, long long rows, long long inputs, long long outputs, const void *dy,
                                    long long lddy, const void *x, long long ldx, const void *weight,
                                    long long ldw, int activation, const void *z, long long ldz, void *dx,
                                    long long lddx, void *dweight, long long lddw, void *dbias, void *workspace,
                                    long long workspace_bytes, void *stream);
/* Workspace bytes of mace_dense_backward, or -1. */
MACE_EXPORT long long mace_dense_backward_workspace(int type, long long rows, long long inputs, long long outputs,
                                                    const void *dy, long long lddy, const void *x, long long ldx,
                                                    const void *weight, long long ldw, int activation);
/* y = act(xhat gamma + beta), xhat = (x - mean) rstd, rstd = 1 / sqrt(variance + eps), with mean
 * and (biased) variance over each row of x [rows][width].  gamma, beta [width] or NULL (1, 0).
 * mean, rstd [rows], kept for mace_layer_norm_backward, or both NULL.  y may be x itself (same
 * address and ld). */
MACE_EXPORT int mace_layer_norm(int type, long long rows, long long width, const void *x, long long ldx,
                                const void *gamma, const void *beta, float eps, int activation, void *y,
                                long long ldy, float *mean, float *rstd, void *stream);
/* Gradients of mace_layer_norm for dy [rows][width]: with dz = dy act'(xhat gamma + beta) and
 * g = dz gamma, dx = rstd (g - mean(g) - xhat mean(g xhat)), dgamma = sum over rows of dz xhat,
 * dbeta = sum over rows of dz; each of dx, dgamma and dbeta may be NULL.  gamma and beta as in
 * the forward call (beta is read only with an activation).  dx may be dy itself (same address
 * and ld).  With rows = 0, dgamma and dbeta are zero. */
MACE_EXPORT int mace_layer_norm_backward(int type, long long rows, long long width, const void *dy, long long lddy,
                                         const void *x, long long ldx, const float *mean, const float *rstd,
                                         const void *gamma, const void *beta, int activation, void *dx,
                                         long long lddx, void *dgamma, void *dbeta, void *workspace,
                                         long long workspace_bytes, void *stream);
/* Workspace bytes of mace_layer_norm_backward, or -1. */
MACE_EXPORT long long mace_layer_norm_backward_workspace(int type, long long rows, long long width);
#ifdef __cplusplus
}
#endif
