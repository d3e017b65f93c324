/*
 * cgdr_rms_norm.h -- C ABI of the root-mean-square norm that stands before
 * (with the residual's addition) and behind (with a silu gate) a recurrent
 * layer, on B200 (sm_100a).  Per row of D columns:
 *     z = x + residual                 rounded to x's type and stored
 *     y = z r weight silu(gate)        r = (mean(z^2) + eps)^(-1/2)
 * residual and gate are optional.  The norm is that of z as it is stored, so
 * the backward pass, which reads the stored z, is the derivative of what the
 * forward pass computed.
 *
 *     x, residual, gate, z, y   [R, D]  bf16, fp16 or fp32, one type
 *     weight                    [D]     the same type, or fp32
 * with D <= 16384, R < 2^31 - 4096, innermost dimensions contiguous and rows
 * less than 2^30 elements apart.  Rows whose address and length are multiples
 * of 16 bytes are read in 16-byte pieces.  Sums are held in fp32; y is rounded
 * once.
 *
 * Each call checks its arguments (no device work on failure) and enqueues
 * its kernels on `stream`, whose device must be current.
 */
#ifndef CGDR_RMS_NORM_H_
#define CGDR_RMS_NORM_H_

#include "cgdr_fwd_h.h"

#ifdef __cplusplus
extern "C" {
#endif

#define CGDR_DT_FP8_E4M3 6 /* cgdrDataType of an 8-bit output */

/* y in x's type (y_scale NULL), or in 8 bits: y is then CGDR_DT_FP8_E4M3 and
 * y_scale [R, D / group] fp32, contiguous, receives one scale per group of
 * `group` neighbouring columns,
 *     scale = max(amax |y|, 1e-12) / 448,   y = e4m3(y / scale),
 * where group is D, or 32, 64 or 128 and divides D.  residual, gate and z
 * may be NULL (z is required with a residual and refused without). */
cgdrStatus cgdrRmsNorm(
    const cgdrTensor* x, const cgdrTensor* weight, const cgdrTensor* residual, const cgdrTensor* gate, double eps,
    int64_t group, const cgdrTensor* y, const cgdrTensor* y_scale, const cgdrTensor* z, void* stream);

/* Bytes of device workspace that the backward pass needs (partial sums of
 * dweight; 0 when dweight is NULL). */
cgdrStatus cgdrRmsNormBackwardGetWorkspaceSize(const cgdrTensor* z, const cgdrTensor* dweight,
                                               uint64_t* workspace_size);

/* The gradients.  z is the stored sum (x itself without a residual), dy [R, D]
 * has its type and is required; dz [R, D] is the gradient that reaches z
 * directly (NULL: none).  With n = z r, a = silu(gate), u = dy weight a:
 *     dx = r (u - n mean(u n)) + dz     (the residual's gradient is the same)
 *     dweight = sum over rows of dy a n,   dgate = dy n weight silu'(gate)
 * dx, dweight (weight's type) and dgate (x's type) may each be NULL, not all.
 * dweight is summed in a fixed order.  The workspace must be 16-byte aligned. */
cgdrStatus cgdrRmsNormBackward(
    const cgdrTensor* z, const cgdrTensor* weight, const cgdrTensor* gate, double eps, const cgdrTensor* dy,
    const cgdrTensor* dz, const cgdrTensor* dx, const cgdrTensor* dweight, const cgdrTensor* dgate, void* workspace,
    uint64_t workspace_size, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* CGDR_RMS_NORM_H_ */
