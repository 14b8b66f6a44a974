/*
 * nsd_mx.h -- C ABI of the microscaled (OCP MX) weights: 4-bit weights, 8-bit
 * activations, and the products of the two, for the projections of a layer.
 *
 * A row is cut into blocks of 32 values along the inner dimension (n_in, a
 * multiple of 32).  A block is one scale byte s, which stands for 2^(s - 127)
 * (255: NaN, every value of the block), and 32 codes:
 *
 *   MXFP4 (weights)      E2M1: 0 .5 1 1.5 2 3 4 6 and their negatives.  Scale:
 *                        floor(log2(m)) - 2 with m the block's largest
 *                        magnitude; values round to the nearest code, ties to
 *                        the even one, past 6 to 6.
 *   MXFP8 (activations)  E4M3 (largest 448).  Scale: the smallest power of two
 *                        with m <= 448 times it; nearest, ties to even.
 *
 * A block of zeros has scale byte 0, one with an infinity or a NaN 255.  The
 * reference has no counterpart (its projections are fp16 `linear` calls,
 * swiftLLM/swiftllm/worker/kernels/linear.py:3-12).
 *
 * Kernel layouts (the byte counts are in nsd_mx_bytes), over tiles of 16 rows x 128
 * k (the last ones padded with zero codes; T = ceil(n_in / 128) tiles a row):
 *   codes  4 bits: [row tile][T][4 blocks of 32 k][16 rows][16 bytes, even k in
 *          the low half]; 8 bits: [row tile][T][8 runs of 16 k][16 rows][16 bytes]
 *   scales [ceil(T / 4)][row tile][4 blocks][16 rows][4 tiles of k]
 *
 * Every entry point follows nsd_attn.h's contract: stream-ordered, no host
 * synchronisation, no allocation, an int status, nsd_last_error().  Pointers
 * are 16-byte aligned.
 */
#ifndef NSD_MX_H
#define NSD_MX_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define NSD_DTYPE_F16 0
#define NSD_DTYPE_BF16 1
#define NSD_DTYPE_F32 2

/* Bytes of the codes and the scales of n_rows x n_in values at `bits` (4 or 8) bits. */
int nsd_mx_bytes(int bits, int64_t n_rows, int64_t n_in, int64_t* codes, int64_t* scales);

/*
 * nsd_mxfp4_quantize: w [n_out, n_in] row-major (dtype NSD_DTYPE_*) to MXFP4.
 * nsd_mxfp4_pack: the same from row-major codes [n_out, n_in / 2] (even k in
 * the low half) and scale bytes [n_out, n_in / 32], as checkpoints hold them.
 * nsd_mxfp4_dequantize: the values, row-major, in `dtype`, rounded to nearest
 * where it does not hold them (bf16 and fp32 hold all that a quantiser makes).
 * None works in place: buffers that overlap are refused (NSD_ERR_INVALID).
 */
int nsd_mxfp4_quantize(const void* w, int dtype, int64_t n_out, int64_t n_in, void* codes, void* scales,
                       void* stream);
int nsd_mxfp4_pack(const void* row_codes, const void* row_scales, int64_t n_out, int64_t n_in, void* codes,
                   void* scales, void* stream);
int nsd_mxfp4_dequantize(const void* codes, const void* scales, int64_t n_out, int64_t n_in, void* out, int dtype,
                         void* stream);

/* The same for activations: x [n_rows, n_in] fp16 to MXFP8, and back. */
int nsd_mxfp8_quantize(const void* x, int64_t n_rows, int64_t n_in, void* codes, void* scales, void* stream);
int nsd_mxfp8_dequantize(const void* codes, const void* scales, int64_t n_rows, int64_t n_in, void* out, int dtype,
                         void* stream);

/*
 * nsd_mxfp4_linear: y [n_rows, n_out] fp16 = fp16(sum over k of X[r][k] W[n][k]),
 * W the MXFP4 values and X the MXFP8 values of x [n_rows, n_in] fp16, quantised
 * in the call; or, with x null, the ones given as x_codes and x_scales.  Sums are
 * held in fp32; among eight products that the matrix instruction adds at a time,
 * bits 13 below the exponent of the largest are cut.
 *
 * nsd_mxfp4_up_gate_silu_and_mul: y [n_rows, inter] fp16 = fp16(up * g / (1 +
 * exp(-g))) in fp32, up and g the products with weight rows j and inter + j of
 * a [2 * inter, n_in] weight; inter a multiple of 16.
 *
 * y must not overlap x, the weight or the workspace, nor the workspace x or the
 * weight (NSD_ERR_INVALID).  The same call gives the same bits; in a batch of
 * another size, or given as codes instead of fp16, a row's sums may be added in
 * another order (another kernel or split of k serves them) and end in another
 * last place.  n_rows up to 2^21, n_out up to 2^27, n_in up to 2^20.
 *
 * workspace: nsd_mx_workspace bytes for the call's shape on the current device
 * (n_out: the weight's rows; gated: of nsd_mxfp4_up_gate_silu_and_mul; quantised:
 * x is given as codes; 0 for no rows), contents irrelevant; calls that overlap
 * each need their own.
 */
int nsd_mx_workspace(int64_t n_rows, int64_t n_out, int64_t n_in, int gated, int quantised, int64_t* bytes);
int nsd_mxfp4_linear(const void* x, const void* x_codes, const void* x_scales, const void* w_codes,
                     const void* w_scales, void* y, int64_t n_rows, int64_t n_out, int64_t n_in, void* workspace,
                     int64_t workspace_bytes, void* stream);
int nsd_mxfp4_up_gate_silu_and_mul(const void* x, const void* x_codes, const void* x_scales, const void* w_codes,
                                   const void* w_scales, void* y, int64_t n_rows, int64_t inter, int64_t n_in,
                                   void* workspace, int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* NSD_MX_H */
