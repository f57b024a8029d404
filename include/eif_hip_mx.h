/*
 * eif_hip_mx.h -- microscaled 4-bit (MXFP4) operators on one MI355X: quantisation of rows, resident matrices, their
 * products with quantised token rows, and the products of token rows sorted by expert with a stack of matrices.
 *
 * The format (no counterpart in the reference): a row is cut into blocks of 32 columns, the last one filled with zeros.
 * A block has one scale byte b, the power of two 2^(b - 127) (b = 255: NaN, every value of the block is NaN), and 32 codes
 * of 4 bits, two to a byte, the even column in the low nibble: bit 3 is the sign, bits 0..2 the magnitudes
 * 0, 0.5, 1, 1.5, 2, 3, 4, 6.
 *
 * As in eif_hip.h, pointers are DEVICE pointers unless a comment says otherwise, `stream` is a hipStream_t (NULL = the null
 * stream), calls are asynchronous on it and return 0 or a negative EIF_HIP_E_* code. The current device must be the
 * one that the memory, the stream and the weight belong to (a product on another device than its weight's returns
 * EIF_HIP_E_ARG). Calls keep no memory between them besides the weights: any number of them may run at once, also on one
 * weight, and they may be captured into graphs (eif_hip_mx4_weight_create and _destroy, which allocate and free, may not).
 * Strides are in elements (codes and scales: bytes). No input may overlap an output. Pointers are aligned to their elements
 * where a call asks for no more, else EIF_HIP_E_ARG.
 */
#ifndef EIF_HIP_MX_H
#define EIF_HIP_MX_H

#include <stddef.h>
#include <stdint.h>

#include "eif_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of rows. */
enum { EIF_HIP_F32 = 0, EIF_HIP_F16 = 1, EIF_HIP_BF16 = 2 };

/* Columns of an operand row of the products: cols rounded up to a multiple of 256 (0 for cols < 1 or beyond 2^24). */
int eif_hip_mx4_kpad(int cols);

/* Rows x [rows, ldx] of `type` -> MXFP4. Per block: a = the largest magnitude; b = max(0, floor(log2 a) + 125), 0 where
 * a = 0; code = x / 2^(b - 127) rounded to the nearest magnitude (of two as near the one with the even code; beyond 6: 6),
 * with x's sign. A block that holds an infinity or NaN gets b = 255 and codes 0.
 *   codes [rows, ldc] (16-byte aligned, ldc a multiple of 16, >= kpad / 2) and scales [rows, lds] (8-byte aligned, lds a
 *   multiple of 8, >= kpad / 32): columns cols .. kpad - 1 get zero codes, blocks without columns scale 0. Bytes beyond are
 *   left as they were. Both may be NULL;
 *   values [rows, ldv] FP32 or NULL: what the codes stand for.
 * One launch up to 2^26 - 4 runs of 256 columns (a last one of fewer counts), several beyond. cols beyond 2^24, or
 * 2^33 - 3 such runs and more: EIF_HIP_E_LIMIT. */
int eif_hip_mx4_quant_rows(const void *x, int type, int64_t ldx, int rows, int cols, uint8_t *codes, int64_t ldc,
                           uint8_t *scales, int64_t lds, float *values, int64_t ldv, void *stream);

typedef struct eif_hip_mx4_weight eif_hip_mx4_weight;

/* `experts` matrices [rows, cols] in the format above (row r of matrix e: codes + (e rows + r) ldc, ldc >=
 * (cols + 1) / 2; scales alike, lds >= (cols + 31) / 32; any alignment) -> the GPU layout, resident on the current device
 * until eif_hip_mx4_weight_destroy. Host pointers (src_on_device = 0; the bytes between the rows are read too) or device pointers
 * (1). Synchronous. More than 4096 experts, 2^30 rows, 2^24 columns or 2^31 - 1 tiles of 16 rows of all experts, or sources of
 * 2^63 bytes and more: EIF_HIP_E_LIMIT. */
int eif_hip_mx4_weight_create(eif_hip_mx4_weight **out, int experts, int rows, int cols, const uint8_t *codes,
                              int64_t ldc, const uint8_t *scales, int64_t lds, int src_on_device, void *stream);
void eif_hip_mx4_weight_destroy(eif_hip_mx4_weight *w);

/* Shape of a weight, the padded columns of its operand rows and its device bytes (any pointer may be NULL). */
int eif_hip_mx4_weight_info(const eif_hip_mx4_weight *w, int *experts, int *rows, int *cols, int *kpad, size_t *bytes);

/* y [M, ldy] FP32 = A W^T (+ bias [rows], or NULL) of M token rows quantised as eif_hip_mx4_quant_rows leaves them (codes
 * [M, ldc], scales [M, lds], their alignment as there) and a weight of one matrix. FP32 sums of the exact products,
 * in an order that depends on the shapes alone. Sums below the smallest normal number may come out as 0, and a sum whose
 * partial sums leave FP32's range as an infinity or NaN.
 * glu != 0: the matrix stacks gate rows (0 .. rows/2 - 1) over up rows (rows/2 .. rows - 1); y [M, rows/2] =
 * SiLU(g) u = (g / (1 + e^-g)) u of the two products with their biases, the exponential and the quotient with the GPU's own
 * instructions: of the FP32 sums g and u, within (2^-21 + 2^-23 |g|) |y| + 2^-119 |u| + 2^-149 (below g = -87.3 y may be 0).
 * rows a multiple of 32, else EIF_HIP_E_LIMIT.
 * M beyond 2^30, and products that take 2^32 threads and more (256 for 32 to 128 token rows and 128 or 256 matrix rows;
 * of up to 16 token rows a matrix, and of small matrices, 512 for 16 or 32 and 16 to 128): EIF_HIP_E_LIMIT. */
int eif_hip_mx4_linear(const eif_hip_mx4_weight *w, const uint8_t *codes, int64_t ldc, const uint8_t *scales, int64_t lds,
                       const float *bias, int glu, float *y, int64_t ldy, int M, void *stream);

/* The same for M <= 8 token rows x [M, ldx] of `type`, quantised within the call: one launch, the result of
 * eif_hip_mx4_quant_rows and eif_hip_mx4_linear but for the order of the sums. More rows, or more than 16384
 * columns: EIF_HIP_E_LIMIT (use the two calls). */
int eif_hip_mx4_linear_rows(const eif_hip_mx4_weight *w, const void *x, int type, int64_t ldx, const float *bias, int glu,
                            float *y, int64_t ldy, int M, void *stream);

/* Products by expert: the rows [offsets[e], offsets[e + 1]) of y [M, ldy] take matrix e of the weight (and bias
 * [experts, rows] or NULL, and glu as above). offsets [experts + 1] int32 in device memory, non-decreasing, taken as if
 * cut to [0, M]; experts may have no rows. Row i of y takes the quantised row row_index[i] (int32 in device memory; NULL:
 * i) of `rows_in` rows. Rows of y before offsets[0] and from offsets[experts] on, and rows whose index is not in
 * [0, rows_in), are left as they were. The form goes by M / experts, since the host does not see the offsets: up to 16 rows an
 * expert on average read a matrix once for every 16 rows that it has, which is slow where many rows meet in one expert.
 * (Where offsets decrease, so that ranges overlap, it is open which of their rows are written, and with whose products.) */
int eif_hip_mx4_linear_grouped(const eif_hip_mx4_weight *w, const uint8_t *codes, int64_t ldc, const uint8_t *scales,
                               int64_t lds, int rows_in, const int32_t *row_index, const int32_t *offsets,
                               const float *bias, int glu, float *y, int64_t ldy, int M, void *stream);

#ifdef __cplusplus
}
#endif

#endif
