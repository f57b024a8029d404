/*
 * eif_hip_adapters.h -- low-rank adapters of many requests beside one shared projection, on one MI355X.
 *
 * A projection of `cols` inputs and `rows` outputs serves all requests; a request may have an adapter of its own, a product of two
 * thin matrices A [rank, cols] and B [rows, rank] and a scale, that is added to the projection's output. No counterpart in the
 * reference. As in eif_hip.h, pointers are DEVICE pointers unless a comment says otherwise, `stream` is a hipStream_t (NULL = the null
 * stream), and calls return 0 or a negative EIF_HIP_E_* code. The current device must be the one that the memory, the stream and
 * the adapters belong to (on another one than the adapters': EIF_HIP_E_ARG). Strides are in elements. No input may overlap
 * an output (but `base` and y).
 */
#ifndef EIF_HIP_ADAPTERS_H
#define EIF_HIP_ADAPTERS_H

#include <stddef.h>
#include <stdint.h>

#include "eif_hip.h"
#include "eif_hip_mx.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct eif_hip_adapters eif_hip_adapters;

/* Room for `slots` adapters of a projection [rows, cols], of ranks up to max_rank, their matrices kept in `type` (EIF_HIP_F32, _F16 or
 * _BF16, eif_hip_mx.h); all slots are empty. slots 1 .. 65536, max_rank 1 .. 256, rows and cols 1 .. 2^20, else EIF_HIP_E_LIMIT
 * (below 1: EIF_HIP_E_ARG). Synchronous; not inside a graph capture. */
int eif_hip_adapters_create(eif_hip_adapters **out, int slots, int rows, int cols, int max_rank, int type);
void eif_hip_adapters_destroy(eif_hip_adapters *a);

/* Puts an adapter into a slot, in the place of what it held: A [rank, lda >= cols], B [rows, ldb >= rank] of the adapters' type, host
 * pointers (src_on_device = 0; the elements between the rows are read too) or device pointers (1). rank 0 empties the slot (A and B are
 * not read). Not inside a graph capture. In the stream's order, and synchronous: it returns after the copy. From host memory it allocates
 * and frees device memory for the copy, which may wait for other streams' work. Calls of eif_hip_adapters_linear that are under way on
 * other streams meanwhile must not name this slot; other slots are not touched. */
int eif_hip_adapters_set(eif_hip_adapters *a, int slot, int rank, const void *A, int64_t lda, const void *B, int64_t ldb, float scale,
                         int src_on_device, void *stream);

/* Shape and device bytes (any pointer may be NULL). */
int eif_hip_adapters_info(const eif_hip_adapters *a, int *slots, int *rows, int *cols, int *max_rank, int *type, size_t *bytes);

/* y[m] = base[m] + scale B (A x[m]) with the adapter in slot[m], for M token rows x [M, ldx] of `type`.
 *   slot [M] int32: rows in any order of slots; a row whose slot is empty or outside of [0, slots) gets base[m].
 *   base [M, ldbase] FP32, e.g. the projection's output; it may be y itself (ldbase == ldy), or NULL (0).
 *   y [M, ldy] FP32.
 * The form goes by M and max_rank, since the host does not see the slots: up to 512 rows (256 where max_rank is more than 16) each row is
 * worked on by itself; of more rows those that share an adapter should lie together.
 * Products and sums in FP32, in an order that M and the shapes set, not the slots of other rows. An infinity or NaN in an adapter's
 * matrices reaches outputs of the rows that name it alone, which are infinite or NaN: which of the two goes by the form, since many rows
 * are multiplied in parts, whose zeros make NaN of an infinity. What of x and of A x lies below 2^-133 may be left out.
 * One launch; nothing is allocated and nothing kept, so that any number of calls may run at once and be captured into graphs. M up to
 * 2^24, else EIF_HIP_E_LIMIT. */
int eif_hip_adapters_linear(const eif_hip_adapters *a, const void *x, int type, int64_t ldx, const int32_t *slot, const float *base,
                            int64_t ldbase, float *y, int64_t ldy, int M, void *stream);

#ifdef __cplusplus
}
#endif

#endif
