/* C-ABI of libspnc_hip, second part: operators on device-resident rows around compiled kernels. They make up gated
 * mixtures of kernels, p(x) = sum_j w_j(x) p_j(x): a sum node whose weights depend on the row and of whose children each
 * row visits a few. The gate picks k experts a row, the rows are sorted by expert so that every kernel reads one
 * contiguous segment (spnc_hip_execute_device, spnc_hip.h), and the results come back in row order with weights
 * applied. Dropout marks features as missing for kernels compiled with marginalisation, or zeroes and scales activations.
 * The reference compiles one query at a time and has no counterpart of these.
 *
 * All pointers are device pointers unless stated otherwise, aligned to their elements; every call enqueues on `stream` (a
 * hipStream_t, NULL for the default stream) of the current device and does not wait, allocates nothing, keeps no state
 * between calls and may be captured into a graph. What a call writes must not overlap what it reads or writes elsewhere,
 * except where it is said; such calls are refused. Rows of one operand may lie between those of another. Functions
 * return 0 on success and a non-zero code on failure, with the message available from spnc_hip_last_error(); an error that
 * another call left for hipGetLastError is neither read nor cleared. Results do not depend on the order in which blocks
 * run: no atomics on results. */
#ifndef SPNC_HIP_ROWS_H
#define SPNC_HIP_ROWS_H

#include "spnc_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* element types of rows, values and weights */
enum { SPNC_HIP_FLOAT32 = 0, SPNC_HIP_FLOAT64 = 1, SPNC_HIP_FLOAT16 = 2, SPNC_HIP_BFLOAT16 = 3 };

#define SPNC_HIP_MAX_EXPERTS 1024u
#define SPNC_HIP_MAX_CHOICES 64u

/* flags of the gate */
enum {
  SPNC_HIP_GATE_ALL = 1, /* weights are normalised over all experts (default: over the chosen ones) */
  SPNC_HIP_GATE_LOG = 2  /* logarithms of the weights */
};

/* logits [n, experts], rows `stride` elements apart -> index int32 [n, k], weight [n, k] (float64 for float64 logits,
 * else float32): the k largest logits of a row in descending order, equal ones by ascending index, NaN above everything.
 * Minus infinity closes an expert to a row: it is never chosen, and slots left over hold index -1 and weight 0 (log
 * weight minus infinity). 1 <= k <= min(experts, SPNC_HIP_MAX_CHOICES), experts <= SPNC_HIP_MAX_EXPERTS, stride < 2^20. */
SPNC_HIP_API int spnc_hip_gate(const void* logits, int dtype, size_t n, unsigned experts, size_t stride, unsigned k, unsigned flags,
                               int32_t* index, void* weight, void* stream);

/* grad_weight [n, k] -> grad_logits [n, experts] (contiguous, the logits' type). index and weight are what
 * spnc_hip_gate returned; `logits` is read only under SPNC_HIP_GATE_ALL. Slots with index -1 pass no gradient. */
SPNC_HIP_API int spnc_hip_gate_backward(const void* logits, int dtype, size_t n, unsigned experts, size_t stride, unsigned k, unsigned flags,
                                        const int32_t* index, const void* weight, const void* grad_weight, void* grad_logits, void* stream);

/* Bytes of workspace spnc_hip_route needs for this many slots (n * k) and experts; 0 for small calls. */
SPNC_HIP_API size_t spnc_hip_route_workspace(size_t slots, unsigned experts);

/* index [slots] -> position [slots]: the row of the sorted buffer that holds the slot. A stable sort by expert: segment e
 * is the rows starts[e] ... starts[e] + counts[e] - 1, in ascending order of the slots; starts [experts + 1] are multiples
 * of `align`, starts[experts] is where the last segment ends, rounded up. An index outside [0, experts) is not routed:
 * position -1. slots + experts * (align - 1) must be below 2^31. */
SPNC_HIP_API int spnc_hip_route(const int32_t* index, size_t slots, unsigned experts, unsigned align, int32_t* position, int32_t* starts,
                                int32_t* counts, void* workspace, size_t workspace_bytes, void* stream);

/* out[position[i * k + j]] = rows[i] for all slots with 0 <= position < capacity: rows of row_bytes bytes, stride_bytes apart in `rows`,
 * contiguous in `out` [capacity]. zero_unused != 0 clears the rows of `out` that belong to no segment (starts and counts
 * as spnc_hip_route wrote them); otherwise they are left as they were and starts and counts may be NULL. A row is shorter
 * than 2 GiB, n * k and the capacity are below 2^31, here and below. */
SPNC_HIP_API int spnc_hip_dispatch(const void* rows, size_t n, size_t row_bytes, size_t stride_bytes, const int32_t* position, unsigned k,
                                   size_t capacity, const int32_t* starts, const int32_t* counts, unsigned experts, int zero_unused, void* out,
                                   void* stream);

/* out[i] = sum over j of weight[i * k + j] * values[position[i * k + j]], summed in 32 bits (64 for float64), in the order of
 * j: values [capacity, width] rows `stride` elements apart, out [n, width] contiguous. weight is float32, or float64 with
 * float64 values, or NULL for ones (the gradient of spnc_hip_dispatch). Slots with a position outside [0, capacity) are
 * left out; a row without slots becomes zero. */
SPNC_HIP_API int spnc_hip_combine(const void* values, int dtype, size_t capacity, size_t width, size_t stride, const int32_t* position, size_t n,
                                  unsigned k, const void* weight, int weight_dtype, void* out, void* stream);

/* grad_out [n, width], rows grad_stride elements apart -> grad_values [capacity, width] contiguous (rows of no segment
 * become zero) and grad_weight [n, k] (the weights' type; 0 where not routed). Either may be NULL. */
SPNC_HIP_API int spnc_hip_combine_backward(const void* values, int dtype, size_t capacity, size_t width, size_t stride, const int32_t* position,
                                           size_t n, unsigned k, const void* weight, int weight_dtype, const void* grad_out, size_t grad_stride,
                                           const int32_t* starts, const int32_t* counts, unsigned experts, void* grad_values, void* grad_weight,
                                           void* stream);

/* out[i] = log sum over j of exp(log_weight[i * k + j] + values[position[i * k + j]]): values [capacity] and out [n] float32 or
 * float64, log_weight float32 or float64. Slots that are not routed or whose log weight is minus infinity are left out, whatever
 * value stands there; a row without slots becomes minus infinity, as a sum node whose children are all impossible. share [n, k] of the values'
 * type, if not NULL, receives every slot's part of its row's sum for spnc_hip_combine_log_backward: 0 for slots that are left out and in
 * rows whose sum is empty. */
SPNC_HIP_API int spnc_hip_combine_log(const void* values, int dtype, size_t capacity, const int32_t* position, size_t n, unsigned k,
                                      const void* log_weight, int weight_dtype, void* out, void* share, void* stream);

/* grad_out [n] -> grad_values [capacity] (0 in rows of no segment) and grad_log_weight [n, k] of weight_dtype; either may be NULL. Both
 * are the output's gradient times the slot's share, 0 where that is 0. position is read for grad_values only. */
SPNC_HIP_API int spnc_hip_combine_log_backward(const void* share, int dtype, size_t capacity, const int32_t* position, size_t n, unsigned k,
                                               int weight_dtype, const void* grad_out, const int32_t* starts, const int32_t* counts,
                                               unsigned experts, void* grad_values, void* grad_log_weight, void* stream);

/* What a dropped element becomes. */
enum {
  SPNC_HIP_DROPOUT_ZERO = 0,    /* 0, and kept elements are multiplied by 1 / (1 - p) */
  SPNC_HIP_DROPOUT_MARGINAL = 1, /* NaN, a missing feature; kept elements stay as they are */
  SPNC_HIP_DROPOUT_MASK = 2     /* 0, kept elements stay as they are: the gradient of SPNC_HIP_DROPOUT_MARGINAL */
};

/* x [n, width] -> out [n, width], rows stride and out_stride elements apart; out may be x, with the same stride. Element e (counted without
 * the strides) is dropped where word e % 4 of Philox4x32-10 with key `seed` and counter (e / 4, offset), low words first,
 * is below round(p * 2^32). The mask is a function of seed, offset and e alone: the same call on the output's gradient
 * (ZERO, or MASK after MARGINAL) is the gradient. offset_device, if not NULL, points to the offset on the device and
 * replaces `offset`, so that a captured graph draws another mask at each replay. 0 <= p <= 1. */
SPNC_HIP_API int spnc_hip_dropout(const void* x, int dtype, size_t n, size_t width, size_t stride, void* out, size_t out_stride, double p, int mode,
                                  uint64_t seed, uint64_t offset, const uint64_t* offset_device, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* SPNC_HIP_ROWS_H */
