/* ssla_ops.h -- C ABI of the recurrent-state operators of libssla_b200.so:
 * linear attention with a decay per head (chunked and one token at a time),
 * the 8-bit cache of recurrent states, and the channels-last group norm with
 * an activation.
 *
 * Conventions of ssla_b200.h: device pointers are global-memory pointers of
 * `device`, `stream` is a cudaStream_t (NULL = the legacy default stream),
 * every call is asynchronous on it, returns SSLA_OK or an SSLA_ERR_* code
 * and never aborts; ssla_last_error() gives the message.  Arguments are
 * checked before any CUDA call.  Calls keep nothing between them: what a
 * call needs beyond its arguments is in the workspace that the caller hands
 * it, so calls on different streams or in different captured graphs never
 * share memory unless the caller lets them.
 */
#ifndef SSLA_OPS_H
#define SSLA_OPS_H

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

enum { SSLA_DT_F32 = 0, SSLA_DT_BF16 = 1, SSLA_DT_F16 = 2 };
enum { SSLA_FMT_INT8 = 0, SSLA_FMT_E4M3 = 1 };
enum { SSLA_ACT_NONE = 0, SSLA_ACT_SILU = 1 };

enum { SSLA_LINATTN_MAX_DK = 128, SSLA_LINATTN_MAX_DV = 256 };

/* Linear attention.  For head h of a sequence, with 32-bit state S [dk][dv]:
 *     S <- exp(decay) S + k v^T,   out = scale * S^T q      (token by token)
 * Rows are tokens.  q, k: [n_rows][q_heads or k_heads][dk]; v, out:
 * [n_rows][heads][dv]; the last index is contiguous, row and head strides are
 * in elements.  Head h reads query head h / (heads / q_heads), keys alike.
 * decay: logarithms, at most 0, strides decay_row and decay_head (decay_row 0:
 * one decay per head); -infinity clears the state before the token, NaN and
 * infinities in it too (where there are any, the chunked form goes through
 * that part of the sequence token by token: 0.7 to 3.5 us a token).
 * state: [n_slots][heads][dk][dv], contiguous, updated in place.  `out` and
 * `state` overlap neither each other nor an input (the address ranges are
 * compared). */
typedef struct SslaLinAttn {
    const void *q, *k, *v;
    void* out;
    const float* decay;
    float* state;
    long long q_row, q_head, k_row, k_head, v_row, v_head, out_row, out_head, decay_row, decay_head;
    int n_rows, heads, q_heads, k_heads, dk, dv;
    int dtype;                 /* SSLA_DT_* of q, k, v and out */
    int n_slots;
    int device;
    float scale;
} SslaLinAttn;

/* Chunked form: sequence i is the `lengths[i]` rows from `offsets[i]`
 * (lengths NULL: up to offsets[i + 1], n_seq + 1 offsets; otherwise n_seq).
 * Sequence i starts from and updates state slot slots[i] (-1: starts from
 * zero, the last state is dropped; slots NULL: slot i); no slot occurs twice.
 * offsets, lengths and slots are host arrays, as a drain's part_offsets are.
 * Sequences may not overlap; rows outside all of them are left as they were,
 * and so is the state of a sequence of length 0.  state may be NULL if every
 * slot is -1.  A token's non-finite value makes the outputs of its own and
 * later tokens non-finite where they depend on it, never earlier ones.
 * `workspace`: ssla_linattn_chunk_workspace bytes, 16-byte aligned, apart from
 * the tensors. */
int ssla_linattn_chunk(const SslaLinAttn* a, const int* offsets, const int* lengths, const int* slots, int n_seq,
                       void* workspace, size_t workspace_bytes, void* stream);
int ssla_linattn_chunk_workspace(const SslaLinAttn* a, const int* offsets, const int* lengths, int n_seq,
                                 size_t* bytes);

/* Status bits of the chunked form's kernels on `device` since the last call
 * (0: fine).  SSLA_LINATTN_TIMED_OUT: a bounded wait inside a kernel ran out,
 * and what the calls since wrote is not valid.  Synchronises the device. */
enum { SSLA_LINATTN_TIMED_OUT = 1 };
int ssla_linattn_status(int device, unsigned* status);

/* Recurrent form: one token per row, at most 65535 rows.  Row r updates state slot slots[r]
 * (device array; NULL: slot r, n_rows <= n_slots).  Rows that name the same
 * slot are applied in row order.  A slot outside [0, n_slots) marks a padding
 * row: its output is zero and no state is touched.  slots overlaps neither
 * `out` nor `state`. */
int ssla_linattn_step(const SslaLinAttn* a, const int* slots, void* stream);

/* 8-bit cache of recurrent states.  A state is `rows` rows of `cols` values;
 * each `block` consecutive values of a row (the last block may be shorter)
 * share one 32-bit scale = max|x| / 127 (int8) or / 448 (e4m3), and a code is
 * x / scale, rounded to 32 bits and then to the format's nearest value (ties
 * to even); where 127 (448) x scale would overflow the scale is the next
 * smaller float; all-zero blocks have scale 0 and codes 0, blocks holding a
 * non-finite value the scale NaN and codes 0.
 * codes: [n_slots][rows][cols] bytes, scales: [n_slots][rows][blocks],
 * contiguous.  x: state stride x_state, row stride x_row (elements), columns
 * contiguous.
 * store writes state i to slot slots[i] (device array; NULL: slot i); where a
 * slot is named twice the last state naming it is kept; slots outside
 * [0, n_slots) are skipped; at most 65535 states a call.  load reads slot slots[i] into x[i]; a slot
 * outside [0, n_slots) gives zeros. */
typedef struct SslaStateCache {
    void* codes;
    float* scales;
    const int* slots;
    long long x_state, x_row;
    int n, n_slots, rows, cols, block;
    int format;                /* SSLA_FMT_* */
    int dtype;                 /* SSLA_DT_* of x */
    int device;
} SslaStateCache;

int ssla_state_store(const SslaStateCache* c, const void* x, void* stream);
int ssla_state_load(const SslaStateCache* c, void* x, void* stream);

/* Group norm with an activation, channels last.  x, y: [n][positions]
 * [channels], channels contiguous, sample and position strides in elements;
 * per sample and group of channels / groups channels,
 *     y = act((x - mean) / sqrt(var + eps) * weight + bias),
 * mean and (biased) variance over the group's positions and channels.
 * weight and bias: [channels] 32-bit, each may be NULL.  y may be x itself.
 * At most 2^24 channels, 2^40 values a sample, 2^31 - 2^16 positions and as
 * many slabs (samples x groups).
 * `workspace`: ssla_group_norm_workspace bytes, 16-byte aligned, apart from
 * the tensors. */
typedef struct SslaGroupNorm {
    const void* x;
    void* y;
    const float *weight, *bias;
    long long x_sample, x_pos, y_sample, y_pos;
    int n, positions, channels, groups;
    int dtype;                 /* SSLA_DT_* of x and y */
    int activation;            /* SSLA_ACT_* */
    int device;
    float eps;
} SslaGroupNorm;

int ssla_group_norm(const SslaGroupNorm* a, void* workspace, size_t workspace_bytes, void* stream);
int ssla_group_norm_workspace(const SslaGroupNorm* a, size_t* bytes);

#ifdef __cplusplus
}
#endif
#endif /* SSLA_OPS_H */
