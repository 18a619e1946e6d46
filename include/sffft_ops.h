/* sffft_ops.h - C ABI of the sequence-mixing operators beside the long convolution
 * (libsffft_ops.so): linear attention with a decay for each head, rotary positions, and the norms
 * before and after a block fused with its gate and residual scale. The reference has none of them
 * (its one operator is the convolution); no counterparts.
 *
 * Conventions (as sffft.h, whose error codes these calls return)
 *  - All pointers are device pointers. Activations are fp32 or bf16 (`io`), token-major
 *    [batch][token][head][channel]; parameters, states and their gradients are fp32.
 *  - Inputs take element strides (batch, token, head), so that views of a fused projection need no
 *    copy; channels are contiguous. Outputs are contiguous. Offsets are 64-bit.
 *  - `stream` is a hipStream_t (NULL = default stream). Calls are asynchronous on that stream,
 *    allocate nothing, keep nothing between calls, and may be captured, the first one too.
 *  - Outputs and workspace may overlap no input, unless a call says otherwise.
 *  - Sizes whose kernels would need 2^32 threads are refused (attention: B * H from 2^24 / 6 on in the
 *    backward pass at the least, 2^23 forward, 2^24 for single tokens; norms: 2^19 gates that rows share).
 *  - Sums, states and statistics are fp32; every sum has a fixed order (no atomics), so equal
 *    calls give equal bits.
 */
#ifndef SFFFT_OPS_H
#define SFFFT_OPS_H
#include "sffft.h"

#ifdef __cplusplus
extern "C" {
#endif

#define SFFFT_IO_F32 0
#define SFFFT_IO_BF16 1

/* Linear attention with a decay for each head. With g = exp(log_decay[h]), key/value head
 * h / (H / Hk), and n = lengths[b] tokens of sequence b (T if lengths is NULL):
 *   S_t = g S_{t-1} + k_t v_t^T (t < n),   o_t = scale S_t^T q_t (t < n; 0 from n on)
 * S_{-1} is the initial state (zero if NULL); the final state is S_{n-1} (the initial one if n = 0).
 * States are [B][H][Dk][Dv] fp32. Tokens from n on are never read, whatever they hold. log_decay
 * <= 0 is meant (-inf: nothing is remembered); a positive one grows until it overflows, NaN makes NaN. lengths
 * outside 0..T are taken as the nearest of these. An infinity or NaN at a token that counts reaches the
 * outputs that the definition lets it reach, no earlier tokens and no other channels; in later ones an
 * infinity may count as NaN. */
typedef struct sffft_linattn {
  int io;                 /* SFFFT_IO_F32 or SFFFT_IO_BF16: q, k, v, o and their gradients */
  int B, T, H, Hk;        /* H a multiple of Hk, at most 2^23 - 64 channels in all its heads */
  int Dk, Dv;             /* multiples of 8, at most 128 */
  float scale;
  long long q[3], k[3], v[3]; /* element strides (batch, token, head): multiples of 16 bytes, the token's
                               * at most 2^24 - 128 */
  long long go[3];        /* of o's gradient (backward only) */
} sffft_linattn;

/* Workspace of a forward (backward = 0) or backward call, 16-byte aligned; 0 where none is needed
 * (NULL is then allowed) and for arguments that the call refuses. */
size_t sffft_linattn_work_bytes(const sffft_linattn* p, int backward);

/* o [B][T][H][Dv], final_state may be NULL. final_state may be initial_state itself. */
int sffft_linattn_fwd(const sffft_linattn* p, const void* q, const void* k, const void* v, const float* log_decay,
                      const float* initial_state, const int* lengths, void* o, float* final_state, void* work,
                      size_t work_bytes, void* stream);

/* Gradients dq [B][T][H][Dk], dk [B][T][Hk][Dk], dv [B][T][Hk][Dv] (summed over the query heads that
 * share a key/value head; zero from n on) and, unless NULL, d_initial_state, from o's gradient `go`
 * and, unless NULL, the final state's d_final_state. The decays get no gradient. */
int sffft_linattn_bwd(const sffft_linattn* p, const void* q, const void* k, const void* v, const float* log_decay,
                      const float* initial_state, const int* lengths, const void* go, const float* d_final_state,
                      void* dq, void* dk, void* dv, float* d_initial_state, void* work, size_t work_bytes,
                      void* stream);

/* One token for each of B sequences: p->T must be 1. state [slots][H][Dk][Dv] is updated in place;
 * sequence b uses row slot[b] of it (row b if slot is NULL), which must be within 0..slots-1 and
 * different for each b; a sequence whose slot is outside that range has no state: its output is 0
 * and nothing is updated. */
int sffft_linattn_step(const sffft_linattn* p, const void* q, const void* k, const void* v, const float* log_decay,
                       float* state, int slots, const int* slot, void* o, void* stream);

/* Rotary positions of q [B][T][H][D] and k [B][T][Hk][D] (k NULL with Hk = 0: q alone). `table` is
 * [positions][R] fp32: row p holds cos, then sin, of the R/2 angles of position p
 * (sffft_rotary_table). Pair i of a head is its channels (i, i + R/2), or (2i, 2i + 1) if
 * interleaved:  a' = a cos - b sin,  b' = b cos + a sin; channels from R on are copied. With
 * inverse = 1 by the negative angle (the gradient). Token t of sequence b has position
 * pos[b][t] (pos_bits 32 or 64), t if pos is NULL; a position outside the table gives NaN in the
 * rotated channels and reads nothing. (H + Hk) * D / 2 is at most 65535. qo may be q and ko k, with
 * equal strides; else they overlap neither. No two elements of the outputs, nor one of an output in place
 * and one of the other input, are the same; q and k may be parts of one array. */
typedef struct sffft_rotary {
  int io;
  int B, T, H, Hk, D;
  int R;                  /* D and R even, R at most D */
  int interleaved, inverse;
  int positions;          /* rows of the table */
  int pos_bits;           /* 32 or 64 */
  long long q[3], k[3], qo[3], ko[3]; /* element strides (batch, token, head) of inputs and outputs */
} sffft_rotary;
int sffft_rotary_apply(const sffft_rotary* p, const void* q, const void* k, const float* table, const void* pos,
                       void* qo, void* ko, void* stream);

/* Fills host memory `table` [positions][R] for sffft_rotary_apply, evaluated in fp64 and rounded
 * once. Pair i turns by f_i = base^(-2i/R) per position, changed by `scaling` for contexts `factor`
 * times longer than the `trained` length:
 *   SFFFT_ROTARY_NONE       as it is
 *   SFFFT_ROTARY_LINEAR     f_i / factor
 *   SFFFT_ROTARY_STRETCHED  base raised to base * factor^(R / (R - 2)): the slowest pair is divided by
 *                           factor, the fastest stays (R = 2: as it is)
 *   SFFFT_ROTARY_PARTS      f_i / factor for pairs that turn less than once over the trained
 *                           length, f_i for those that turn more than 32 times, linear between
 * cos and sin are multiplied by `magnitude` (1 for a plain rotation). Host code: needs no GPU. */
#define SFFFT_ROTARY_NONE 0
#define SFFFT_ROTARY_LINEAR 1
#define SFFFT_ROTARY_STRETCHED 2
#define SFFFT_ROTARY_PARTS 3
int sffft_rotary_table(int positions, int R, double base, int scaling, double factor, int trained, double magnitude,
                       float* table);

/* The step between two blocks of a network: y, the output of a block, is normalised, gated,
 * scaled and added to the residual x, and the sum is normalised for the next block:
 *   norm(z) = z / sqrt(mean(z^2) + eps)      (over the C channels of a token)
 *   r = x + scale . act(gate) . norm(y) . w_post,    h = norm(r) . w_pre
 * x, y, r, h [rows][C]; gate has one row for every gate_rows rows (1: a gate for each token; T: one
 * for each sequence of T tokens; rows must be a multiple of it). Without w_post (NULL) y is not
 * normalised; without gate and scale these factors are 1. h is the norm of the unrounded r. With
 * y NULL only h = norm(x) . w_pre is computed (r, w_post, gate, scale NULL): the first norm. */
#define SFFFT_ACT_NONE 0
#define SFFFT_ACT_SIGMOID 1
#define SFFFT_ACT_SILU 2
typedef struct sffft_blocknorm {
  int io;
  long long rows;
  int C;                  /* 1..16384 */
  int act;
  long long gate_rows;
  float eps;              /* >= 0 */
  long long x, y, gate;   /* element strides of a row */
  long long gr, gh;       /* of the gradients of r and h (backward only) */
} sffft_blocknorm;
int sffft_blocknorm_fwd(const sffft_blocknorm* p, const void* x, const void* y, const void* gate, const float* w_pre,
                        const float* w_post, const float* scale, void* r, void* h, void* stream);

/* Gradients dx, dy [rows][C], dgate [rows / gate_rows][C], dw_pre, dw_post, dscale [C] from the
 * gradients gr of r (NULL: zero) and gh of h (NULL: zero, not both). Outputs of inputs that are
 * NULL are NULL. The sums over rows are fp32, in parts whose order depends on the sizes alone. */
size_t sffft_blocknorm_work_bytes(const sffft_blocknorm* p, int has_y, int has_gate);
int sffft_blocknorm_bwd(const sffft_blocknorm* p, const void* x, const void* y, const void* gate, const float* w_pre,
                        const float* w_post, const float* scale, const void* gr, const void* gh, void* dx, void* dy,
                        void* dgate, float* dw_pre, float* dw_post, float* dscale, void* work, size_t work_bytes,
                        void* stream);

/* Text of the last HIP error recorded by a call of this library on this thread ("" if none). */
const char* sffft_ops_last_error(void);

#ifdef __cplusplus
}
#endif
#endif /* SFFFT_OPS_H */
