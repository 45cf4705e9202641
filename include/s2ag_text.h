/*
 * s2ag_text.h -- C ABI of the text-model operators of libs2ag_hip.so (gfx950): word-embedding lookup with a scale and its
 * gradient by sorted ids, softmax cross entropy of a linear layer over a large vocabulary without keeping the logits, and the
 * global norm of many gradients with clipping.
 *
 * Conventions (those of s2ag_hip.h): plain pointers and sizes; pointers are DEVICE memory unless marked "host"; every call is
 * asynchronous on `stream` (a hipStream_t), allocates nothing, never synchronises and records kernels only, so it can be
 * captured into a graph.  Returns 0, a positive hipError_t or a negative S2AG_E_* code; a refused call has launched nothing.
 * Tensors are fp32 or bf16 (`bf16` = 0 / 1); sums, softmax statistics and norms are held in 32 bits or more.  No result depends
 * on the order in which workgroups run: two calls on the same inputs give the same bits.
 */
#ifndef S2AG_TEXT_H
#define S2AG_TEXT_H

#include "s2ag_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- gradient norm and clipping ------------------------------------------------------------------------------------------
 * norm = (sum over all tensors of g^2)^(1/2), or max |g| with norm_inf; factor = min(1, max_norm / (norm + 1e-6)) in fp32;
 * dst = factor * src, rounded once to dst's type.  A norm that is NaN gives a factor of NaN, an infinite one a factor of 0. */
typedef struct {
    const void* src;
    void* dst; /* may be src (in place; nothing is written where the factor is 1); null: the norm alone */
    long long n;
    int src_bf16, dst_bf16;
} s2ag_clip_tensor;
/* fp64 words of `partials` that a call on these tensors needs */
long long s2ag_clip_partials(const s2ag_clip_tensor* t /*host*/, int tensors);
int s2ag_clip_grads(const s2ag_clip_tensor* t /*host*/, int tensors, float max_norm, int norm_inf, double* partials,
                    float* norm /*one word, written*/, void* stream);

/* ---- embedding -------------------------------------------------------------------------------------------------------------
 * out[i] = round(scale * table[ids[i]]), rows of `dim` elements, contiguous.  An id outside [0, n_entries) reads as zeros. */
int s2ag_emb_lookup(const void* ids, int ids_i32, const void* table, int bf16, long long n, int dim, long long n_entries,
                    float scale, void* out, void* stream);
/* dtable[v] = round(scale * sum of dy[i] over the i with ids[i] == v, in an order that the ids decide); rows without an id and
 * the row `padding_idx` (-1: none) are written as zeros.  accumulate: fp32 only, dtable[v] += ... and rows without an id are left as
 * they are.  `ldy`: row pitch of dy in elements.  ids outside [0, n_entries) send nothing.  n < 2^31 - 2^16, n_entries < 2^30. */
long long s2ag_emb_grad_workspace_bytes(long long n, int dim, long long n_entries);
int s2ag_emb_grad(const void* ids, int ids_i32, const void* dy, long long ldy, int bf16, long long n, int dim,
                  long long n_entries, long long padding_idx, float scale, void* dtable, int accumulate, void* workspace,
                  long long workspace_bytes, void* stream);

/* ---- linear cross entropy ----------------------------------------------------------------------------------------------------
 * z = x w^T (rows x vocab, never stored whole); loss_i = log(sum_v exp z_iv) - z_{i, target_i}, 0 for target_i == ignore_index.
 * A target outside [0, vocab) that is not ignore_index makes that row's loss NaN.
 * bf16: the gradient of z is rounded to bf16 before the products that make dx and dw.  Rows that are ignored get a gradient of zero
 * whatever grad_out is, and so does dw where all are.
 * The backward call takes the forward call's sizes, types, w, ldw and `state`; x and target have to be there and are not read again. */
#define S2AG_LCE_MEAN 0 /* over the rows that are not ignored; 0 if there are none */
#define S2AG_LCE_SUM 1
#define S2AG_LCE_NONE 2
typedef struct {
    const void *x, *w;       /* (rows, dim) pitch ldx; (vocab, dim) pitch ldw */
    const void* target;      /* rows */
    int target_i32, bf16;
    long long rows, vocab, ldx, ldw, ignore_index;
    int dim, reduction;
    float* loss;             /* forward: one word, or `rows` of them with S2AG_LCE_NONE */
    int keep;                /* forward: a backward call will follow (its operands stay in `state`) */
    void* state;             /* s2ag_lce_state_bytes: written by the forward call, read by the backward call */
    const float* grad_out;   /* backward: one word, or `rows` of them */
    void *dx, *dw;           /* backward: contiguous, either may be null */
    int dw_accumulate;       /* fp32 only: dw += */
    void* workspace;
    long long workspace_bytes;
} s2ag_lce_args;
long long s2ag_lce_state_bytes(const s2ag_lce_args* a /*host*/);
long long s2ag_lce_workspace_bytes(const s2ag_lce_args* a /*host*/, int backward);
int s2ag_lce_fwd(const s2ag_lce_args* a /*host*/, void* stream);
int s2ag_lce_bwd(const s2ag_lce_args* a /*host*/, void* stream);

#ifdef __cplusplus
}
#endif
#endif
