/*
 * lora_head.h — C ABI of the operators on the LoRA head that answer questions
 * about its distribution, or train it on another's:
 *
 *   score     log probability of a given token, entropy, top alternatives
 *   distill   KL divergence from a teacher's top logits, with its gradients
 *
 * Both take the head as the training step (include/lora_ce.h) sees it,
 *
 *   z[t] = h[t].W^T + scale.(h[t].A).B      h = f16(H), as lora_ce_step reads it
 *
 * and never write the T x V logits to memory.  As in the step, ranks above 4 have
 * scale.(h.A) and B as pairs of f16: a magnitude of 65,520 or more counts as an
 * infinity (calls of few positions take it as it is).  They keep no state: every
 * buffer is the caller's and lies on the current device (a pointer to other
 * memory is refused), the work is enqueued on `stream` (a cudaStream_t; NULL =
 * legacy default stream) and the call returns without waiting.  The workspace
 * needs no initialisation and may be used again as soon as the call's work is
 * done; calls that can overlap (streams, graphs captured from them) need one
 * each.  The calls can be captured into a CUDA graph.  Results do not depend on
 * what else runs, and a call repeated gives the same bits.
 *
 * Conventions as lora_ce.h: 0 or a negative LORA_CE_E* code, nothing aborts;
 * lora_head_last_error() describes the last failure on the calling thread.
 * An error found on the host enqueues nothing, but for a launch that fails
 * ("kernel launch failed"): those ahead of it have been enqueued, so wait for the
 * stream before freeing the call's buffers.  A device-side error (a bounded wait that
 * expired) turns every output into NaN, and ids into -1.
 */
#ifndef LORA_HEAD_H
#define LORA_HEAD_H

#include <stddef.h>
#include <stdint.h>

#include "lora_ce.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Device pointers: W [vocab][dim] f16 bits (16-byte aligned), A [dim][rank] and
 * B [rank][vocab] f32 (reference layouts).  rank 0 is the base model: A and B
 * are not read and may be NULL. */
typedef struct lora_head {
    const uint16_t* W;
    const float* A;
    const float* B;
    int32_t dim;   /* a multiple of 64, 64..640 */
    int32_t vocab; /* 1..2^19 */
    int32_t rank;  /* 0..64 (lora_head_distill with gradients: 1..64) */
    float scale;   /* alpha / r */
} lora_head;

#define LORA_HEAD_MAX_TOP 128        /* largest top_k, largest teacher list */
#define LORA_HEAD_MAX_TOKENS 1048576 /* largest T */

/* Bytes of device workspace (256-byte aligned) that a call of these sizes
 * needs; 0 for sizes that the call would refuse. */
size_t lora_head_score_workspace(const lora_head* head, int32_t T, int32_t top_k);
size_t lora_head_distill_workspace(const lora_head* head, int32_t T, int32_t K, int32_t grads);

/* Per position t of H [T][dim] (h_dtype LORA_CE_BF16, _F16 or _F32; 16-byte
 * aligned):
 *   logprob[t]          z[tokens[t]] - log sum e^z; NaN for a token outside
 *                       [0, vocab).  tokens and logprob may both be NULL.
 *   entropy[t]          -sum p log p, in nats; may be NULL
 *   top_ids[t][k], top_logprobs[t][k]   the top_k (0..128, <= vocab) largest
 *                       logits in descending order, equal ones by ascending id
 *                       (ordered by logits computed with 64-bit sums); not
 *                       read with top_k 0.  Where more than 24 further tokens
 *                       come within 2^-18 G of the last one, those of them
 *                       with the lowest ids are ordered.
 * A position whose logits hold a NaN or an infinity gets NaN, and ids -1.
 *
 * Accuracy.  A logit's f32 sum is off by up to n 2^-23 G[t], n <= dim / 16 + 12,
 *   G[t] = |h| max |W[v]| + |scale h.A| max |B[:, v]| + |scale| |h| max |A[:, j]| max |B[:, v]|
 * (the norms of W and B in the bound above: of 1,024 rows spread over the vocabulary), as
 * G bounds its partial sums; log sum e^z, and with it logprob, entropy and the losses
 * below, by as much at worst.  That is where channels of h cancel; where the partial
 * sums grow evenly towards the logit it is about 2e-7 |z|. */
int lora_head_score(const lora_head* head, const void* H, int32_t h_dtype, int32_t T,
                    const int32_t* tokens, int32_t top_k, float* logprob, float* entropy,
                    int32_t* top_ids, float* top_logprobs, void* workspace,
                    size_t workspace_bytes, void* stream);

/* Distillation.  ids, teacher [T][K] (K 1..128): the teacher's top logits (or
 * log probabilities; a constant per row cancels) and their token ids.  An entry
 * with a negative id is absent and its logit not looked at; so is one of an id
 * below vocab with a logit of -inf; entries of one row with the same id add up.  With
 *   q = softmax(teacher[t] / temperature) over the row's entries,
 *   p = softmax(z[t] / temperature) over the vocabulary,
 *   loss[t] = weight[t] temperature^2 sum_k q_k (log q_k - log p[ids_k]).
 * weight [T] may be NULL (1).  A row of weight 0, or without entries, has loss
 * 0 and adds nothing to the gradients, whatever its hidden state holds.
 * gA [dim][rank], gB [rank][vocab]: gradients of sum_t loss[t] (overwritten);
 * both NULL for the loss alone.  With one entry per row and temperature 1 this
 * is the cross-entropy of lora_ce_step (without its 1e-12).  A counted row with
 * an id >= vocab, a logit of NaN or +inf, or a NaN in its hidden state gets loss
 * NaN and makes the gradients NaN.  temperature: 0.01..100. */
int lora_head_distill(const lora_head* head, const void* H, int32_t h_dtype, int32_t T, int32_t K,
                      const int32_t* ids, const float* teacher, float temperature,
                      const float* weight, float* loss, float* gA, float* gB, void* workspace,
                      size_t workspace_bytes, void* stream);

const char* lora_head_last_error(void);

#ifdef __cplusplus
}
#endif
#endif /* LORA_HEAD_H */
