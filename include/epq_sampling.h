/* epq_sampling.h -- which drafted tokens a target model keeps (libepq.so).
 *
 * Not part of the reference's op interface (include/epq.h): the reference generates through
 * the Hugging Face model.  Conventions are those of epq.h: plain pointers, epq_dtype codes,
 * a cudaStream_t passed as void*, EPQ_OK or a negative status with epq_last_error().
 */
#ifndef EPQ_SAMPLING_H
#define EPQ_SAMPLING_H

#include <stdint.h>

#include "epq.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Probabilities [batch, steps, vocab] (element strides; a row's values are contiguous). */
typedef struct epq_probs {
    const void* data;
    int64_t stride_row;
    int64_t stride_step;
} epq_probs;

/* Verification of drafted tokens by rejection: target holds p [batch, drafts + 1, vocab],
 * draft q [batch, drafts, vocab] (draft NULL: every drafted token had probability 1), both of
 * dtype, tokens the drafts x [batch, drafts] and uniforms random numbers u of [0, 1)
 * [batch, drafts + 1].  A row's drafts end at its first negative token.  Draft i is accepted
 * while u_i q_i(x_i) < p_i(x_i); behind the n accepted ones a token is drawn with u_drafts:
 * the first v whose weights w_0 .. w_v sum to more than u_drafts times their whole sum, where
 *     w = max(p_n - q_n, 0) at a refused draft (p_n without x_n where draft is NULL, and p_n
 *         itself where nothing is left), else w = p_n.
 * Products are 64-bit, sums keep 45 bits or more of the weights' (whose sum lies in float32's
 * range).  Weights that are negative or NaN count as 0; where the sum reaches no token (u of 1,
 * say) the last with a weight is taken, and -1 where none has one.
 * out [batch, drafts + 1] receives the accepted drafts, the drawn token and -1 behind it;
 * accepted [batch] receives n.  A drafted token of vocab or more ends its row's drafts and is
 * reported by epq_device_error (bit 3); what lies behind the end of a row's drafts is not looked
 * at.  The probabilities need only the alignment of their
 * type. */
int epq_verify_drafts(const epq_probs* target, const epq_probs* draft, const int64_t* tokens, int64_t tokens_stride,
                      const float* uniforms, int64_t uniforms_stride, int64_t batch, int32_t drafts, int64_t vocab,
                      int32_t dtype, int64_t* out, int64_t* accepted, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* EPQ_SAMPLING_H */
