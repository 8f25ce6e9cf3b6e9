/* VKLLM_OP_ADJUST_LOGITS: penalties for tokens already used, token biases and a grammar's mask on a batch's logits. No
 * counterpart in the reference.
 *
 * The tensor and srcs[0] are logits [1, 1, B, V], both fp16 or both fp32. The other sources are optional (NULL), of uint32:
 * srcs[1] the tokens used, [1, 1, B, 1 + T]: a row's count, then its tokens (needs srcs[2]); srcs[2] the rules,
 * [1, 1, B, 4 + 2 N]: a struct vkllm_logit_rules and up to N struct vkllm_logit_bias; srcs[3] the mask, [1, 1, B, W],
 * W >= ceil(V / 32): token t is allowed if bit t % 32 of word t / 32 is set. With n the times that a row's history holds a
 * token:
 *     n > 0:                 y = (x > 0 ? x / repetition : x * repetition) - (frequency * n + presence)
 *     a bias for the token:  y += value (its last one, if it has several)
 *     not allowed:           y = -inf, whatever x is
 * in 32 bits, rounded once. Tokens at or past V are ignored; counts end at the row's width. No source lies
 * in the tensor's memory. */
#ifndef VKLLM_OP_ADJUST_LOGITS_H
#define VKLLM_OP_ADJUST_LOGITS_H
#include <stdbool.h>
#include <stdint.h>
#include "vkllm_commands.h"
#include "vkllm_context.h"
#include "vkllm_tensor.h"
#ifdef __cplusplus
extern "C" {
#endif

/* the first words of a row of rules; 1, 0, 0, 0 changes nothing */
struct vkllm_logit_rules
{
    float repetition;
    float frequency;
    float presence;
    uint32_t n_biases;
};
struct vkllm_logit_bias
{
    uint32_t token;
    float value;
};
extern vkllm_err_t vkllm_op_adjust_logits_init(struct vkllm_context *context, struct vkllm_commands *commands,
                                    struct vkllm_tensor *tensor);
extern vkllm_err_t vkllm_op_adjust_logits_run(struct vkllm_context *context, struct vkllm_commands *commands,
                                   struct vkllm_tensor *tensor);
extern vkllm_err_t vkllm_op_adjust_logits_post_run(struct vkllm_context *context, struct vkllm_commands *commands,
                                        struct vkllm_tensor *tensor);

#ifdef __cplusplus
}
#endif
#endif
