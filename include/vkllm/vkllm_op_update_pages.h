/* VKLLM_OP_UPDATE_PAGES: new tokens' keys and values into a paged cache, in place. No counterpart in the reference (its
 * VKLLM_OP_UPDATE_ROWS writes consecutive rows of one sequence).
 *
 * The tensor is the cache, packed, fp16 or fp32 [pages, 2 * KV, page_rows, head_dim]: each page holds KV heads of keys, then KV
 * heads of values; head_dim is a multiple of 8, at most 256. srcs are the keys and the values, [1, T, KV, head_dim] of the
 * cache's type and any strides, and the slot map (VKLLM_OP_SLOT_MAP, uint32 [1, 1, T, 2]). Token t's rows go to its slot; keys are
 * rotated to its position first (unless rope_base is 0) and rounded once. Tokens whose slot is not one of the cache's
 * (VKLLM_NO_SLOT) write nothing, and rows that no token names stay as they were. The slots of a step differ, as
 * those of one slot map over unshared pages do: of two tokens with one slot either one's values may remain. */
#ifndef VKLLM_OP_UPDATE_PAGES_H
#define VKLLM_OP_UPDATE_PAGES_H
#include <stdbool.h>
#include <stdint.h>
#include "vkllm_commands.h"
#include "vkllm_context.h"
#include "vkllm_tensor.h"
#ifdef __cplusplus
extern "C" {
#endif

struct vkllm_op_update_pages_params
{
    float rope_base; /* pair w turns by position * rope_base^(-2w / head_dim); 0: keys are stored as they are */
    bool neox_style; /* pairs (w, w + head_dim / 2) instead of (2w, 2w + 1), as in VKLLM_OP_ROPE */
};
extern vkllm_err_t vkllm_op_update_pages_init(struct vkllm_context *context, struct vkllm_commands *commands,
                                    struct vkllm_tensor *tensor);
extern vkllm_err_t vkllm_op_update_pages_run(struct vkllm_context *context, struct vkllm_commands *commands,
                                   struct vkllm_tensor *tensor);
extern vkllm_err_t vkllm_op_update_pages_post_run(struct vkllm_context *context, struct vkllm_commands *commands,
                                        struct vkllm_tensor *tensor);

#ifdef __cplusplus
}
#endif
#endif
