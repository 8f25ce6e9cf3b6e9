/* VKLLM_OP_PAGED_ATTN: attention of one new token of each sequence of a batch over a paged cache. No counterpart in the
 * reference.
 *
 * The tensor and srcs[0], the queries, are [1, B, H, head_dim] of any strides; srcs[1] is the cache (VKLLM_OP_UPDATE_PAGES,
 * [pages, 2 * KV, page_rows, head_dim], packed, page_rows a multiple of 16, H a multiple of KV: query head h reads key
 * head h / (H / KV)), all fp16 or all fp32; srcs[2] is the page table (VKLLM_OP_PAGE_TABLE, uint32 [1, 1, B, 1 + P], B <= 4096).
 * P * page_rows is at most 2^31.
 * Row b is the last token of its sequence (one token a row: the tokens of a prompt do not attend through this operator), whose
 * keys and values the cache holds already: over positions j < length
 * out = sum_j softmax_j(scale * q . k_j) v_j, with q rotated to position length - 1 (unless rope_base is 0). Softmax and
 * sums are in 32 bits, and the result is rounded once. A row of length 0, and one whose every score is -inf, gives zeros;
 * lengths end at P * page_rows, and positions on pages that the cache does not have count as absent. Rows of the cache
 * past a sequence's end are never used, whatever they hold. Infinite and undefined numbers in those that are count as in the
 * formula in 32 bits: a key whose score is -inf has no weight, a score of +inf or NaN leaves its head undefined, and an infinite
 * value makes its dim infinite under any weight that is not 0 (undefined under 0, or with one of the other sign).
 * Partial results go through a workspace of the context, made by _init: captured into a hipGraph, the call is replayed on
 * the context's stream, and every tensor of it has been run once before (otherwise it is refused). */
#ifndef VKLLM_OP_PAGED_ATTN_H
#define VKLLM_OP_PAGED_ATTN_H
#include <stdbool.h>
#include <stdint.h>
#include "vkllm_commands.h"
#include "vkllm_context.h"
#include "vkllm_tensor.h"
#ifdef __cplusplus
extern "C" {
#endif

struct vkllm_op_paged_attn_params
{
    float scale;
    float rope_base; /* as in vkllm_op_update_pages_params */
    bool neox_style;
};
extern vkllm_err_t vkllm_op_paged_attn_init(struct vkllm_context *context, struct vkllm_commands *commands,
                                    struct vkllm_tensor *tensor);
extern vkllm_err_t vkllm_op_paged_attn_run(struct vkllm_context *context, struct vkllm_commands *commands,
                                   struct vkllm_tensor *tensor);
extern vkllm_err_t vkllm_op_paged_attn_post_run(struct vkllm_context *context, struct vkllm_commands *commands,
                                        struct vkllm_tensor *tensor);

#ifdef __cplusplus
}
#endif
#endif
