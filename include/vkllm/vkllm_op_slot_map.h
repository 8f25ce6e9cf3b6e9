/* VKLLM_OP_SLOT_MAP: where a step's new tokens go in a paged cache. No counterpart in the reference.
 *
 * The tensor is uint32 [1, 1, T, 2]: for each token its slot (page * page_rows + row of the page) and its position in its
 * sequence. srcs are the page table (VKLLM_OP_PAGE_TABLE, [1, 1, B, 1 + P], B <= 4096), the lengths that it was asked for and the
 * tokens that are new among them, both uint32 [1, 1, 1, B]. The new tokens lie row after row: token i of row b is at position
 * lengths[b] - counts[b] + i. A token whose position the table's row does not hold (the row could not grow) and the tokens
 * of [.., T, ..] behind the last one get (VKLLM_NO_SLOT, 0); those past T get none. A row with a count of 0 takes no place
 * among the tokens: where token b has to be row b's, as VKLLM_OP_PAGED_ATTN reads its queries, rows without a sequence are given a
 * count of 1 as well, and with their length of 0 get (VKLLM_NO_SLOT, 0). */
#ifndef VKLLM_OP_SLOT_MAP_H
#define VKLLM_OP_SLOT_MAP_H
#include <stdbool.h>
#include <stdint.h>
#include "vkllm_commands.h"
#include "vkllm_context.h"
#include "vkllm_tensor.h"
#ifdef __cplusplus
extern "C" {
#endif

#define VKLLM_NO_SLOT 0xFFFFFFFFu

struct vkllm_op_slot_map_params
{
    uint32_t page_rows; /* positions per page, at least 1 */
};
extern vkllm_err_t vkllm_op_slot_map_init(struct vkllm_context *context, struct vkllm_commands *commands,
                                    struct vkllm_tensor *tensor);
extern vkllm_err_t vkllm_op_slot_map_run(struct vkllm_context *context, struct vkllm_commands *commands,
                                   struct vkllm_tensor *tensor);
extern vkllm_err_t vkllm_op_slot_map_post_run(struct vkllm_context *context, struct vkllm_commands *commands,
                                        struct vkllm_tensor *tensor);

#ifdef __cplusplus
}
#endif
#endif
