/* VKLLM_OP_PAGE_TABLE: the page table of a batch of sequences for the lengths that the caller wants next. No counterpart in
 * the reference.
 *
 * The tensor is the table, uint32 [1, 1, B, 1 + P], B <= 4096: row b holds a sequence's length, then the ids of the pages
 * of `page_rows` positions that it occupies, in order, then VKLLM_NO_PAGE. srcs[0] is the wanted lengths, uint32
 * [1, 1, 1, B]. srcs[1], optional, is the table so far, of the same shape and in memory of its own; without it the tensor
 * is brought up to date in place (its first contents, a zero in every row's first word, are uploaded by the caller).
 *
 * Row b keeps its first pages, as many as the shorter of both lengths needs. Pages that no row keeps are free (a page that
 * several rows hold is free when none of them keeps it), and are given to the rows that grow: in row order, lowest id first. A row
 * grows if its pages and those that the rows before it asked for are there; otherwise, and where the wanted length is
 * over P * page_rows, it stays as it was, which its first word tells. A length of 0 ends a sequence. Page ids at or past
 * `pages` in the table so far are carried along and occupy nothing.
 * Captured into a hipGraph, the call is replayed on the context's stream, and has been run once before (otherwise it is
 * refused).
 * The last page of a row that shares pages with another has to be full: tokens that follow go to pages of its own. */
#ifndef VKLLM_OP_PAGE_TABLE_H
#define VKLLM_OP_PAGE_TABLE_H
#include <stdbool.h>
#include <stdint.h>
#include "vkllm_commands.h"
#include "vkllm_context.h"
#include "vkllm_tensor.h"
#ifdef __cplusplus
extern "C" {
#endif

#define VKLLM_NO_PAGE 0xFFFFFFFFu

struct vkllm_op_page_table_params
{
    uint32_t page_rows; /* positions per page, at least 1 */
    uint32_t pages;     /* pages of the cache, 1..524288 */
};
extern vkllm_err_t vkllm_op_page_table_init(struct vkllm_context *context, struct vkllm_commands *commands,
                                    struct vkllm_tensor *tensor);
extern vkllm_err_t vkllm_op_page_table_run(struct vkllm_context *context, struct vkllm_commands *commands,
                                   struct vkllm_tensor *tensor);
extern vkllm_err_t vkllm_op_page_table_post_run(struct vkllm_context *context, struct vkllm_commands *commands,
                                        struct vkllm_tensor *tensor);

#ifdef __cplusplus
}
#endif
#endif
