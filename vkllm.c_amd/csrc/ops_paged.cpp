// Host side of the operators of batched generation over a paged cache: argument validation and launches of
// VKLLM_OP_PAGE_TABLE, SLOT_MAP, UPDATE_PAGES, PAGED_ATTN and ADJUST_LOGITS. No counterpart in the reference.
#include <cmath>
#include <cstring>

#include "ops_common.h"
#include "vkllm/vkllm_op_adjust_logits.h"
#include "vkllm/vkllm_op_page_table.h"
#include "vkllm/vkllm_op_paged_attn.h"
#include "vkllm/vkllm_op_slot_map.h"
#include "vkllm/vkllm_op_update_pages.h"

// uint32 rows [1, 1, B, W] whose words are contiguous
static bool word_rows(const vkllm_tensor *t)
{
    return t->dtype == vkllm_dtype_uint32 && t->shapes[0] == 1 && t->shapes[1] == 1 && t->strides[3] == 4;
}

// uint32 [1, 1, 1, B]
static bool word_list(const vkllm_tensor *t, uint32_t n)
{
    return t->dtype == vkllm_dtype_uint32 && t->shapes[0] == 1 && t->shapes[1] == 1 && t->shapes[2] == 1 &&
           t->shapes[3] == n;
}

// a page table [1, 1, B, 1 + P]
static bool is_page_table(const vkllm_tensor *t)
{
    return word_rows(t) && t->shapes[2] <= vk::kPagedMaxRows && t->shapes[3] >= 2;
}

static bool packed(const vkllm_tensor *t)
{
    return t->strides[3] == dtype_bytes(t->dtype) && t->strides[2] == t->shapes[3] * t->strides[3] &&
           t->strides[1] == t->shapes[2] * t->strides[2] && t->strides[0] == t->shapes[1] * t->strides[1];
}

// a cache [pages, 2 KV, page_rows, head_dim]; pool memory starts on 256-byte boundaries
static bool is_paged_cache(const vkllm_tensor *t)
{
    return is_float(t->dtype) && packed(t) && t->shapes[1] % 2 == 0 && t->shapes[3] % 8 == 0 &&
           t->shapes[3] <= vk::kPagedMaxHd;
}

static bool same_memory(vkllm_tensor *a, vkllm_tensor *b)
{
    return tensor_base(a) == tensor_base(b);
}

static vk::PageTableView table_view(const vk::TView &v)
{
    return {(uint32_t *)v.p, v.n[2], v.n[3] - 1, v.s[2]};
}

static bool rope_base_ok(float base)
{
    return base == 0.f || (base > 0.f && std::isfinite(base));
}

static vk::PagedRope rope_of(float base, bool neox, uint32_t hd)
{
    vk::PagedRope r;
    r.style = base == 0.f ? 0 : neox ? 2 : 1;
    // a power per call and a product per pair: 128 of them are off by 1.5e-14 at most, a billionth of a turn at
    // position 10^5
    const double ratio = r.style ? pow((double)base, -2.0 / hd) : 0.0;
    double turns = 1.0 / 6.283185307179586476925;
    for (uint32_t w = 0; w < hd / 2; ++w, turns *= ratio)
        r.turns[w] = turns;
    return r;
}

// Memory that a first call makes cannot be made while the context's stream is captured into a hipGraph: the call is refused
// and the capture goes on
static vkllm_err_t may_allocate(vkllm_context *context, const char *what)
{
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    HIP_TRY(hipStreamIsCapturing(context->device->stream, &status));
    if (status == hipStreamCaptureStatusNone)
        return VKLLM_ERR_OK;
    log_error("%s has no memory yet: run it once before the stream is captured", what);
    return VKLLM_ERR_ARGS;
}

// the node's tensor and its sources
static vkllm_err_t node_memory(vkllm_context *context, vkllm_tensor *tensor)
{
    if (!tensor_base(tensor)->data.dev)
        _CHECK(may_allocate(context, tensor->name));
    for (vkllm_tensor *src : tensor->srcs)
        if (src && !tensor_base(src)->data.dev)
            _CHECK(may_allocate(context, src->name));
    return VKLLM_ERR_OK;
}

// The context's workspace and arrival counters, made at the first use and kept until the context is freed
static vkllm_err_t paged_memory(vkllm_context *context, float **work, size_t *work_elems)
{
    vkllm_gpu_device *dev = context->device;
    if (!dev->op_work || !dev->paged_arrivals)
        _CHECK(may_allocate(context, "the operators' workspace"));
    _CHECK(op_workspace(context, work, work_elems));
    if (!*work)
        return VKLLM_ERR_ALLOC;
    if (dev->paged_arrivals)
        return VKLLM_ERR_OK;
    uint32_t *p = nullptr;
    HIP_TRY(hipMalloc(&p, vk::kPagedArrivals * sizeof(uint32_t)));
    hipError_t e = hipMemsetAsync(p, 0, vk::kPagedArrivals * sizeof(uint32_t), dev->stream);
    if (e == hipSuccess)
        e = hipStreamSynchronize(dev->stream);
    if (e != hipSuccess)
    {
        (void)hipFree(p);
        return hip_fail(e, "clearing the arrival counters", __FILE__, __LINE__);
    }
    dev->paged_arrivals = p;
    return VKLLM_ERR_OK;
}

// =============================================================================================================
// PAGE_TABLE
extern "C" vkllm_err_t vkllm_op_page_table_init(struct vkllm_context *context, struct vkllm_commands *commands,
                                                struct vkllm_tensor *tensor)
{
    DeviceScope device_scope(context);
    _CHECK_ARGS(context && commands && tensor);
    _CHECK_ARGS(tensor->srcs[0]);
    _CHECK_ARGS(tensor->op == VKLLM_OP_PAGE_TABLE);
    _CHECK_ARGS(is_page_table(tensor) && packed(tensor));
    _CHECK_ARGS(word_list(tensor->srcs[0], tensor->shapes[2]));
    _CHECK_ARGS(!same_memory(tensor, tensor->srcs[0]));
    vkllm_tensor *old = tensor->srcs[1];
    if (old)
    {
        _CHECK_ARGS(is_page_table(old) && same_shape(old, tensor));
        _CHECK_ARGS(!same_memory(tensor, old)); // in place is asked for by leaving the source out
    }
    vkllm_op_page_table_params p;
    memcpy(&p, tensor->params, sizeof(p));
    _CHECK_ARGS(p.page_rows > 0 && p.pages > 0 && p.pages <= vk::kPagedMaxPages);
    _CHECK_ARGS((uint64_t)p.pages * p.page_rows < VKLLM_NO_SLOT);
    tensor->pipeline = pipeline_of(context, KID_PAGE_TABLE);
    return VKLLM_ERR_OK;
}

extern "C" vkllm_err_t vkllm_op_page_table_run(struct vkllm_context *context, struct vkllm_commands *commands,
                                               struct vkllm_tensor *tensor)
{
    DeviceScope device_scope(context);
    _CHECK(vkllm_op_page_table_init(context, commands, tensor));
    CHECK_VIEW(tensor->srcs[0]);
    if (tensor->srcs[1])
        CHECK_VIEW(tensor->srcs[1]);
    CHECK_VIEW(tensor);
    _CHECK(node_memory(context, tensor));
    vkllm_op_page_table_params p;
    memcpy(&p, tensor->params, sizeof(p));
    vk::TView want = tview(context, tensor->srcs[0]), out = tview(context, tensor), old{};
    NEED_DEV(want);
    NEED_DEV(out);
    if (tensor->srcs[1])
    {
        old = tview(context, tensor->srcs[1]);
        NEED_DEV(old);
    }
    float *work = nullptr;
    size_t work_elems = 0;
    _CHECK(paged_memory(context, &work, &work_elems));
    LAUNCH(context, KID_PAGE_TABLE,
           vk::launch_page_table(context->device->stream, table_view(out), (const uint32_t *)old.p, old.s[2],
                                 (const uint32_t *)want.p, want.s[3], p.page_rows, p.pages, work, work_elems,
                                 context->device->paged_arrivals, context->device->cu_count));
    commands_note_write(commands, tensor);
    return VKLLM_ERR_OK;
}

extern "C" vkllm_err_t vkllm_op_page_table_post_run(struct vkllm_context *, struct vkllm_commands *,
                                                    struct vkllm_tensor *)
{
    return VKLLM_ERR_OK;
}

// =============================================================================================================
// SLOT_MAP
extern "C" vkllm_err_t vkllm_op_slot_map_init(struct vkllm_context *context, struct vkllm_commands *commands,
                                              struct vkllm_tensor *tensor)
{
    DeviceScope device_scope(context);
    _CHECK_ARGS(context && commands && tensor);
    _CHECK_ARGS(tensor->srcs[0] && tensor->srcs[1] && tensor->srcs[2]);
    _CHECK_ARGS(tensor->op == VKLLM_OP_SLOT_MAP);
    _CHECK_ARGS(word_rows(tensor) && packed(tensor) && tensor->shapes[3] == 2);
    const vkllm_tensor *table = tensor->srcs[0];
    _CHECK_ARGS(is_page_table(table));
    _CHECK_ARGS(word_list(tensor->srcs[1], table->shapes[2]) && word_list(tensor->srcs[2], table->shapes[2]));
    for (int i = 0; i < 3; ++i)
        _CHECK_ARGS(!same_memory(tensor, tensor->srcs[i]));
    vkllm_op_slot_map_params p;
    memcpy(&p, tensor->params, sizeof(p));
    _CHECK_ARGS(p.page_rows > 0);
    tensor->pipeline = pipeline_of(context, KID_SLOT_MAP);
    return VKLLM_ERR_OK;
}

extern "C" vkllm_err_t vkllm_op_slot_map_run(struct vkllm_context *context, struct vkllm_commands *commands,
                                             struct vkllm_tensor *tensor)
{
    DeviceScope device_scope(context);
    _CHECK(vkllm_op_slot_map_init(context, commands, tensor));
    for (int i = 0; i < 3; ++i)
        CHECK_VIEW(tensor->srcs[i]);
    CHECK_VIEW(tensor);
    _CHECK(node_memory(context, tensor));
    vkllm_op_slot_map_params p;
    memcpy(&p, tensor->params, sizeof(p));
    vk::TView table = tview(context, tensor->srcs[0]), lengths = tview(context, tensor->srcs[1]),
              counts = tview(context, tensor->srcs[2]), out = tview(context, tensor);
    NEED_DEV(table);
    NEED_DEV(lengths);
    NEED_DEV(counts);
    NEED_DEV(out);
    LAUNCH(context, KID_SLOT_MAP,
           vk::launch_slot_map(context->device->stream, table_view(table), (const uint32_t *)lengths.p, lengths.s[3],
                               (const uint32_t *)counts.p, counts.s[3], (uint32_t *)out.p, out.n[2], p.page_rows));
    commands_note_write(commands, tensor);
    return VKLLM_ERR_OK;
}

extern "C" vkllm_err_t vkllm_op_slot_map_post_run(struct vkllm_context *, struct vkllm_commands *,
                                                  struct vkllm_tensor *)
{
    return VKLLM_ERR_OK;
}

// =============================================================================================================
// UPDATE_PAGES
extern "C" vkllm_err_t vkllm_op_update_pages_init(struct vkllm_context *context, struct vkllm_commands *commands,
                                                  struct vkllm_tensor *tensor)
{
    DeviceScope device_scope(context);
    _CHECK_ARGS(context && commands && tensor);
    _CHECK_ARGS(tensor->srcs[0] && tensor->srcs[1] && tensor->srcs[2]);
    _CHECK_ARGS(tensor->op == VKLLM_OP_UPDATE_PAGES);
    vkllm_tensor *k = tensor->srcs[0], *v = tensor->srcs[1], *map = tensor->srcs[2];
    if (!is_float(tensor->dtype) || k->dtype != tensor->dtype || v->dtype != tensor->dtype)
    {
        log_error("update_pages: unsupported dtypes %s, %s -> %s", vkllm_dtype_s(k->dtype), vkllm_dtype_s(v->dtype),
                  vkllm_dtype_s(tensor->dtype));
        return VKLLM_ERR_ARGS;
    }
    _CHECK_ARGS(is_paged_cache(tensor));
    _CHECK_ARGS(same_shape(k, v) && k->shapes[0] == 1 && k->shapes[2] * 2 == tensor->shapes[1] &&
                k->shapes[3] == tensor->shapes[3]);
    _CHECK_ARGS(word_rows(map) && map->shapes[2] == k->shapes[1] && map->shapes[3] == 2);
    _CHECK_ARGS(!same_memory(tensor, k) && !same_memory(tensor, v) && !same_memory(tensor, map));
    vkllm_op_update_pages_params p;
    memcpy(&p, tensor->params, sizeof(p));
    _CHECK_ARGS(rope_base_ok(p.rope_base));
    tensor->pipeline = pipeline_of(context, KID_UPDATE_PAGES);
    return VKLLM_ERR_OK;
}

extern "C" vkllm_err_t vkllm_op_update_pages_run(struct vkllm_context *context, struct vkllm_commands *commands,
                                                 struct vkllm_tensor *tensor)
{
    DeviceScope device_scope(context);
    _CHECK(vkllm_op_update_pages_init(context, commands, tensor));
    for (int i = 0; i < 3; ++i)
        CHECK_VIEW(tensor->srcs[i]);
    CHECK_VIEW(tensor);
    _CHECK(node_memory(context, tensor));
    vkllm_op_update_pages_params p;
    memcpy(&p, tensor->params, sizeof(p));
    vk::TView k = tview(context, tensor->srcs[0]), v = tview(context, tensor->srcs[1]),
              map = tview(context, tensor->srcs[2]), cache = tview(context, tensor);
    NEED_DEV(k);
    NEED_DEV(v);
    NEED_DEV(map);
    NEED_DEV(cache);
    LAUNCH(context, KID_UPDATE_PAGES,
           vk::launch_update_pages(context->device->stream, cache, k, v, (const uint32_t *)map.p, map.s[2],
                                   rope_of(p.rope_base, p.neox_style, cache.n[3])));
    commands_note_write(commands, tensor);
    return VKLLM_ERR_OK;
}

extern "C" vkllm_err_t vkllm_op_update_pages_post_run(struct vkllm_context *, struct vkllm_commands *,
                                                      struct vkllm_tensor *)
{
    return VKLLM_ERR_OK;
}

// =============================================================================================================
// PAGED_ATTN
extern "C" vkllm_err_t vkllm_op_paged_attn_init(struct vkllm_context *context, struct vkllm_commands *commands,
                                                struct vkllm_tensor *tensor)
{
    DeviceScope device_scope(context);
    _CHECK_ARGS(context && commands && tensor);
    _CHECK_ARGS(tensor->srcs[0] && tensor->srcs[1] && tensor->srcs[2]);
    _CHECK_ARGS(tensor->op == VKLLM_OP_PAGED_ATTN);
    vkllm_tensor *q = tensor->srcs[0], *cache = tensor->srcs[1], *table = tensor->srcs[2];
    if (!is_float(tensor->dtype) || q->dtype != tensor->dtype || cache->dtype != tensor->dtype)
    {
        log_error("paged_attn: unsupported dtypes %s, %s -> %s", vkllm_dtype_s(q->dtype), vkllm_dtype_s(cache->dtype),
                  vkllm_dtype_s(tensor->dtype));
        return VKLLM_ERR_ARGS;
    }
    _CHECK_ARGS(same_shape(q, tensor) && q->shapes[0] == 1);
    _CHECK_ARGS(is_paged_cache(cache) && cache->shapes[2] % 16 == 0 && cache->shapes[3] == q->shapes[3]);
    _CHECK_ARGS(q->shapes[2] % (cache->shapes[1] / 2) == 0);
    _CHECK_ARGS(is_page_table(table) && table->shapes[2] == q->shapes[1]);
    _CHECK_ARGS((uint64_t)(table->shapes[3] - 1) * cache->shapes[2] <= 1ull << 31);
    _CHECK_ARGS(!same_memory(tensor, q) && !same_memory(tensor, cache) && !same_memory(tensor, table));
    vkllm_op_paged_attn_params p;
    memcpy(&p, tensor->params, sizeof(p));
    _CHECK_ARGS(std::isfinite(p.scale) && rope_base_ok(p.rope_base));
    float *work = nullptr;
    size_t work_elems = 0;
    _CHECK(paged_memory(context, &work, &work_elems));
    tensor->pipeline = pipeline_of(context, KID_PAGED_ATTN);
    return VKLLM_ERR_OK;
}

extern "C" vkllm_err_t vkllm_op_paged_attn_run(struct vkllm_context *context, struct vkllm_commands *commands,
                                               struct vkllm_tensor *tensor)
{
    DeviceScope device_scope(context);
    _CHECK(vkllm_op_paged_attn_init(context, commands, tensor));
    for (int i = 0; i < 3; ++i)
        CHECK_VIEW(tensor->srcs[i]);
    CHECK_VIEW(tensor);
    _CHECK(node_memory(context, tensor));
    vkllm_op_paged_attn_params p;
    memcpy(&p, tensor->params, sizeof(p));
    vk::TView q = tview(context, tensor->srcs[0]), cache = tview(context, tensor->srcs[1]),
              table = tview(context, tensor->srcs[2]), out = tview(context, tensor);
    NEED_DEV(q);
    NEED_DEV(cache);
    NEED_DEV(table);
    NEED_DEV(out);
    float *work = nullptr;
    size_t work_elems = 0;
    _CHECK(paged_memory(context, &work, &work_elems));
    LAUNCH(context, KID_PAGED_ATTN,
           vk::launch_paged_attn(context->device->stream, q, cache, table_view(table), out, p.scale,
                                 rope_of(p.rope_base, p.neox_style, q.n[3]), work, work_elems,
                                 context->device->paged_arrivals, context->device->cu_count));
    commands_note_write(commands, tensor);
    return VKLLM_ERR_OK;
}

extern "C" vkllm_err_t vkllm_op_paged_attn_post_run(struct vkllm_context *, struct vkllm_commands *,
                                                    struct vkllm_tensor *)
{
    return VKLLM_ERR_OK;
}

// =============================================================================================================
// ADJUST_LOGITS
extern "C" vkllm_err_t vkllm_op_adjust_logits_init(struct vkllm_context *context, struct vkllm_commands *commands,
                                                   struct vkllm_tensor *tensor)
{
    DeviceScope device_scope(context);
    _CHECK_ARGS(context && commands && tensor);
    _CHECK_ARGS(tensor->srcs[0]);
    _CHECK_ARGS(tensor->op == VKLLM_OP_ADJUST_LOGITS);
    vkllm_tensor *x = tensor->srcs[0], *history = tensor->srcs[1], *rules = tensor->srcs[2], *mask = tensor->srcs[3];
    _CHECK_ARGS(same_shape(x, tensor) && x->shapes[0] == 1 && x->shapes[1] == 1);
    if (tensor->dtype != x->dtype || !is_float(x->dtype))
    {
        log_error("adjust_logits: unsupported dtypes %s -> %s", vkllm_dtype_s(x->dtype), vkllm_dtype_s(tensor->dtype));
        return VKLLM_ERR_ARGS;
    }
    _CHECK_ARGS(x->strides[3] == dtype_bytes(x->dtype) && tensor->strides[3] == dtype_bytes(x->dtype));
    for (vkllm_tensor *src : {x, history, rules, mask})
        _CHECK_ARGS(!src || !same_memory(tensor, src));
    const uint32_t B = x->shapes[2], V = x->shapes[3];
    _CHECK_ARGS(B <= 65535); // a workgroup row each
    if (history)
        _CHECK_ARGS(rules && word_rows(history) && history->shapes[2] == B);
    if (rules)
        _CHECK_ARGS(word_rows(rules) && rules->shapes[2] == B && rules->shapes[3] >= 4 && rules->shapes[3] % 2 == 0);
    if (mask)
        _CHECK_ARGS(word_rows(mask) && mask->shapes[2] == B && mask->shapes[3] >= (V - 1) / 32 + 1);
    tensor->pipeline = pipeline_of(context, KID_ADJUST_LOGITS);
    return VKLLM_ERR_OK;
}

extern "C" vkllm_err_t vkllm_op_adjust_logits_run(struct vkllm_context *context, struct vkllm_commands *commands,
                                                  struct vkllm_tensor *tensor)
{
    DeviceScope device_scope(context);
    _CHECK(vkllm_op_adjust_logits_init(context, commands, tensor));
    for (vkllm_tensor *src : tensor->srcs)
        if (src)
            CHECK_VIEW(src);
    CHECK_VIEW(tensor);
    _CHECK(node_memory(context, tensor)); // before any view is made: that gives a source memory
    vk::WordRows rows[3] = {};
    for (int i = 1; i < 4; ++i)
    {
        if (!tensor->srcs[i])
            continue;
        vk::TView w = tview(context, tensor->srcs[i]);
        NEED_DEV(w);
        rows[i - 1] = {(const uint32_t *)w.p, w.s[2], w.n[3]};
    }
    vk::TView x = tview(context, tensor->srcs[0]), out = tview(context, tensor);
    NEED_DEV(x);
    NEED_DEV(out);
    LAUNCH(context, KID_ADJUST_LOGITS,
           vk::launch_adjust_logits(context->device->stream, x, out, rows[0], rows[1], rows[2]));
    commands_note_write(commands, tensor);
    return VKLLM_ERR_OK;
}

extern "C" vkllm_err_t vkllm_op_adjust_logits_post_run(struct vkllm_context *, struct vkllm_commands *,
                                                       struct vkllm_tensor *)
{
    return VKLLM_ERR_OK;
}
