// Argument checks and launch macros that the files of VKLLM_OP_* operators share.
#pragma once
#include "runtime.h"

inline bool same_shape(const vkllm_tensor *a, const vkllm_tensor *b)
{
    return a->shapes[0] == b->shapes[0] && a->shapes[1] == b->shapes[1] && a->shapes[2] == b->shapes[2] &&
           a->shapes[3] == b->shapes[3];
}

inline bool is_float(vkllm_dtype_t d)
{
    return d == vkllm_dtype_float16 || d == vkllm_dtype_float32;
}

// Every view a kernel is given must stay inside its base allocation.
inline bool view_in_bounds(const vkllm_tensor *t)
{
    const vkllm_tensor *b = t;
    while (b->data.is_ref && b->srcs[0])
        b = b->srcs[0];
    uint64_t last = 0;
    for (int i = 0; i < 4; ++i)
        last += (uint64_t)(t->shapes[i] - 1) * t->strides[i];
    return last + dtype_bytes(t->dtype) <= b->bytes;
}

#define CHECK_VIEW(_t)                                                                                              \
    do                                                                                                              \
    {                                                                                                               \
        if (!view_in_bounds(_t))                                                                                    \
        {                                                                                                           \
            log_error("tensor %s: view exceeds its allocation", (_t)->name);                                        \
            return VKLLM_ERR_ARGS;                                                                                  \
        }                                                                                                           \
    } while (0)

#define LAUNCH(_ctx, _kid, _call)                                                                                   \
    do                                                                                                              \
    {                                                                                                               \
        hipError_t _e = timed((_ctx), pipeline_of((_ctx), (_kid)), [&]() { return (_call); });                     \
        if (_e != hipSuccess)                                                                                       \
            return hip_fail(_e, #_call, __FILE__, __LINE__);                                                        \
    } while (0)

#define NEED_DEV(_v)                                                                                                \
    do                                                                                                              \
    {                                                                                                               \
        if (!(_v).p)                                                                                                \
            return VKLLM_ERR_ALLOC;                                                                                 \
    } while (0)

// the context's operator workspace (see its definition)
vkllm_err_t op_workspace(vkllm_context *ctx, float **work, size_t *elems);
