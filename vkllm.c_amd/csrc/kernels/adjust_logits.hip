// VKLLM_OP_ADJUST_LOGITS: penalties for used tokens, token biases and a grammar's mask. No counterpart in the reference.
//
// A workgroup has one tile of one row's vocabulary. It counts the tile's tokens in the row's history and notes their last
// bias in LDS (whole numbers and a maximum of entry numbers, so the order of the atomics changes nothing), then
// passes over the logits once. Bound by HBM for batches; every tile of a row reads the row's history again, from L2.
#include "device_common.h"

namespace vk
{

struct AdjustArgs
{
    TView x, out;
    WordRows history, rules, mask;
    uint32_t tile;
    bool vec; // rows start on 16-byte boundaries
};

// dynamic LDS: counts [tile] (if there is a history), last bias entries + 1 [tile] (if there are rules)
template <typename T> __global__ __launch_bounds__(256) void adjust_logits_kernel(AdjustArgs a)
{
    extern __shared__ uint32_t lds[];
    const uint32_t t = threadIdx.x, b = blockIdx.y, V = a.x.n[3];
    const uint32_t v0 = blockIdx.x * a.tile, n = min(a.tile, V - v0);
    uint32_t *count = lds, *last = a.history.p ? lds + a.tile : lds;
    const uint32_t *rules = a.rules.p ? a.rules.p + (size_t)b * a.rules.stride : nullptr;
    float rep = 1.f, freq = 0.f, pres = 0.f;
    if (rules)
    {
        const uint32_t n_bias = min(rules[3], (a.rules.n - 4) / 2);
        rep = __uint_as_float(rules[0]);
        freq = __uint_as_float(rules[1]);
        pres = __uint_as_float(rules[2]);
        for (uint32_t i = t; i < n; i += 256)
        {
            last[i] = 0;
            if (a.history.p)
                count[i] = 0;
        }
        __syncthreads();
        if (a.history.p)
        {
            const uint32_t *h = a.history.p + (size_t)b * a.history.stride;
            const uint32_t used = min(h[0], a.history.n - 1);
#pragma unroll 4
            for (uint32_t i = t; i < used; i += 256)
            {
                const uint32_t v = h[1 + i] - v0;
                if (v < n)
                    atomicAdd(&count[v], 1u);
            }
        }
        for (uint32_t i = t; i < n_bias; i += 256)
        {
            const uint32_t v = rules[4 + 2 * i] - v0;
            if (v < n)
                atomicMax(&last[v], i + 1);
        }
        __syncthreads();
    }
    const uint32_t *mask = a.mask.p ? a.mask.p + (size_t)b * a.mask.stride : nullptr;
    const T *x = (const T *)a.x.p + (size_t)b * a.x.s[2] + v0;
    T *out = (T *)a.out.p + (size_t)b * a.out.s[2] + v0;
    auto adjust = [&](float y, uint32_t v, bool allowed) {
        if (rules)
        {
            const uint32_t c = a.history.p ? count[v] : 0;
            if (c)
                y = (y > 0.f ? y / rep : y * rep) - (freq * (float)c + pres);
            if (last[v])
                y += __uint_as_float(rules[5 + 2 * (last[v] - 1)]);
        }
        return (T)(allowed ? y : -INFINITY);
    };
    constexpr uint32_t N = 16 / sizeof(T);
    typedef T TN __attribute__((ext_vector_type(N)));
    const uint32_t nv = a.vec ? n / N : 0;
    for (uint32_t i = t; i < nv; i += 256)
    {
        TN y = *(const TN *)(x + i * N);
        const uint32_t bits = mask ? mask[(v0 + i * N) / 32] >> ((v0 + i * N) % 32) : ~0u;
#pragma unroll
        for (uint32_t k = 0; k < N; ++k)
            y[k] = adjust((float)y[k], i * N + k, (bits >> k) & 1);
        *(TN *)(out + i * N) = y;
    }
    for (uint32_t i = nv * N + t; i < n; i += 256)
        out[i] = adjust((float)x[i], i, !mask || (mask[(v0 + i) / 32] >> ((v0 + i) % 32)) & 1);
}

hipError_t launch_adjust_logits(hipStream_t st, const TView &x, const TView &out, const WordRows &history,
                                const WordRows &rules, const WordRows &mask)
{
    const uint32_t B = x.n[2], V = x.n[3], N = x.dt == DT_F16 ? 8 : 4;
    auto vec = [N](const TView &t) { return (t.n[2] == 1 || t.s[2] % N == 0) && (uintptr_t)t.p % 16 == 0; };
    // whole mask words per tile; small batches take small tiles, so that the GPU is filled
    uint32_t tile = 8192;
    while (tile > 1024 && (uint64_t)B * ((V - 1) / tile + 1) < 512)
        tile /= 2;
    const AdjustArgs a{x, out, history, rules, mask, tile, vec(x) && vec(out)};
    const size_t lds = rules.p ? (history.p ? 8 : 4) * (size_t)tile : 0;
    const dim3 grid((V - 1) / tile + 1, B);
    if (x.dt == DT_F16)
        adjust_logits_kernel<_Float16><<<grid, 256, lds, st>>>(a);
    else
        adjust_logits_kernel<float><<<grid, 256, lds, st>>>(a);
    return hipGetLastError();
}

} // namespace vk
