// VKLLM_OP_ADJUST_LOGITS: penalties for used tokens, token biases and a grammar's mask. No counterpart in the reference.
//
// A workgroup takes tiles of one row's vocabulary, 32 bytes of logits a thread. It counts the tile's tokens in the row's
// history and notes their last bias in LDS (whole numbers and a maximum of entry numbers, so the order of the atomics
// changes nothing), and passes over the logits once, looking every token up. Bound by HBM for batches, by latency for a row.
// Tiles are as large as still fill the GPU, since each goes through the row's history; a workgroup with several keeps its
// share of the history in registers and has the next tile's logits on their way while it works on one. 256 rows of 131072
// fp16 logits, 4096 used tokens, 300 biases and a mask: a tile per workgroup 47 us, 34 now (4.2 TB/s); with nothing to look
// up 26. The same in fp32 56 us (4.9 TB/s).
#include <algorithm>

#include "device_common.h"
#include "paged_common.h"

namespace vk
{

constexpr uint32_t kBiasesInLds = 1024;
constexpr uint32_t kMaxThreads = 1024, kMinThreads = 256, kMinTile = 2048, kWorkgroups = 512;
// two vectors of logits a thread and tile: with four, fp32 held one workgroup of 1024 threads a CU
constexpr uint32_t tokens_per_thread(uint32_t size)
{
    return 32 / size;
}

struct AdjustArgs
{
    TView x, out;
    WordRows history, rules, mask;
    uint32_t tile;
};

// 16 bytes of logits: rows of odd widths start anywhere
template <typename T, uint32_t N> struct __attribute__((packed, aligned(sizeof(T)))) Logits
{
    T v __attribute__((ext_vector_type(N)));
};

// Dynamic LDS, if there are rules: a word per token of the tile, its count in the low half and the number of its last
// bias in the high one; WIDE, for histories or biases past 16 bits: a word each.
template <typename T, bool WIDE> __global__ __launch_bounds__(1024) void adjust_logits_kernel(AdjustArgs a)
{
    constexpr uint32_t N = 16 / sizeof(T), VECS = 2;
    typedef T TN __attribute__((ext_vector_type(N)));
    typedef Logits<T, N> Vec;
    extern __shared__ __align__(16) uint32_t lds[]; // also read as 16-byte vectors
    __shared__ float values[kBiasesInLds]; // the first biases' values
    const uint32_t t = threadIdx.x, threads = blockDim.x, b = blockIdx.y, V = a.x.n[3], tile = a.tile;
    uint32_t *count = lds, *last = WIDE ? lds + tile : lds;
    const uint32_t *rules = a.rules.p ? a.rules.p + (size_t)b * a.rules.stride : nullptr;
    const uint32_t *mask = a.mask.p ? a.mask.p + (size_t)b * a.mask.stride : nullptr;
    const T *row = (const T *)a.x.p + (size_t)b * a.x.s[2];
    T *out = (T *)a.out.p + (size_t)b * a.out.s[2];
    const uint32_t step = gridDim.x * tile;
    uint32_t v0 = blockIdx.x * tile;
    TN y[VECS];
    uint32_t bits[VECS];
    auto load = [&](uint32_t v0) {
#pragma unroll
        for (uint32_t j = 0; j < VECS; ++j)
        {
            const uint32_t v = v0 + (t + j * threads) * N;
            bits[j] = ~0u;
            if ((t + j * threads) * N < tile && v + N <= V)
            {
                y[j] = ((const Vec *)(row + v))->v;
                if (mask)
                    bits[j] = mask[v / 32];
            }
        }
    };
    load(v0);
    float rep = 1.f, inverse = 1.f, freq = 0.f, pres = 0.f;
    uint32_t n_bias = 0, used = 0;
    const uint32_t *h = nullptr;
    u32x4 mine = {~0u, ~0u, ~0u, ~0u}; // this thread's first part of the history, and its first bias: no token
    uint32_t my_bias = ~0u;
    if (rules)
    {
        // everything is asked for as far as its row goes, and cut to what the row has of it when that is known
        const uint32_t most_biases = (a.rules.n - 4) / 2;
        if (t < most_biases)
            my_bias = rules[4 + 2 * t];
        float value = t < most_biases ? __uint_as_float(rules[5 + 2 * t]) : 0.f;
        if (a.history.p)
        {
            h = a.history.p + (size_t)b * a.history.stride + 1;
            if (t < (a.history.n - 1) / 4)
                mine = ((const Word4 *)h)[t].v;
            used = min(scalar_word(h - 1), a.history.n - 1);
        }
        n_bias = min(scalar_word(rules + 3), most_biases);
        rep = __uint_as_float(scalar_word(rules));
        inverse = 1.f / rep;
        freq = __uint_as_float(scalar_word(rules + 1));
        pres = __uint_as_float(scalar_word(rules + 2));
        if (t >= used / 4)
            mine = (u32x4){~0u, ~0u, ~0u, ~0u};
        for (uint32_t i = t; i < min(n_bias, kBiasesInLds); i += threads)
        {
            values[i] = value;
            if (i + threads < min(n_bias, kBiasesInLds))
                value = __uint_as_float(rules[5 + 2 * (i + threads)]);
        }
        for (uint32_t i = t; i < (WIDE ? 2 : 1) * tile / 4; i += threads)
            ((u32x4 *)lds)[i] = (u32x4){0, 0, 0, 0};
    }
    auto bias_of = [&](uint32_t entry) {
        return entry <= kBiasesInLds ? values[entry - 1] : __uint_as_float(rules[5 + 2 * (entry - 1)]);
    };
    // the logit of token v0 + v
    auto adjusted = [&](float y, uint32_t v) {
        const uint32_t c = WIDE ? count[v] : count[v] & 0xFFFFu, e = WIDE ? last[v] : last[v] >> 16;
        // fp32: the quotient itself, which is also right where 1 / rep is no number of 32 bits (256 rows of 131072 56.3 us for
        // 55.7 with a product). fp16: a product, off by one roundoff of 32 bits more, a 2^-13th of the result's own; where 1 / rep
        // is no number of 32 bits, the quotient is none of 16.
        const float less = sizeof(T) == 4 ? y / rep : y * inverse;
        const float p = (y > 0.f ? less : y * rep) - (freq * (float)c + pres);
        y = c ? p : y;
        return e ? y + bias_of(e) : y;
    };
    for (; v0 < V; v0 += step)
    {
        const uint32_t n = min(tile, V - v0), nv = n / N;
        if (rules)
        {
            lds_barrier(); // the words are zero
            auto note = [&](uint32_t token) {
                if (token - v0 < n)
                    atomicAdd(&count[token - v0], 1u);
            };
#pragma unroll
            for (int k = 0; k < 4; ++k)
                note(mine[k]);
            for (uint32_t i = t + threads; i < used / 4; i += threads)
            {
                const u32x4 w = ((const Word4 *)h)[i].v;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    note(w[k]);
            }
            if (t < used % 4)
                note(h[used / 4 * 4 + t]);
            lds_barrier();
            for (uint32_t i = t; i < n_bias; i += threads)
            {
                const uint32_t v = (i == t ? my_bias : rules[4 + 2 * i]) - v0;
                if (v < n) // the counts stand, so the largest word is that of the last entry
                    atomicMax(&last[v], WIDE ? i + 1 : (i + 1) << 16 | (count[v] & 0xFFFFu));
            }
            lds_barrier();
        }
        TN z[VECS];
        uint32_t ok[VECS];
#pragma unroll
        for (uint32_t j = 0; j < VECS; ++j)
        {
            z[j] = y[j];
            ok[j] = bits[j] >> ((v0 + (t + j * threads) * N) % 32);
        }
        if (v0 + step < V)
            load(v0 + step);
#pragma unroll
        for (uint32_t j = 0; j < VECS; ++j)
        {
            const uint32_t v = (t + j * threads) * N;
            if (t + j * threads >= nv)
                continue;
            if (rules)
            {
                u32x4 w[N / 4], any = {0, 0, 0, 0};
#pragma unroll
                for (uint32_t k = 0; k < N / 4; ++k)
                {
                    w[k] = *(const u32x4 *)(count + v + 4 * k);
                    any |= w[k];
                    if (WIDE)
                        any |= *(const u32x4 *)(last + v + 4 * k);
                }
                if (any[0] | any[1] | any[2] | any[3])
                {
#pragma unroll
                    for (uint32_t k = 0; k < N; ++k)
                        z[j][k] = (T)adjusted((float)z[j][k], v + k);
#pragma unroll
                    for (uint32_t k = 0; k < N / 4; ++k)
                    {
                        *(u32x4 *)(count + v + 4 * k) = (u32x4){0, 0, 0, 0};
                        if (WIDE)
                            *(u32x4 *)(last + v + 4 * k) = (u32x4){0, 0, 0, 0};
                    }
                }
            }
#pragma unroll
            for (uint32_t k = 0; k < N; ++k)
                z[j][k] = (ok[j] >> k) & 1 ? z[j][k] : (T)-INFINITY;
            ((Vec *)(out + v0 + v))->v = z[j];
        }
        for (uint32_t v = nv * N + t; v < n; v += threads)
        {
            float y = (float)row[v0 + v];
            if (rules)
            {
                y = adjusted(y, v);
                count[v] = 0;
                last[v] = 0;
            }
            out[v0 + v] = !mask || (mask[(v0 + v) / 32] >> ((v0 + v) % 32)) & 1 ? (T)y : (T)-INFINITY;
        }
    }
}

template <typename T, bool WIDE> static hipError_t launch_as(hipStream_t st, const AdjustArgs &a)
{
    const uint32_t threads = std::max(a.tile / tokens_per_thread(sizeof(T)), kMinThreads), V = a.x.n[3], B = a.x.n[2];
    const size_t lds = a.rules.p ? (WIDE ? 8 : 4) * (size_t)a.tile : 0;
    static uint64_t done = 0;
    const hipError_t e = lds_attr_once((const void *)adjust_logits_kernel<T, WIDE>, 8 * kMaxThreads * tokens_per_thread(sizeof(T)), done);
    if (e != hipSuccess)
        return e;
    const uint32_t tiles = (V - 1) / a.tile + 1;
    const uint32_t groups = std::min(tiles, (kWorkgroups - 1) / B + 1);
    adjust_logits_kernel<T, WIDE><<<dim3(groups, B), threads, lds, st>>>(a);
    return hipGetLastError();
}

hipError_t launch_adjust_logits(hipStream_t st, const TView &x, const TView &out, const WordRows &history,
                                const WordRows &rules, const WordRows &mask)
{
    const uint32_t B = x.n[2], V = x.n[3];
    uint32_t tile = kMaxThreads * tokens_per_thread(x.dt == DT_F16 ? 2 : 4); // whole mask words per tile
    while (tile > kMinTile && (uint64_t)B * ((V - 1) / tile + 1) < kWorkgroups)
        tile /= 2;
    const AdjustArgs a{x, out, history, rules, mask, tile};
    const bool wide = std::max(history.n, rules.n) > 65535;
    if (x.dt == DT_F16)
        return wide ? launch_as<_Float16, true>(st, a) : launch_as<_Float16, false>(st, a);
    return wide ? launch_as<float, true>(st, a) : launch_as<float, false>(st, a);
}

} // namespace vk
