// Device code that the kernels over a paged cache share.
#pragma once
#include "device_common.h"

namespace vk
{

constexpr uint32_t kNoPage = 0xFFFFFFFFu;

// 4 words at any word's address
struct __attribute__((packed, aligned(4))) Word4
{
    u32x4 v;
};

// the workgroup meets; what it wrote to LDS is seen. Loads from memory stay in flight, which __syncthreads would wait for.
__device__ __forceinline__ void lds_barrier()
{
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// A word at an address that the whole wave shares and that nothing writes while the kernel runs, as a scalar load: it counts
// on a counter of its own, so that waiting for it waits for no vector load.
__device__ __forceinline__ uint32_t scalar_word(const uint32_t *p)
{
    return *(const __attribute__((address_space(4))) uint32_t *)(uintptr_t)p;
}

// (cos, sin) of position * turns full turns. The product is in 64 bits and only its fraction goes on: at position 10^5
// a 32-bit angle would be off by 2^-8. What the fraction's 32 bits leave out turns the result a little further, by less than
// 2 pi 2^-26, which is its own sine; without it fp32 rows are 1.4 times as far off as their arithmetic makes them, 1.07 with it.
__device__ __forceinline__ float2 turn_at(uint32_t position, double turns)
{
    const double full = (double)position * turns, part = full - rint(full);
    const float near = (float)part, rest = 6.283185307f * (float)(part - (double)near);
    float s, c;
    sincospif(2.0f * near, &s, &c);
    return {fmaf(-s, rest, c), fmaf(c, rest, s)};
}

template <int ctrl, int row_mask> __device__ __forceinline__ uint64_t dpp_add64(uint64_t v)
{
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (uint32_t)v, ctrl, row_mask, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (uint32_t)(v >> 32), ctrl, row_mask, 0xF, false);
    return v + ((uint64_t)hi << 32 | lo);
}

// sum of `v` over the wave's lanes up to this one
__device__ __forceinline__ uint64_t wave_scan(uint64_t v)
{
    v = dpp_add64<0x111, 0xF>(v); // row_shr:1, 2, 4, 8 within rows of 16
    v = dpp_add64<0x112, 0xF>(v);
    v = dpp_add64<0x114, 0xF>(v);
    v = dpp_add64<0x118, 0xF>(v);
    v = dpp_add64<0x142, 0xA>(v); // row_bcast:15 -> rows 1, 3
    v = dpp_add64<0x143, 0xC>(v); // row_bcast:31 -> rows 2, 3
    return v;
}

__device__ __forceinline__ uint64_t read_lane(uint64_t v, uint32_t lane)
{
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(v >> 32), lane) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((uint32_t)v, lane);
}

// Sum of `v` over the threads before this one, and the workgroup's in `total`; `part` holds a word per wave. Every thread
// calls it; it starts and ends with the workgroup together.
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t *part, uint64_t &total)
{
    const uint32_t lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint64_t s = wave_scan(v);
    __syncthreads();
    if (lane == kWave - 1)
        part[wave] = s;
    __syncthreads();
    // the waves' sums by the same scan: one after the other, 16 of them took 0.7 us
    const uint64_t upto = wave_scan(lane < blockDim.x / kWave ? part[lane] : 0);
    total = read_lane(upto, kWave - 1);
    return (wave ? read_lane(upto, wave - 1) : 0) + s - v;
}

// the last b < n with start[b] <= k, for start[0] = 0 and sums that do not fall
__device__ __forceinline__ uint32_t last_at_most(const uint32_t *start, uint32_t n, uint32_t k)
{
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1)
    {
        const uint32_t mid = (lo + hi) / 2;
        if (start[mid] <= k)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

} // namespace vk
