// Device code that the kernels over a paged cache share.
#pragma once
#include "device_common.h"

namespace vk
{

constexpr uint32_t kNoPage = 0xFFFFFFFFu;

// (cos, sin) of position * turns full turns. The product is in 64 bits and only its fraction goes on: at position 10^5
// a 32-bit angle would be off by 2^-8.
__device__ __forceinline__ float2 turn_at(uint32_t position, double turns)
{
    const double full = (double)position * turns;
    float2 r;
    sincospif(2.0f * (float)(full - rint(full)), &r.y, &r.x);
    return r;
}

// Sum of `v` over the threads before this one, and the workgroup's in `total`; `part` holds a word per wave. Every thread
// calls it; it starts and ends with the workgroup together.
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t *part, uint64_t &total)
{
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave, waves = blockDim.x / kWave;
    uint64_t s = v;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1)
    {
        const uint64_t up = __shfl_up((unsigned long long)s, o, kWave);
        s += lane >= o ? up : 0;
    }
    __syncthreads();
    if (lane == kWave - 1)
        part[wave] = s;
    __syncthreads();
    uint64_t before = 0;
    total = 0;
    for (int i = 0; i < waves; ++i)
    {
        before += i < wave ? part[i] : 0;
        total += part[i];
    }
    return before + s - v;
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
