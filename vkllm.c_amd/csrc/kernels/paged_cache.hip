// The page table of a batch, the slot map of a step's new tokens, and the writes into a paged cache
// (VKLLM_OP_PAGE_TABLE, SLOT_MAP, UPDATE_PAGES). No counterpart in the reference.
#include "device_common.h"
#include "paged_common.h"

namespace vk
{

// ---------------------------------------------------------------------------------------------------------------
// VKLLM_OP_PAGE_TABLE. With had and want a row's lengths so far and next (want past the row's width: had), the row keeps
// keep = ceil(min(had, want) / R) pages and asks for need = ceil(want / R) - keep. A bit per page says whether a row keeps
// it; the k-th free page goes to the row whose demand, summed in row order, covers k. Rows whose sum passes
// the number of free pages keep what they had.
//
// Workgroup 0 does that: bits and prefix sums stand in its LDS, so the table is built in one launch without an
// exchange between workgroups. It writes the lengths and the columns [keep, keep + need). The others write
// the remaining columns, which hang on a row's own lengths only: the kept ids (unless in place) and NO_PAGE behind.
constexpr int kTableThreads = 1024;
constexpr uint32_t kListLen = 4096; // free pages handed out at a time

struct PageTableArgs
{
    PageTableView out;
    const uint32_t *old; // nullptr: out itself
    uint32_t old_stride;
    const uint32_t *want;
    uint32_t want_s, R, pages;
};

__device__ __forceinline__ uint32_t ceil_pages(uint32_t len, uint32_t R)
{
    return len / R + (len % R != 0);
}

struct RowPages
{
    uint32_t had, want, keep, need;
};
__device__ __forceinline__ RowPages row_pages(uint32_t had, uint32_t want, uint32_t R, uint32_t P)
{
    const uint64_t most = (uint64_t)P * R;
    had = had > most ? (uint32_t)most : had;
    want = want > most ? had : want;
    const uint32_t keep = ceil_pages(had < want ? had : want, R);
    return {had, want, keep, ceil_pages(want, R) - keep};
}

__global__ __launch_bounds__(kTableThreads) void page_table_kernel(PageTableArgs a)
{
    extern __shared__ uint32_t lds[];
    const uint32_t t = threadIdx.x, B = a.out.B, P = a.out.P, R = a.R;
    if (blockIdx.x > 0)
    {
        // the columns of rows b, b + gridDim.x - 1, ...: a thread per column
        for (uint32_t b = blockIdx.x - 1; b < B; b += gridDim.x - 1)
        {
            const uint32_t want = a.want[(size_t)b * a.want_s];
            uint32_t *to = a.out.p + (size_t)b * a.out.stride + 1;
            if (!a.old)
            {
                for (uint32_t c = (want > (uint64_t)P * R ? P : ceil_pages(want, R)) + t; c < P; c += kTableThreads)
                    to[c] = kNoPage;
                continue;
            }
            const uint32_t *from = a.old + (size_t)b * a.old_stride;
            const RowPages r = row_pages(from[0], want, R, P);
            for (uint32_t c = t; c < P; c += kTableThreads)
                if (c < r.keep || c >= r.keep + r.need)
                    to[c] = c < r.keep ? from[1 + c] : kNoPage;
        }
        return;
    }
    const uint32_t words = (a.pages + 31) / 32;
    uint32_t *used = lds, *start = used + words, *keeps = start + B + 1, *list = keeps + B;
    __shared__ uint64_t scan[kTableThreads / kWave];
    const uint32_t *old = a.old ? a.old : a.out.p;
    const uint32_t old_stride = a.old ? a.old_stride : a.out.stride;
    for (uint32_t w = t; w < words; w += kTableThreads) // bits past the last page count as used
        used[w] = w * 32 + 32 <= a.pages ? 0u : ~0u << (a.pages % 32);
    // demands, summed in row order: thread t has rows t * per .. t * per + per - 1
    const uint32_t per = (B + kTableThreads - 1) / kTableThreads;
    uint64_t mine = 0;
    for (uint32_t b = t * per; b < t * per + per && b < B; ++b)
    {
        const RowPages r = row_pages(old[(size_t)b * old_stride], a.want[(size_t)b * a.want_s], R, P);
        keeps[b] = r.keep;
        mine += r.need;
    }
    uint64_t total;
    uint64_t at = block_scan(mine, scan, total);
    for (uint32_t b = t * per; b < t * per + per && b < B; ++b)
    {
        const RowPages r = row_pages(old[(size_t)b * old_stride], a.want[(size_t)b * a.want_s], R, P);
        start[b] = (uint32_t)at; // sums past 32 bits are past the last page, too (below)
        at += r.need;
    }
    if (t == 0)
        start[B] = (uint32_t)total;
    __syncthreads();
    // mark the kept pages: a wave takes 8 rows at a time, so that 8 reads are in flight
    const uint32_t lane = t % kWave, wave = t / kWave, waves = kTableThreads / kWave;
    for (uint32_t b0 = wave * 8; b0 < B; b0 += waves * 8)
    {
        uint32_t most = 0;
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i)
            most = max(most, b0 + i < B ? keeps[b0 + i] : 0u);
        for (uint32_t c = lane; c < most; c += kWave)
        {
            uint32_t id[8];
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i)
            {
                const uint32_t b = min(b0 + i, B - 1);
                id[i] = b0 + i < B && c < keeps[b] ? old[(size_t)b * old_stride + 1 + c] : kNoPage;
            }
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i)
                if (id[i] < a.pages)
                    atomicOr(&used[id[i] / 32], 1u << (id[i] % 32));
        }
    }
    __syncthreads();
    // free pages before thread t's words
    const uint32_t wper = (words + kTableThreads - 1) / kTableThreads;
    uint64_t free_mine = 0;
    for (uint32_t w = t * wper; w < t * wper + wper && w < words; ++w)
        free_mine += __popc(~used[w]);
    uint64_t nfree;
    const uint64_t rank0 = block_scan(free_mine, scan, nfree);
    // the rows that fit: a demand of total pages ends at min(total, nfree) of the list
    const uint32_t last = (uint32_t)(total < nfree ? total : nfree);
    for (uint32_t base = 0; base < last; base += kListLen)
    {
        uint64_t rank = rank0;
        for (uint32_t w = t * wper; w < t * wper + wper && w < words && rank < (uint64_t)base + kListLen; ++w)
            for (uint32_t m = ~used[w]; m; m &= m - 1, ++rank)
                if (rank >= base && rank < (uint64_t)base + kListLen)
                    list[rank - base] = w * 32 + __ffs(m) - 1;
        __syncthreads();
        const uint32_t n = min(kListLen, last - base);
        for (uint32_t i = t; i < n; i += kTableThreads)
        {
            // the row with start[b] <= k < start[b + 1]: the last whose start is at most k (rows without demand before it
            // have the same start)
            const uint32_t k = base + i, b = last_at_most(start, B, k);
            const uint32_t need = start[b + 1] - start[b];
            if ((uint64_t)start[b] + need <= nfree)
                a.out.p[(size_t)b * a.out.stride + 1 + keeps[b] + (k - start[b])] = list[i];
        }
        __syncthreads();
    }
    // lengths, and NO_PAGE where a row that does not fit would have had its pages
    for (uint32_t b = t; b < B; b += kTableThreads)
    {
        const RowPages r = row_pages(old[(size_t)b * old_stride], a.want[(size_t)b * a.want_s], R, P);
        const bool fits = r.need == 0 || (uint64_t)start[b] + r.need <= nfree;
        uint32_t *row = a.out.p + (size_t)b * a.out.stride;
        if (!fits)
            for (uint32_t c = 0; c < r.need; ++c)
                row[1 + r.keep + c] = kNoPage;
        row[0] = fits ? r.want : r.had;
    }
}

hipError_t launch_page_table(hipStream_t st, const PageTableView &out, const uint32_t *old, uint32_t old_stride,
                             const uint32_t *want, uint32_t want_s, uint32_t page_rows, uint32_t pages, int cu_count)
{
    const size_t lds = ((pages + 31) / 32 + 2 * (size_t)out.B + 1 + kListLen) * 4;
    static uint64_t done = 0;
    const hipError_t e = lds_attr_once((const void *)page_table_kernel, 128 << 10, done);
    if (e != hipSuccess)
        return e;
    const uint32_t fill = min(out.B, (uint32_t)cu_count);
    page_table_kernel<<<1 + fill, kTableThreads, lds, st>>>(
        PageTableArgs{out, old, old_stride, want, want_s, page_rows, pages});
    return hipGetLastError();
}

// ---------------------------------------------------------------------------------------------------------------
// VKLLM_OP_SLOT_MAP: a thread per token finds its row in the prefix sums of the counts, which every workgroup forms for
// itself (B words), and looks its page up.
__global__ __launch_bounds__(256) void slot_map_kernel(PageTableView table, const uint32_t *lengths, uint32_t lengths_s,
                                                       const uint32_t *counts, uint32_t counts_s, uint2 *map,
                                                       uint32_t T, uint32_t R)
{
    extern __shared__ uint32_t start[]; // [B + 1], sums that end at T
    __shared__ uint64_t scan[4];
    const uint32_t t = threadIdx.x, B = table.B, per = (B + 255) / 256;
    uint64_t mine = 0, total;
    for (uint32_t b = t * per; b < t * per + per && b < B; ++b)
        mine += counts[(size_t)b * counts_s];
    uint64_t at = block_scan(mine, scan, total);
    for (uint32_t b = t * per; b < t * per + per && b < B; ++b)
    {
        start[b] = (uint32_t)min(at, (uint64_t)T);
        at += counts[(size_t)b * counts_s];
    }
    if (t == 0)
        start[B] = (uint32_t)min(total, (uint64_t)T);
    __syncthreads();
    const uint32_t i = blockIdx.x * 256 + t;
    if (i >= T)
        return;
    uint2 out = {kNoPage, 0};
    if (i < start[B])
    {
        const uint32_t b = last_at_most(start, B, i);
        const uint32_t *row = table.p + (size_t)b * table.stride;
        const uint64_t most = (uint64_t)table.P * R;
        const uint32_t len = row[0] > most ? (uint32_t)most : row[0];
        // a count over the length puts the position below 0, past every length in 32 bits or not held all the same
        const int64_t pos = (int64_t)lengths[(size_t)b * lengths_s] - counts[(size_t)b * counts_s] + (i - start[b]);
        if (pos >= 0 && pos < len)
        {
            const uint64_t slot = (uint64_t)row[1 + (uint32_t)pos / R] * R + (uint32_t)pos % R;
            if (slot < kNoPage)
                out = {(uint32_t)slot, (uint32_t)pos};
        }
    }
    map[i] = out;
}

hipError_t launch_slot_map(hipStream_t st, const PageTableView &table, const uint32_t *lengths, uint32_t lengths_s,
                           const uint32_t *counts, uint32_t counts_s, uint32_t *map, uint32_t T, uint32_t page_rows)
{
    slot_map_kernel<<<(T - 1) / 256 + 1, 256, ((size_t)table.B + 1) * 4, st>>>(table, lengths, lengths_s, counts,
                                                                               counts_s, (uint2 *)map, T, page_rows);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------------------------------------------
// VKLLM_OP_UPDATE_PAGES. A workgroup has one token (or a share of its heads): the rotations of its position go
// into LDS once, then a thread moves units of 8 elements of a head: elements 8u .. 8u + 7, or for pairs of halves
// 4u .. 4u + 3 and as many behind the half. Bound by HBM for prompts, by latency for a token.
struct UpdatePagesArgs
{
    TView cache, k, v;
    const uint32_t *map;
    uint32_t map_s;
    uint32_t units; // of a share: 2 KV heads x hd / 8 over gridDim.y shares
    bool vec;       // k and v rows are contiguous and start on 16-byte boundaries
    PagedRope rope;
};

template <typename T> __device__ __forceinline__ void load4(const T *p, size_t stride, bool vec, float x[4])
{
    typedef T T4 __attribute__((ext_vector_type(4)));
    if (vec)
    {
        const T4 v = *(const T4 *)p;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            x[i] = (float)v[i];
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        x[i] = (float)p[i * stride];
}
template <typename T> __device__ __forceinline__ void store4(T *p, const float x[4])
{
    typedef T T4 __attribute__((ext_vector_type(4)));
    T4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        v[i] = (T)x[i];
    *(T4 *)p = v;
}

template <typename T> __global__ __launch_bounds__(256) void update_pages_kernel(UpdatePagesArgs a)
{
    __shared__ float2 cs[kPagedMaxHd / 2];
    const uint32_t tok = blockIdx.x, t = threadIdx.x;
    const uint32_t slot = a.map[(size_t)tok * a.map_s], pos = a.map[(size_t)tok * a.map_s + 1];
    const uint32_t R = a.cache.n[2], hd = a.cache.n[3], KV = a.cache.n[1] / 2, page = slot / R;
    if (page >= a.cache.n[0])
        return;
    const int style = a.rope.style;
    if (style)
    {
        if (t < hd / 2)
            cs[t] = turn_at(pos, a.rope.turns[t]);
        __syncthreads();
    }
    const uint32_t per = hd / 8, all = 2 * KV * per;
    T *to = (T *)a.cache.p + (size_t)page * a.cache.s[0] + (size_t)(slot % R) * hd;
    for (uint32_t u = blockIdx.y * a.units + t; u < min(all, (blockIdx.y + 1) * a.units); u += 256)
    {
        const uint32_t h = u / per, c = u % per;
        const TView &src = h < KV ? a.k : a.v;
        const T *from = (const T *)src.p + (size_t)tok * src.s[1] + (size_t)(h < KV ? h : h - KV) * src.s[2];
        T *row = to + (size_t)h * a.cache.s[1];
        const bool halves = style == 2 && h < KV;
        const uint32_t d0 = halves ? 4 * c : 8 * c, d1 = halves ? hd / 2 + 4 * c : 8 * c + 4;
        float x[4], y[4];
        load4(from + (size_t)d0 * src.s[3], src.s[3], a.vec, x);
        load4(from + (size_t)d1 * src.s[3], src.s[3], a.vec, y);
        if (halves)
        {
#pragma unroll
            for (int i = 0; i < 4; ++i)
            {
                const float2 r = cs[4 * c + i];
                const float p = x[i], q = y[i];
                x[i] = r.x * p - r.y * q;
                y[i] = r.y * p + r.x * q;
            }
        }
        else if (style && h < KV)
        {
#pragma unroll
            for (int i = 0; i < 2; ++i)
            {
                const float2 r = cs[4 * c + i], s = cs[4 * c + 2 + i];
                float p = x[2 * i], q = x[2 * i + 1];
                x[2 * i] = r.x * p - r.y * q;
                x[2 * i + 1] = r.y * p + r.x * q;
                p = y[2 * i];
                q = y[2 * i + 1];
                y[2 * i] = s.x * p - s.y * q;
                y[2 * i + 1] = s.y * p + s.x * q;
            }
        }
        store4(row + d0, x);
        store4(row + d1, y);
    }
}

hipError_t launch_update_pages(hipStream_t st, const TView &cache, const TView &k, const TView &v, const uint32_t *map,
                               uint32_t map_s, const PagedRope &rope)
{
    auto vec = [](const TView &t) {
        return t.s[3] == 1 && t.s[2] % 8 == 0 && t.s[1] % 8 == 0 && (uintptr_t)t.p % 16 == 0;
    };
    const uint32_t T = k.n[1], all = cache.n[1] * (cache.n[3] / 8);
    const uint32_t shares = min((all - 1) / 256 + 1, T >= 1024 ? 1u : (1023 / T) + 1);
    const uint32_t units = (all - 1) / shares + 1;
    const UpdatePagesArgs a{cache, k, v, map, map_s, units, vec(k) && vec(v), rope};
    const dim3 grid(T, shares);
    if (cache.dt == DT_F16)
        update_pages_kernel<_Float16><<<grid, 256, 0, st>>>(a);
    else
        update_pages_kernel<float><<<grid, 256, 0, st>>>(a);
    return hipGetLastError();
}

} // namespace vk
