// The page table of a batch, the slot map of a step's new tokens, and the writes into a paged cache
// (VKLLM_OP_PAGE_TABLE, SLOT_MAP, UPDATE_PAGES). No counterpart in the reference.
#include <algorithm>

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
// The first `markers` workgroups mark the kept pages, each those of its share of the rows, in bits in LDS. The last of them to
// arrive (none waits) takes the others' bits from the workspace, and has the prefix sums, the free pages' ranks and the lengths
// in its own LDS: it writes the lengths and the columns [keep, keep + need). The other workgroups write the remaining columns,
// which hang on a row's own lengths only: the kept ids (unless in place) and NO_PAGE behind. One launch. Bound by latency
// and by a CU's rate of LDS atomics: 256 rows of up to 512 pages of 65536 take 10.2 us, 16.8 with one marking workgroup; 1000
// rows of up to 700 of 400000 26.5 us, in place 27; a step that hands out 14000 pages 56.
constexpr uint32_t kMaxTableThreads = 1024, kMinTableThreads = 256;

struct PageTableArgs
{
    PageTableView out;
    const uint32_t *old; // nullptr: out itself
    uint32_t old_stride;
    const uint32_t *want;
    uint32_t want_s, R, pages;
    uint32_t markers;
    uint32_t *bits;     // [markers][bits of all pages], even numbers of words
    uint32_t *arrivals; // zero between launches
};
constexpr uint32_t kMarkColumns = 256; // columns of a row that a wave marks at once
// 16 pieces: 16 rows of 700 columns 9.7 us for 8.8. us with up to 4 / 8 / 16 / 32 markers: 256 rows of 512 11.0 / 9.8 / 10.2 / 10.4,
// 256 of 2048 23.2 / 18.4 / 17.7 / 22.0, 1000 of 700 32.7 / 26.6 / 27.0 / 28.8, 30 of 8192 14.5 / 12.0 / 11.7 / 13.7; only many
// narrow rows want more: 4000 of 64 38.1 / 26.3 / 21.5 / 21.9.
constexpr uint32_t kMarkPieces = 32, kMaxMarkers = 8;

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

__global__ __launch_bounds__(kMaxTableThreads) void page_table_kernel(PageTableArgs a)
{
    extern __shared__ __align__(16) uint32_t lds[]; // also read as 64-bit words
    const uint32_t t = threadIdx.x, threads = blockDim.x, B = a.out.B, P = a.out.P, R = a.R;
    if (blockIdx.x >= a.markers)
    {
        // the columns of rows b, b + (such workgroups), ...: a thread per column
        for (uint32_t b = blockIdx.x - a.markers; b < B; b += gridDim.x - a.markers)
        {
            const uint32_t want = a.want[(size_t)b * a.want_s];
            uint32_t *to = a.out.p + (size_t)b * a.out.stride + 1;
            if (!a.old)
            {
                // A wanted length over the row's width leaves the row as it is. Its own length may just be rewritten, cut to
                // the width: either way it is as many pages.
                const uint32_t kept = want > (uint64_t)P * R ? row_pages(to[-1], want, R, P).keep : ceil_pages(want, R);
                for (uint32_t c = kept + t; c < P; c += threads)
                    to[c] = kNoPage;
                continue;
            }
            const uint32_t *from = a.old + (size_t)b * a.old_stride;
            const RowPages r = row_pages(from[0], want, R, P);
            for (uint32_t c = t; c < P; c += threads)
                if (c < r.keep || c >= r.keep + r.need)
                    to[c] = c < r.keep ? from[1 + c] : kNoPage;
        }
        return;
    }
    const uint32_t words = (a.pages + 63) / 64 * 2;
    uint32_t *used = lds, *start = used + words, *keeps = start + B + 1, *hads = keeps + B, *wants = hads + B,
             *ranks = wants + B;
    __shared__ uint64_t scan[kMaxTableThreads / kWave];
    __shared__ uint32_t arrived;
    const uint32_t *old = a.old ? a.old : a.out.p;
    const uint32_t old_stride = a.old ? a.old_stride : a.out.stride;
    for (uint32_t w = t; w < words; w += threads) // bits past the last page count as used
        used[w] = w * 32 + 32 <= a.pages ? 0u : w * 32 >= a.pages ? ~0u : ~0u << (a.pages % 32);
    // demands, summed in row order: thread t has rows t * per .. t * per + per - 1
    const uint32_t per = (B + threads - 1) / threads;
    uint64_t mine = 0;
    for (uint32_t b = t * per; b < t * per + per && b < B; ++b)
    {
        const RowPages r = row_pages(old[(size_t)b * old_stride], a.want[(size_t)b * a.want_s], R, P);
        keeps[b] = r.keep;
        hads[b] = r.had;
        wants[b] = r.want;
        start[b] = r.need;
        mine += r.need;
    }
    uint64_t total;
    uint64_t at = block_scan(mine, scan, total);
    for (uint32_t b = t * per; b < t * per + per && b < B; ++b)
    {
        const uint32_t need = start[b];
        start[b] = (uint32_t)at; // a table has fewer than 2^30 columns in all
        at += need;
    }
    if (t == 0)
        start[B] = (uint32_t)total;
    __syncthreads();
    // Marks: a wave takes 256 columns of 4 rows at a time, neighbouring lanes neighbouring columns, 16 ids a lane on their way
    const uint32_t lane = t % kWave, wave = __builtin_amdgcn_readfirstlane(t / kWave), waves = threads / kWave;
    const uint32_t chunks = (P - 1) / kMarkColumns + 1, rows = (B - 1) / a.markers + 1, first = blockIdx.x * rows;
    const uint32_t items = first < B ? min(rows, B - first) * chunks : 0;
    for (uint32_t i0 = wave * 4; i0 < items; i0 += waves * 4)
    {
        uint32_t id[4][4], keep[4], c[4];
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
        {
            // columns past the kept ones repeat the last, so that no load is conditional
            const uint32_t item = min(i0 + i, items - 1), b = first + item / chunks;
            const uint32_t *row = old + (size_t)b * old_stride;
            c[i] = item % chunks * kMarkColumns;
            keep[i] = __builtin_amdgcn_readfirstlane(keeps[b]);
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k)
                id[i][k] = row[min(1 + c[i] + k * kWave + lane, keep[i])];
        }
        // all are asked for before the first is looked at (the compiler would move each load to its use)
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
            asm volatile("" : "+v"(id[i][0]), "+v"(id[i][1]), "+v"(id[i][2]), "+v"(id[i][3]));
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k)
                if (c[i] + k * kWave + lane < keep[i] && id[i][k] < a.pages)
                    atomicOr(&used[id[i][k] / 32], 1u << (id[i][k] % 32));
    }
    __syncthreads();
    if (a.markers > 1)
    {
        uint64_t *bits = (uint64_t *)a.bits;
        const uint64_t *mine = (const uint64_t *)used;
        for (uint32_t w = t; w < words / 2; w += threads)
            __hip_atomic_store(bits + (size_t)blockIdx.x * (words / 2) + w, mine[w], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __builtin_amdgcn_s_waitcnt(0); // this thread's bits are there
        __syncthreads();
        if (t == 0)
        {
            arrived = __hip_atomic_fetch_add(a.arrivals, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (arrived == a.markers - 1)
                __hip_atomic_store(a.arrivals, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); // for the next launch
        }
        __syncthreads();
        if (arrived != a.markers - 1)
            return;
        for (uint32_t w = t; w < words / 2; w += threads)
        {
            uint64_t any = mine[w], theirs[kMaxMarkers];
#pragma unroll
            for (uint32_t g = 0; g < kMaxMarkers; ++g) // all on their way at once
                theirs[g] = g < a.markers ? __hip_atomic_load(bits + (size_t)g * (words / 2) + w, __ATOMIC_RELAXED,
                                                              __HIP_MEMORY_SCOPE_AGENT)
                                          : 0;
#pragma unroll
            for (uint32_t g = 0; g < kMaxMarkers; ++g)
                any |= theirs[g];
            ((uint64_t *)used)[w] = any;
        }
        __syncthreads();
    }
    // free pages before thread t's words
    const uint32_t wper = (words + threads - 1) / threads;
    uint64_t free_mine = 0;
    for (uint32_t w = t * wper; w < t * wper + wper && w < words; ++w)
        free_mine += __popc(~used[w]);
    uint64_t nfree;
    const uint64_t rank0 = block_scan(free_mine, scan, nfree);
    ranks[t] = (uint32_t)rank0;
    __syncthreads();
    // The k-th free page to the row with start[b] <= k < start[b + 1], a thread per k: the page is found from the ranks of the
    // threads' words, counts of bits and halves of a word
    const uint32_t last = (uint32_t)(total < nfree ? total : nfree);
    for (uint32_t k = t; k < last; k += threads)
    {
        const uint32_t owner = last_at_most(ranks, threads, k);
        uint32_t w = owner * wper, nth = k - ranks[owner], at = 0;
        for (; nth >= (uint32_t)__popc(~used[w]); ++w)
            nth -= __popc(~used[w]);
        uint32_t bits = ~used[w];
#pragma unroll
        for (uint32_t half = 16; half > 0; half /= 2)
        {
            const uint32_t below = __popc(bits & ((1u << half) - 1));
            const bool up = nth >= below;
            nth -= up ? below : 0;
            at += up ? half : 0;
            bits = up ? bits >> half : bits;
        }
        // the last row whose start is at most k (rows without demand before it have the same start)
        const uint32_t b = last_at_most(start, B, k), need = start[b + 1] - start[b];
        if ((uint64_t)start[b] + need <= nfree)
            a.out.p[(size_t)b * a.out.stride + 1 + keeps[b] + (k - start[b])] = w * 32 + at;
    }
    // lengths, and NO_PAGE where a row that does not fit would have had its pages
    for (uint32_t b = t; b < B; b += threads)
    {
        const uint32_t need = start[b + 1] - start[b];
        const bool fits = need == 0 || (uint64_t)start[b] + need <= nfree;
        uint32_t *row = a.out.p + (size_t)b * a.out.stride;
        if (!fits)
            for (uint32_t c = 0; c < need; ++c)
                row[1 + keeps[b] + c] = kNoPage;
        row[0] = fits ? wants[b] : hads[b];
    }
}

hipError_t launch_page_table(hipStream_t st, const PageTableView &out, const uint32_t *old, uint32_t old_stride,
                             const uint32_t *want, uint32_t want_s, uint32_t page_rows, uint32_t pages, float *work,
                             size_t work_elems, uint32_t *arrivals, int cu_count)
{
    const uint32_t words = (pages + 63) / 64 * 2;
    const size_t lds = (words + 4 * (size_t)out.B + 1 + kMaxTableThreads) * 4; // 132 KB at most
    static uint64_t done = 0;
    const hipError_t e = lds_attr_once((const void *)page_table_kernel, 134 << 10, done);
    if (e != hipSuccess)
        return e;
    // at least kMarkPieces pieces of 256 columns to a marking workgroup, and at most 1 MB of bits for the last to read
    const uint64_t pieces = (uint64_t)out.B * ((out.P - 1) / kMarkColumns + 1);
    const uint32_t markers = (uint32_t)std::max<uint64_t>(
        1, std::min<uint64_t>({out.B, pieces / kMarkPieces, kMaxMarkers, (256 << 10) / words, work_elems / words}));
    const uint32_t fill = std::min(out.B, (uint32_t)cu_count);
    // a small table takes fewer waves to bring together: a row of up to 256 pages of 256 takes 4.7 us with 1024 threads,
    // 3.4 with 256; a table of 256 rows has work for all 16 waves
    const uint32_t threads = pieces <= kMinTableThreads / kWave * 4 && pages <= 16384 ? kMinTableThreads : kMaxTableThreads;
    page_table_kernel<<<markers + fill, threads, lds, st>>>(PageTableArgs{
        out, old, old_stride, want, want_s, page_rows, pages, markers, (uint32_t *)work, arrivals});
    return hipGetLastError();
}

// ---------------------------------------------------------------------------------------------------------------
// VKLLM_OP_SLOT_MAP: a thread per token finds its row in the prefix sums of the counts, which every workgroup forms for
// itself (B words), and looks its page up.
__global__ __launch_bounds__(256) void slot_map_kernel(PageTableView table, const uint32_t *lengths, uint32_t lengths_s,
                                                       const uint32_t *counts, uint32_t counts_s, uint2 *map,
                                                       uint32_t T, uint32_t R)
{
    extern __shared__ uint32_t start[]; // [B + 1], sums that end at T; then the rows' lengths, counts and held positions
    __shared__ uint64_t scan[4];
    const uint32_t t = threadIdx.x, B = table.B, per = (B + 255) / 256;
    uint32_t *length = start + B + 1, *count = length + B, *held = count + B;
    const uint64_t most = (uint64_t)table.P * R;
    uint64_t mine = 0, total;
    for (uint32_t b = t * per; b < t * per + per && b < B; ++b)
    {
        const uint32_t len = table.p[(size_t)b * table.stride];
        held[b] = len > most ? (uint32_t)most : len;
        length[b] = lengths[(size_t)b * lengths_s];
        count[b] = counts[(size_t)b * counts_s];
        mine += count[b];
    }
    uint64_t at = block_scan(mine, scan, total);
    for (uint32_t b = t * per; b < t * per + per && b < B; ++b)
    {
        start[b] = (uint32_t)min(at, (uint64_t)T);
        at += count[b];
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
        // a count over the length puts the position below 0
        const int64_t pos = (int64_t)length[b] - count[b] + (i - start[b]);
        if (pos >= 0 && pos < held[b])
        {
            const uint32_t page = table.p[(size_t)b * table.stride + 1 + (uint32_t)pos / R];
            const uint64_t slot = (uint64_t)page * R + (uint32_t)pos % R;
            if (slot < kNoPage)
                out = {(uint32_t)slot, (uint32_t)pos};
        }
    }
    map[i] = out;
}

hipError_t launch_slot_map(hipStream_t st, const PageTableView &table, const uint32_t *lengths, uint32_t lengths_s,
                           const uint32_t *counts, uint32_t counts_s, uint32_t *map, uint32_t T, uint32_t page_rows)
{
    static uint64_t done = 0;
    const hipError_t e = lds_attr_once((const void *)slot_map_kernel, (4 * kPagedMaxRows + 1) * 4, done);
    if (e != hipSuccess)
        return e;
    slot_map_kernel<<<(T - 1) / 256 + 1, 256, (4 * (size_t)table.B + 1) * 4, st>>>(table, lengths, lengths_s, counts,
                                                                               counts_s, (uint2 *)map, T, page_rows);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------------------------------------------
// VKLLM_OP_UPDATE_PAGES. A workgroup has one token (or a share of its heads): the rotations of its position go into LDS
// once, then a thread moves units of a head: neighbouring elements, or for pairs of halves as many of both. Bound by HBM for
// prompts, by latency for a token.
struct UpdatePagesArgs
{
    TView cache, k, v;
    const uint32_t *map;
    uint32_t map_s;
    uint32_t units; // of a share: those of 2 KV heads over gridDim.y shares
    bool vec;       // k and v rows are contiguous and start on 16-byte boundaries
    PagedRope rope;
};

// N neighbouring elements in 32 bits
template <typename T, int N> __device__ __forceinline__ void load_n(const T *p, size_t stride, bool vec, float x[N])
{
    typedef T TN __attribute__((ext_vector_type(N)));
    if (vec)
    {
        const TN v = *(const TN *)p;
#pragma unroll
        for (int i = 0; i < N; ++i)
            x[i] = (float)v[i];
        return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
        x[i] = (float)p[i * stride];
}
template <typename T, int N> __device__ __forceinline__ void store_n(T *p, const float x[N])
{
    typedef T TN __attribute__((ext_vector_type(N)));
    TN v;
#pragma unroll
    for (int i = 0; i < N; ++i)
        v[i] = (T)x[i];
    *(TN *)p = v;
}

// HALF: how many elements of each half of a head a thread takes for pairs of halves; 2 HALF neighbouring ones otherwise
template <typename T, int HALF> __global__ __launch_bounds__(256) void update_pages_kernel(UpdatePagesArgs a)
{
    __shared__ float2 cs[kPagedMaxHd / 2];
    const uint32_t tok = blockIdx.x, t = threadIdx.x;
    const uint32_t slot = a.map[(size_t)tok * a.map_s], pos = a.map[(size_t)tok * a.map_s + 1];
    const uint32_t R = a.cache.n[2], hd = a.cache.n[3], KV = a.cache.n[1] / 2;
    const int style = a.rope.style;
    const uint32_t per = hd / (2 * HALF), end = min(2 * KV * per, (blockIdx.y + 1) * a.units);
    const double turns = t < hd / 2 ? a.rope.turns[t] : 0.0;
    uint32_t u = blockIdx.y * a.units + t, h, d0, d1;
    bool halves;
    float x[HALF], y[HALF];
    auto load = [&]() {
        h = u / per;
        halves = style == 2 && h < KV;
        d0 = HALF * (halves ? u % per : 2 * (u % per));
        d1 = d0 + (halves ? hd / 2 : HALF);
        const TView &src = h < KV ? a.k : a.v;
        const T *from = (const T *)src.p + (size_t)tok * src.s[1] + (size_t)(h < KV ? h : h - KV) * src.s[2];
        load_n<T, HALF>(from + (size_t)d0 * src.s[3], src.s[3], a.vec, x);
        load_n<T, HALF>(from + (size_t)d1 * src.s[3], src.s[3], a.vec, y);
    };
    if (u < end)
        load(); // on its way while the slot and the rotations are
    const uint32_t page = slot / R;
    if (page >= a.cache.n[0])
        return;
    if (style)
    {
        if (t < hd / 2)
            cs[t] = turn_at(pos, turns);
        lds_barrier();
    }
    T *to = (T *)a.cache.p + (size_t)page * a.cache.s[0] + (size_t)(slot % R) * hd;
    while (u < end)
    {
        if (halves)
        {
#pragma unroll
            for (int i = 0; i < HALF; ++i)
            {
                const float2 r = cs[d0 + i];
                const float p = x[i], q = y[i];
                x[i] = r.x * p - r.y * q;
                y[i] = r.y * p + r.x * q;
            }
        }
        else if (style && h < KV)
        {
            auto turn = [&](float *v, uint32_t w) {
#pragma unroll
                for (int i = 0; i < HALF / 2; ++i)
                {
                    const float2 r = cs[w + i];
                    const float p = v[2 * i], q = v[2 * i + 1];
                    v[2 * i] = r.x * p - r.y * q;
                    v[2 * i + 1] = r.y * p + r.x * q;
                }
            };
            turn(x, d0 / 2);
            turn(y, d1 / 2);
        }
        T *row = to + (size_t)h * a.cache.s[1];
        store_n<T, HALF>(row + d0, x);
        store_n<T, HALF>(row + d1, y);
        u += 256;
        if (u < end)
            load();
    }
}

hipError_t launch_update_pages(hipStream_t st, const TView &cache, const TView &k, const TView &v, const uint32_t *map,
                               uint32_t map_s, const PagedRope &rope)
{
    auto vec = [](const TView &t) {
        return t.s[3] == 1 && t.s[2] % 8 == 0 && t.s[1] % 8 == 0 && (uintptr_t)t.p % 16 == 0;
    };
    // 16 bytes of each half where heads allow it (a thread then moves 32); us for 4001 tokens of 32 key heads of 128 in fp16,
    // pairs of halves: 8 bytes 31.2, 16 27.8 (27.4 on the GPU, 4.8 TB/s: a large copy's rate is 4.9)
    const uint32_t hd = cache.n[3], half = cache.dt == DT_F16 && hd % 16 == 0 ? 8 : 4;
    const uint32_t T = k.n[1], all = cache.n[1] * (hd / (2 * half));
    const uint32_t shares = min((all - 1) / 256 + 1, T >= 1024 ? 1u : (1023 / T) + 1);
    const uint32_t units = (all - 1) / shares + 1;
    const UpdatePagesArgs a{cache, k, v, map, map_s, units, vec(k) && vec(v), rope};
    const dim3 grid(T, shares);
    if (cache.dt == DT_F32)
        update_pages_kernel<float, 4><<<grid, 256, 0, st>>>(a);
    else if (half == 8)
        update_pages_kernel<_Float16, 8><<<grid, 256, 0, st>>>(a);
    else
        update_pages_kernel<_Float16, 4><<<grid, 256, 0, st>>>(a);
    return hipGetLastError();
}

} // namespace vk
