// VKLLM_OP_PAGED_ATTN: attention of one new token of each sequence over a paged cache. No counterpart in the reference.
//
// For a sequence and a key head, with its queries q_h (up to 16 heads that share the key head), keys k_j and values v_j:
//   out_h = sum_j p_hj v_j / sum_j p_hj,  p_hj = 2^(log2(e) * scale * q_h . k_j - m_h)
// for any m_h, in one pass over the cache: m_h follows the largest score, and sums formed before it rose are scaled down.
// Every byte of keys and values is read once per tile of 16 query heads and used for 2 operations per query head, so HBM
// bounds it.
//
// Work is split without knowing the lengths on the host: a unit is KT consecutive positions of one (sequence, key head),
// all units of the batch are numbered in that order, and each of a fixed number of workgroups (as many as are resident)
// takes an equal run of them. A (sequence, head) that ends up in several workgroups leaves partial sums in the workspace,
// and whichever workgroup of a group of them is the last to arrive joins the group's, up a tree. A workgroup finds
// its units from prefix sums of the lengths, formed in LDS.
//
// Matrix cores do the products although 16 - G of their 16 columns are idle when G heads share a key head: they have 12
// times the rate that the cache arrives at (fp16, operands in two parts; fp32 3 times), and the layout spares the shuffles
// that dot products of single rows need.
// Scores are K Q^T: a wave's 16 keys x 16 heads, of which lane l gets keys 4 (l / 16) + 0..3 of head l % 16. That is, with
// the contraction numbered accordingly, the operand layout of V^T P^T, so probabilities stay in their lanes. V^T
// wants several keys of one dim in a lane: a lane loads HDP / 16 dims of its 4 (8) keys and pairs them up by byte permutes.
#include <algorithm>
#include <type_traits>

#include "device_common.h"
#include "paged_common.h"

namespace vk
{

typedef _Float16 half2 __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kHeadsPerTile = 16;
// What starting and ending a (sequence, head) costs a workgroup, in units (workgroups with many short rows ended last).
// fp16, us with 0 / 1 / 2: 70 ragged rows of up to 8192 over 9 key heads of 64 80 / 74 / 74, 30 over 5 of 256 86 / 79 / 80,
// 200 of up to 500 over 9 of 128 34 / 36 / 37
constexpr uint32_t kSegmentUnits = 1;
constexpr float kNegInf = -INFINITY;

struct PagedAttnArgs
{
    const void *q, *cache;
    void *out;
    uint32_t qs[3], os[3];            // element strides of q and out: sequence, head, dim
    PageTableView table;
    uint32_t pages, KV, G, hd;        // G query heads per key head
    uint32_t page_tiles;              // tiles of 16 rows in a page
    uint32_t page_bytes, head_bytes;  // of a page, and of one head in it
    uint32_t groups;                  // tiles of 16 query heads per key head
    uint32_t tile_heads;              // min(16, G): rows of a partial result
    uint32_t div_magic, div_shift;    // t / page_tiles = t * div_magic >> div_shift for t < 2^28
    float scale_log2;                 // scale * log2(e)
    float *parts;                     // [workgroups][2] partial results
    uint32_t *arrivals;               // [kJoinLevels][workgroups][2] counters, zero between launches
    PagedRope rope;
};

// a partial result: o [tile_heads][hd], then (m, l) [tile_heads]
__host__ __device__ __forceinline__ uint32_t part_floats(uint32_t tile_heads, uint32_t hd)
{
    return tile_heads * (hd + 2);
}

// Two floats of a partial result, written through to the level that all XCDs share and read from there: no workgroup needs
// a device-wide fence, which would write back a whole L2
__device__ __forceinline__ void put2(float *p, float x, float y)
{
    const uint64_t v = (uint64_t)__float_as_uint(y) << 32 | __float_as_uint(x);
    __hip_atomic_store((uint64_t *)p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 get2(const float *p)
{
    const uint64_t v = __hip_atomic_load((const uint64_t *)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return {__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32))};
}

// A thread joins kJoinFan parts of four dims (of eight, loads of both on their way, where a part has more than 256 fours).
// Where it has 128 or fewer, 2, 4 or 8 lanes share a four, so a level takes up to 64 parts. One row of 2000 positions, us
// against pairs of dims joined through LDS: 16 heads on 1 key head 15.0 for 27, 32 on 8 9.6 for 13.1. 16 parts a thread
// took 0.5 to 2 us more nearly everywhere: a level's cost is the round trip and the code's way to the CU.
constexpr uint32_t kJoinFan = 8, kJoinLevels = 4;
static_assert(1u << 3 * kJoinLevels >= kPagedMaxWorkgroups && kPagedArrivals == 2 * kJoinLevels * kPagedMaxWorkgroups);
__device__ __forceinline__ uint32_t join_ways(uint32_t fours)
{
    return fours > 128 ? 1 : fours > 64 ? 2 : fours > 32 ? 4 : 8;
}
struct Joined
{
    float m, l;
    f32x4 o;
};

template <bool F16, int HDP> struct PagedTile
{
    static constexpr int NT = F16 ? 2 : 1;              // tiles of 16 keys a wave takes at once
    static constexpr int KW = 16 * NT, KT = 4 * KW;     // keys per wave, and per unit
    static constexpr int KS = F16 ? HDP / 32 : HDP / 16; // 16-byte loads per key tile
    static constexpr int VD = HDP / 16;                 // dims of a value row that a lane holds
    static constexpr int VW = F16 ? VD / 2 : VD;        // the same in words
    static constexpr int QP = HDP + (F16 ? 8 : 4);      // row pitch of the queries in LDS
    // rotated fp16 queries are kept as two fp16 parts of their halves (a rotation makes them up to sqrt(2) larger), and
    // probabilities as two parts, too: one part each cost 2^-12 on average in the result, as much as its own rounding does,
    // and the matrix cores have the time. Of an infinite or undefined operand the first part's product alone counts: the
    // second part may be 0 or of the other sign.
    static constexpr int QN = F16 ? 2 : 1;
    static constexpr int NP = kHeadsPerTile * HDP / 2 / 256; // query pairs that a thread stages
    // Workgroups per CU. fp16, us with 1 / 2 / 3: 50 rows of up to 8192 over 5 key heads of 128 56 / 58 / 64, 200 rows of up
    // to 500 over 9 39 / 36 / 42, 30 rows of up to 8192 over 5 of 256 79 / 87 / 97, 70 rows over 9 of 64 72 / 74 / 83, one
    // row of 8000 over 8 of 128 18.6 / 15.5 / 15.6
    static constexpr int PER_CU = HDP == 256 ? 1 : 2;
};

// n / d, d > 0, for n below 2^52: the double's rounding is then too small to reach the next whole number. Shorter than a
// division of 64-bit words, of which the code would hold six.
__device__ __forceinline__ uint64_t quotient(uint64_t n, uint64_t d)
{
    return (uint64_t)((double)n / (double)d);
}

__device__ __forceinline__ float exp2_of(float x)
{
    return __builtin_amdgcn_exp2f(x);
}

// u's first part: 0 for 0 only, so that its product with an infinite key is infinite
__device__ __forceinline__ _Float16 first_part(float u)
{
    const _Float16 h = (_Float16)u;
    return h == (_Float16)0.f && u != 0.f ? (_Float16)copysignf(0x1p-24f, u) : h;
}

// both halves of a word within fp16's finite numbers, and what they are beyond them
__device__ __forceinline__ uint32_t finite_halves(uint32_t w)
{
    const half2 most = {65504.f, 65504.f};
    const half2 v = __builtin_elementwise_min(__builtin_elementwise_max(__builtin_bit_cast(half2, w), -most), most);
    return __builtin_bit_cast(uint32_t, v);
}
__device__ __forceinline__ uint32_t beyond_halves(uint32_t w)
{
    const uint32_t v = finite_halves(w);
    const half2 d = __builtin_bit_cast(half2, w) - __builtin_bit_cast(half2, v);
    return __builtin_bit_cast(uint32_t, d);
}

// dynamic LDS, aligned for 16-byte accesses (left to chance, launches took 1 to 2 us more): lengths [B], queries
// [QN][16][QP], per-wave statistics [4][16][2], per-wave sums [4][tile_heads][hd]
// FULL: head_dim is HDP, else it is smaller
template <bool F16, int HDP, bool FULL>
__global__ __launch_bounds__(256, HDP == 256 ? 1 : 2) void paged_attn_kernel(PagedAttnArgs a)
{
    using Tile = PagedTile<F16, HDP>;
    using T = typename std::conditional<F16, _Float16, float>::type;
    constexpr int NT = Tile::NT, KW = Tile::KW, KT = Tile::KT, KS = Tile::KS, VD = Tile::VD, VW = Tile::VW,
                  QP = Tile::QP, QN = Tile::QN, NP = Tile::NP;
    constexpr uint32_t ES = sizeof(T);
    extern __shared__ __align__(16) uint32_t lds[];
    __shared__ uint64_t scan[4], first_unit;
    __shared__ uint32_t first_row, arrived;
    // the rows whose parts lie in slots 0 and 1: how many parts they have, and the number of this one
    struct Split
    {
        uint32_t b, head0, heads, parts, number;
    };
    __shared__ Split split[2];
    const uint32_t t = threadIdx.x, lane = t % kWave, wave = __builtin_amdgcn_readfirstlane(t / kWave);
    const uint32_t g = lane / 16, c = lane % 16;
    const uint32_t B = a.table.B, hd = FULL ? HDP : a.hd, heads = a.KV * a.groups;
    uint32_t *lens = lds;
    T *qs = (T *)(lens + (B + 3) / 4 * 4);
    float *ml = (float *)(qs + QN * kHeadsPerTile * QP), *sums = ml + 4 * kHeadsPerTile * 2;

    // Units of every row, and this workgroup's run of them. A (sequence, head) counts `extra` units more, before its first:
    // what starting and ending it costs. A sum holds units in its low 40 bits and rows that have any above.
    const uint64_t most = (uint64_t)a.table.P * a.page_tiles * 16;
    auto len_of = [&](uint32_t b) {
        const uint32_t len = a.table.p[(size_t)b * a.table.stride];
        return len > most ? (uint32_t)most : len;
    };
    auto units_of = [&](uint32_t len) { return (uint32_t)((len + (uint64_t)KT - 1) / KT); };
    auto count_of = [&](uint32_t len) { return units_of(len) | (uint64_t)(len > 0) << 40; };
    const uint32_t len0 = lane < B ? len_of(lane) : 0; // asked for before anything else
    // rows of the queries that stay zero, and dims past the head
    for (uint32_t i = t; i < QN * kHeadsPerTile * (QP / 4); i += 256)
        if (i / (QP / 4) % kHeadsPerTile >= a.tile_heads || i % (QP / 4) * 4 >= hd)
            for (uint32_t k = 0; k < 4; ++k)
                qs[4 * i + k] = (T)0.f;
    if (t < 2)
        split[t].parts = 0;

    uint32_t extra;
    uint64_t share, u0, u1, base; // base: the number of the first row's first unit
    uint32_t row0;                // the first row
    auto weigh = [&](uint64_t sum) { return ((sum & ((1ull << 40) - 1)) + extra * (sum >> 40)) * heads; };
    auto divide = [&](uint64_t total) {
        // Long rows of 128 dims go to half of the workgroups, one per CU, the others end here: a unit's 64 KB per CU on their
        // way are enough, and no older workgroup runs ahead of a younger one beside it and leaves it the end. Short rows want
        // the second one's loads meanwhile; few units of few rows would have fewer loads on their way, for the same joins.
        // us with all / half of them: 2 rows of up to 131072 on 4 key heads 76.7 / 71, 1 of 3000 on 32 16.1 / 14.2, 2 of 1100
        // 18.3 / 13, 50 ragged ones of up to 8192 on 5 58 / 56, and fp32 60 / 58.5; but 64 of 8192 on 8 358 / 360 (fp32, of 768,
        // 72 / 74), and kept out 2048 of 100 196 / 216, 64 of 1024 on 8 of 64 dims 27 / 36.
        // With 1 to 4 units a workgroup the gain hangs on how many (sequence, key head)s are cut, and on how large their parts
        // are. 8 totals between 530 and 2000 units, half of the workgroups against all, in the mean (and from, to): 2 and 4 query
        // heads to a key head, 4 pairs +1% (-17, +13), 8 -1% (-12, +12), 12 -10% (-26, +1), 16 -5% (-12, +5), 32 -9% (-21, +1); 5 to
        // 16 query heads, 8 +1% (-8, +21), 12 -8% (-32, +4), 16 +2% (-11, +24), 20 -3% (-35, +25), 24 +4% (-11, +23), 26 -9% (-40,
        // +1), 28 -14%, 32 -14%. So from between 8 and 12 pairs where parts are small, else from between 24 and 26.
        const uint64_t units = (total & ((1ull << 40) - 1)) * heads, rows = (total >> 40) * heads;
        const uint32_t n = gridDim.x;
        const bool alone = FULL && HDP == 128 && units >= 6 * rows &&
                           (units >= 4 * n || (units > n && (a.tile_heads <= 4 ? 48 : 20) * rows >= n));
        const uint32_t sharers = alone ? (n + 1) / 2 : n;
        extra = units > 4 * n ? kSegmentUnits : 0;
        share = quotient(weigh(total) + sharers - 1, sharers);
        u0 = blockIdx.x * share;
        u1 = min(u0 + share, weigh(total));
    };
    if (B <= kWave)
    {
        // every wave for itself
        if (lane < B)
            lens[lane] = len0;
        const uint64_t mine = count_of(len0), upto = wave_scan(mine);
        divide(read_lane(upto, kWave - 1));
        const uint64_t found = __ballot(u0 < weigh(upto) && u0 >= weigh(upto - mine));
        row0 = found ? __ffsll((unsigned long long)found) - 1 : 0;
        base = weigh(read_lane(upto - mine, row0));
    }
    else
    {
        const uint32_t per = (B + 255) / 256;
        uint64_t mine = 0, total;
        for (uint32_t b = t * per; b < t * per + per && b < B; ++b)
        {
            lens[b] = len_of(b);
            mine += count_of(lens[b]);
        }
        uint64_t at = block_scan(mine, scan, total);
        divide(total);
        if (u0 >= weigh(at) && u0 < weigh(at + mine))
        {
            uint32_t b = t * per;
            for (; u0 >= weigh(at + count_of(lens[b])); ++b)
                at += count_of(lens[b]);
            first_unit = weigh(at);
            first_row = b;
        }
        __syncthreads();
        row0 = first_row;
        base = first_unit;
    }
    // sequences without a token
    for (uint32_t b = blockIdx.x; b < B; b += gridDim.x)
        if (lens[b] == 0)
            for (uint32_t e = t; e < a.KV * a.G * hd; e += 256)
                ((T *)a.out)[(size_t)b * a.os[0] + (size_t)(e / hd) * a.os[1] + (size_t)(e % hd) * a.os[2]] = (T)0.f;
    if (u0 >= u1)
        return;

    // A unit's place: sequence b of `len` positions and n units per head, key head h and tile g of its query heads, unit s of
    // number v. The same for the whole workgroup, so it is kept in scalar registers.
    struct Place
    {
        uint32_t b, len, n, h, g, s;
        uint32_t v; // behind u0
    };
    auto row_at = [&](Place &p, uint32_t b) {
        do
            p.len = __builtin_amdgcn_readfirstlane(lens[b]);
        while (p.len == 0 && ++b < B);
        p.b = b;
        p.n = units_of(p.len);
    };
    auto next_of = [&](Place p) {
        ++p.v;
        if (++p.s == p.n)
        {
            p.s = 0;
            p.v += extra;
            if (++p.g == a.groups)
            {
                p.g = 0;
                if (++p.h == a.KV)
                {
                    p.h = 0;
                    row_at(p, min(p.b + 1, B - 1));
                }
            }
        }
        return p;
    };
    Place cur;
    row_at(cur, __builtin_amdgcn_readfirstlane(row0));
    {
        const uint64_t rel = u0 - base;
        const uint32_t n = cur.n + extra, hg = (uint32_t)quotient(rel, n), at = (uint32_t)(rel - (uint64_t)hg * n);
        cur.h = __builtin_amdgcn_readfirstlane(hg / a.groups);
        cur.g = __builtin_amdgcn_readfirstlane(hg % a.groups);
        cur.s = __builtin_amdgcn_readfirstlane(at < extra ? 0 : at - extra);
        cur.v = __builtin_amdgcn_readfirstlane(at < extra ? extra - at : 0);
    }
    const uint32_t end = __builtin_amdgcn_readfirstlane((uint32_t)(u1 - u0));
    if (cur.v >= end)
        return;

    // its query heads: the first of them, and how many
    auto head0_of = [&](const Place &p) { return p.h * a.G + p.g * kHeadsPerTile; };
    auto heads_of = [&](const Place &p) -> uint32_t { return min((uint32_t)kHeadsPerTile, a.G - p.g * kHeadsPerTile); };

    // Queries and their pairs' frequencies: thread t has pairs t + 256 j of tile_heads heads (the other rows in LDS stay
    // zero). They are asked for before the keys of their first unit, and staged when the unit before is done with.
    T qx[NP], qy[NP];
    double turns[NP];
    auto pair_dims = [&](uint32_t w, uint32_t &d0, uint32_t &d1) {
        d0 = a.rope.style == 1 ? 2 * w : w;
        d1 = a.rope.style == 1 ? 2 * w + 1 : w + hd / 2;
    };
    auto load_q = [&](const Place &p) {
        const uint32_t head0 = head0_of(p), Gn = heads_of(p);
#pragma unroll
        for (int j = 0; j < NP; ++j)
            if (256 * j < a.tile_heads * (hd / 2))
            {
                const uint32_t e = t + 256 * j, i = e / (hd / 2), w = e % (hd / 2);
                uint32_t d0, d1;
                pair_dims(w, d0, d1);
                const T *q = (const T *)a.q + (size_t)p.b * a.qs[0] + (size_t)(head0 + (i < Gn ? i : 0)) * a.qs[1];
                qx[j] = q[(size_t)d0 * a.qs[2]];
                qy[j] = q[(size_t)d1 * a.qs[2]];
                turns[j] = a.rope.turns[w];
            }
    };
    auto stage_q = [&](const Place &p) {
        const uint32_t Gn = heads_of(p);
#pragma unroll
        for (int j = 0; j < NP; ++j)
            if (256 * j < a.tile_heads * (hd / 2))
            {
                const uint32_t e = t + 256 * j, i = e / (hd / 2), w = e % (hd / 2);
                uint32_t d0, d1;
                pair_dims(w, d0, d1);
                float u = i < Gn ? (float)qx[j] : 0.f, v = i < Gn ? (float)qy[j] : 0.f;
                if (i >= a.tile_heads)
                    continue;
                if (a.rope.style)
                {
                    const float2 r = turn_at(p.len - 1, turns[j]);
                    const float x = u, y = v;
                    u = r.x * x - r.y * y;
                    v = r.y * x + r.x * y;
                    if constexpr (F16)
                    {
                        const float hu = 0.5f * u, hv = 0.5f * v;
                        u = (float)first_part(hu);
                        v = (float)first_part(hv);
                        qs[(kHeadsPerTile + i) * QP + d0] = (T)(hu - u);
                        qs[(kHeadsPerTile + i) * QP + d1] = (T)(hv - v);
                    }
                }
                qs[i * QP + d0] = (T)u;
                qs[i * QP + d1] = (T)v;
            }
    };

    // pages of the wave's tiles in a unit
    uint32_t pid[NT];
    auto tile_of = [&](const Place &p, int i) { return (p.s * KT + wave * KW) / 16 + i; };
    auto page_of = [&](uint32_t tile) { return (uint32_t)((uint64_t)tile * a.div_magic >> a.div_shift); };
    auto fetch = [&](const Place &p) {
        const uint32_t *row = a.table.p + (size_t)p.b * a.table.stride + 1;
#pragma unroll
        for (int i = 0; i < NT; ++i)
            pid[i] = scalar_word(row + page_of(min(tile_of(p, i), (p.len - 1) / 16)));
    };
    // A tile's rows start at an address of the wave, to which every lane adds an offset of its own that never changes.
    const char *rows[NT];
    uint32_t live[NT]; // the tiles' keys
    auto place = [&](const Place &p) {
#pragma unroll
        for (int i = 0; i < NT; ++i)
        {
            const uint32_t tile = tile_of(p, i);
            // past the end, or an absent page: read page 0, use nothing of it
            const bool there = tile <= (p.len - 1) / 16 && pid[i] < a.pages;
            live[i] = there ? min(16u, p.len - tile * 16) : 0u;
            const uint32_t in_page = tile - page_of(tile) * a.page_tiles;
            const size_t at = (size_t)pid[i] * a.page_bytes + (p.h * a.head_bytes + in_page * (16 * hd * ES));
            rows[i] = (const char *)a.cache + (there ? at : 0);
        }
    };
    u32x4 kr[NT][KS];
    uint32_t vr[NT * 4][VW];
    auto load_k = [&]() {
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int s = 0; s < KS; ++s)
            {
                const uint32_t d = 16 * g + 64 * s; // bytes
                kr[i][s] = *(const u32x4 *)(rows[i] + (c * hd * ES + (FULL || d < hd * ES ? d : 0)));
            }
    };
    auto load_v = [&]() {
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r)
            {
                uint32_t *to = vr[4 * i + r];
                const char *p = rows[i] + (size_t)a.KV * a.head_bytes + r * hd * ES;
                if constexpr (VW == 2)
                {
                    const uint32_t d = 8 * c;
                    const uint2 v = *(const uint2 *)(p + (4 * g * hd * ES + (FULL || d < hd * ES ? d : 0)));
                    to[0] = v.x;
                    to[1] = v.y;
                }
                else
                {
#pragma unroll
                    for (int w = 0; w < VW / 4; ++w)
                    {
                        const uint32_t d = VD * ES * c + 16 * w;
                        const u32x4 v = *(const u32x4 *)(p + (4 * g * hd * ES + (FULL || d < hd * ES ? d : 0)));
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            to[4 * w + k] = v[k];
                    }
                }
            }
    };

    float m, l;
    f32x4 o[VD];
    auto clear = [&]() {
        m = kNegInf;
        l = 0.f;
#pragma unroll
        for (int d = 0; d < VD; ++d)
            o[d] = (f32x4){0.f, 0.f, 0.f, 0.f};
    };
    uint32_t q_at = c * QP + (F16 ? 8 : 4) * g;

    // One unit; `more`: with the loads of the unit `next` (and the pages of the one `after` it). The last unit is code of its
    // own, because where paths with and without newer loads meet, the compiler waits for all of them.
    auto step = [&](auto more, const Place &next, const Place &after) {
        constexpr bool MORE = decltype(more)::value;
        // read again at every step (the compiler is kept from moving that out of the loop): in registers the queries would
        // cost half of the resident waves
        asm volatile("" : "+v"(q_at));
        auto query = [&](int n, int s) {
            return *(const u32x4 *)(qs + q_at + n * kHeadsPerTile * QP + (F16 ? 32 : 16) * s);
        };
        f32x4 x[NT], rest[NT]; // scores; what the queries' second parts add
#pragma unroll
        for (int i = 0; i < NT; ++i)
            x[i] = rest[i] = (f32x4){0.f, 0.f, 0.f, 0.f};
        if constexpr (!FULL)
#pragma unroll
            for (int k = 0; k < KS; ++k)
                if (16 * g + 64 * k >= hd * ES) // past the row: not a number for sure
#pragma unroll
                    for (int i = 0; i < NT; ++i)
                        kr[i][k] = (u32x4){0, 0, 0, 0};
        if constexpr (F16)
        {
            auto score = [&](int n, f32x4(&x)[NT]) {
#pragma unroll
                for (int k = 0; k < KS; ++k)
                {
                    const half8 q = __builtin_bit_cast(half8, query(n, k));
#pragma unroll
                    for (int i = 0; i < NT; ++i)
                        x[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, kr[i][k]), q, x[i], 0, 0, 0);
                }
            };
            score(0, x);
            if (a.rope.style)
                score(1, rest);
        }
        else
        {
#pragma unroll
            for (int k = 0; k < KS; ++k)
            {
                const u32x4 q = query(0, k);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    x[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kr[0][k][e]), __uint_as_float(q[e]), x[0], 0,
                                                                0, 0);
            }
        }
        uint32_t n[NT];
        bool whole = true;
#pragma unroll
        for (int i = 0; i < NT; ++i)
        {
            n[i] = live[i];
            whole = whole && n[i] == 16;
        }
        if constexpr (MORE)
        {
            place(next);
            if (next.s == 0)
                load_q(next);
            load_k();
            fetch(after);
        }
        float top = kNegInf;
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r)
            {
                if constexpr (F16) // where a score is finite, so is the rest
                    x[i][r] += fabsf(rest[i][r]) < INFINITY ? rest[i][r] : 0.f;
                x[i][r] *= a.scale_log2;
                if (!whole && 4 * g + r >= n[i])
                    x[i][r] = kNegInf;
                top = fmaxf(top, x[i][r]);
            }
        // m rises when a score passes it by 7: probabilities then stay below 2^15 at the 2^8 that fp16 ones are scaled by, and
        // those down to 2^-32 of the largest still count
        if (__any(top > m + 7.f))
        {
            top = fmaxf(top, __shfl_xor(top, 16, kWave));
            top = fmaxf(top, __shfl_xor(top, 32, kWave));
            const float high = fmaxf(m, top), f = m == kNegInf ? 0.f : exp2_of(m - high);
            m = high;
            l *= f;
#pragma unroll
            for (int d = 0; d < VD; ++d)
                o[d] *= f;
        }
        const float ref = m == kNegInf ? 0.f : m - (F16 ? 8.f : 0.f);
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r)
            {
                x[i][r] = exp2_of(x[i][r] - ref);
                l += x[i][r];
            }
        if (!whole) // what lies past the end is not a number for sure
        {
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int w = 0; w < VW; ++w)
                        vr[4 * i + r][w] = 4 * g + r < n[i] ? vr[4 * i + r][w] : 0u;
        }
        if constexpr (F16)
        {
            half8 p, q; // p's rest
#pragma unroll
            for (int j = 0; j < 8; ++j)
            {
                p[j] = (_Float16)x[j / 4][j % 4];
                q[j] = (_Float16)(x[j / 4][j % 4] - (float)p[j]);
            }
            auto values = [&](int d) { // 8 keys of dim VD * c + d
                u32x4 v;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    v[j] = __builtin_amdgcn_perm(vr[2 * j + 1][d / 2], vr[2 * j][d / 2], d % 2 ? 0x07060302u : 0x05040100u);
                return v;
            };
            // the values times 0: not a number if one of them is none or infinite. One row of 12000 positions, 32 heads on 8: 18.3
            // us for 18.0 without; batches and long rows level.
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 2 * 4; ++j)
#pragma unroll
                for (int w = 0; w < VW; ++w)
                    sum = __builtin_amdgcn_fdot2(__builtin_bit_cast(half2, vr[j][w]), (half2){0.f, 0.f}, sum, false);
            if (__builtin_expect(__any(sum != sum), 0))
            {
                // What values are beyond the finite numbers (infinite, undefined; 0 for the others) counts once for every
                // weight that is not 0; the rest of them goes the way of all values.
                half8 one;
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    one[j] = x[j / 4][j % 4] > 0.f ? (_Float16)1.f : p[j];
#pragma unroll
                for (int d = 0; d < VD; ++d)
                {
                    u32x4 v = values(d);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        v[j] = beyond_halves(v[j]);
                    o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, v), one, o[d], 0, 0, 0);
                }
#pragma unroll
                for (int j = 0; j < 2 * 4; ++j)
#pragma unroll
                    for (int w = 0; w < VW; ++w)
                        vr[j][w] = finite_halves(vr[j][w]);
            }
#pragma unroll
            for (int d = 0; d < VD; ++d)
            {
                const half8 v = __builtin_bit_cast(half8, values(d));
                o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p, o[d], 0, 0, 0);
                o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, q, o[d], 0, 0, 0);
            }
        }
        else
        {
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int d = 0; d < VD; ++d)
                    o[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vr[r][d]), x[0][r], o[d], 0, 0, 0);
        }
        if constexpr (MORE)
            load_v();
    };

    auto store_out = [&](uint32_t b, uint32_t head, uint32_t d, float o0, float o1, float lsum) {
        T *to = (T *)a.out + (size_t)b * a.os[0] + (size_t)head * a.os[1] + (size_t)d * a.os[2];
        to[0] = (T)(lsum == 0.f ? 0.f : o0 / lsum); // a row of no weight is zero
        to[a.os[2]] = (T)(lsum == 0.f ? 0.f : o1 / lsum);
    };
    // What the workgroup has of p's sequence and heads: its units from `from` to p.s
    auto finish = [&](const Place &p, uint32_t from) {
        const uint32_t Gn = heads_of(p), head0 = head0_of(p);
        l += __shfl_xor(l, 16, kWave);
        l += __shfl_xor(l, 32, kWave);
        if (c < Gn)
        {
            if (g == 0)
            {
                ml[(wave * kHeadsPerTile + c) * 2] = m;
                ml[(wave * kHeadsPerTile + c) * 2 + 1] = l;
            }
            float *to = sums + (size_t)(wave * a.tile_heads + c) * hd;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int d = 0; d < VD; ++d)
                    if (FULL || VD * (4 * g + i) + d < hd)
                        to[VD * (4 * g + i) + d] = o[d][i];
        }
        lds_barrier();
        const bool all = from == 0 && p.s + 1 == p.n;
        // a row that began in another workgroup leaves its part in slot 0, one that goes on in the next in slot 1
        float *part = a.parts + (2 * blockIdx.x + (from == 0 ? 1 : 0)) * part_floats(a.tile_heads, hd);
        for (uint32_t e = t; e < Gn * (HDP / 2); e += 256)
        {
            const uint32_t i = e / (HDP / 2), d = e % (HDP / 2) * 2;
            if (!FULL && d >= hd)
                continue;
            float mw[4], top = kNegInf, lsum = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll
            for (int w = 0; w < 4; ++w)
            {
                mw[w] = ml[(w * kHeadsPerTile + i) * 2];
                top = fmaxf(top, mw[w]);
            }
#pragma unroll
            for (int w = 0; w < 4; ++w)
            {
                const float f = mw[w] == kNegInf ? 0.f : exp2_of(mw[w] - top);
                const float *sum = sums + (size_t)(w * a.tile_heads + i) * hd + d;
                lsum += f * ml[(w * kHeadsPerTile + i) * 2 + 1];
                o0 += f * sum[0];
                o1 += f * sum[1];
            }
            if (all)
                store_out(p.b, head0 + i, d, o0, o1, lsum);
            else
            {
                put2(part + i * hd + d, o0, o1);
                if (d == 0)
                    put2(part + a.tile_heads * hd + 2 * i, top, lsum);
            }
        }
    };

    load_q(cur);
    fetch(cur);
    place(cur);
    load_k();
    load_v();
    Place next = next_of(cur);
    if (next.v < end)
        fetch(next);
    stage_q(cur);
    clear();
    lds_barrier();
    uint32_t from = cur.s;
    auto note = [&](const Place &p, uint32_t from) {
        const uint32_t before = (uint32_t)quotient(from + share - 1, share),
                       behind = (uint32_t)quotient(p.n - p.s - 1 + share - 1, share);
        if (t == 0)
            split[from == 0] = {p.b, head0_of(p), heads_of(p), before + 1 + behind, before};
    };
    while (next.v < end)
    {
        const Place after = next_of(next); // with v >= end, another workgroup's or none
        step(std::true_type(), next, after.v < end ? after : next);
        if (next.s == 0)
        {
            finish(cur, from);
            if (from != 0)
                note(cur, from);
            stage_q(next);
            clear();
            from = 0;
            lds_barrier();
        }
        cur = next;
        next = after;
    }
    step(std::false_type(), cur, cur);
    finish(cur, from);
    if (from != 0 || cur.s + 1 < cur.n)
        note(cur, from);

    // Joins. Parts that lie next to each other form groups of `fan`; the last workgroup of a group to arrive (no workgroup
    // waits for another) joins its parts in their order, into the first one's place, and arrives for the group at the next
    // level. Which parts are joined with which depends on the lengths alone, so results do not hang on the arrivals' order.
    __syncthreads();
#pragma unroll 1
    for (int which = 0; which < 2; ++which)
    {
        uint32_t n = __builtin_amdgcn_readfirstlane(split[which].parts);
        if (n == 0)
            continue;
        const uint32_t head0 = __builtin_amdgcn_readfirstlane(split[which].head0),
                       Gn = __builtin_amdgcn_readfirstlane(split[which].heads);
        uint32_t k = __builtin_amdgcn_readfirstlane(split[which].number), stride = 1;
        const uint32_t first = blockIdx.x - k, fours = Gn * (HDP / 4);
        const uint32_t ways = join_ways(fours), fan = kJoinFan * ways;
        const uint32_t floats = part_floats(a.tile_heads, hd), half = 2 * gridDim.x * floats; // of 2^26 at most
        // the place of part k: the first part's row starts in its workgroup, the others' does not
        auto slot = [&](uint32_t k) { return 2 * (first + k) + (k == 0 ? 1 : 0); };
        for (uint32_t level = 0;; ++level)
        {
            const uint32_t group = k / fan, size = min(fan, n - group * fan), lead = group * fan * stride;
            __builtin_amdgcn_s_waitcnt(0); // what this thread wrote of the part is there
            __syncthreads();
            if (t == 0)
            {
                uint32_t *counter = a.arrivals + 2 * level * gridDim.x + slot(lead);
                arrived = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                if (arrived == size - 1)
                    __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); // for the next launch
            }
            __syncthreads();
            if (arrived != size - 1)
                break;
            // levels write one half of the workspace and read the other, so nothing is overwritten that is still read
            const float *in = a.parts + (level % 2) * half;
            float *to = a.parts + (1 - level % 2) * half + slot(lead) * floats;
            // fours e, e + 256, ... from parts way, way + ways, ... of the group (what lies past it repeats its last)
            auto gather = [&](auto count, Joined *r, uint32_t e, uint32_t way) {
                constexpr int N = decltype(count)::value;
                float2 o[N][kJoinFan][2], ml[N][kJoinFan];
#pragma unroll
                for (int j = 0; j < N; ++j)
                {
                    const uint32_t f = min(e + 256 * j, fours - 1), i = f / (HDP / 4), d = min(f % (HDP / 4) * 4, hd - 4);
#pragma unroll
                    for (uint32_t c = 0; c < kJoinFan; ++c)
                    {
                        o[j][c][0] = o[j][c][1] = ml[j][c] = {0.f, 0.f};
                        if (c * ways >= size)
                            continue;
                        const float *part = in + slot(lead + min(way + c * ways, size - 1) * stride) * floats;
                        o[j][c][0] = get2(part + i * hd + d);
                        o[j][c][1] = get2(part + i * hd + d + 2);
                        ml[j][c] = get2(part + a.tile_heads * hd + 2 * i);
                    }
                }
#pragma unroll
                for (int j = 0; j < N; ++j)
                {
                    Joined x = {kNegInf, 0.f, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
                    for (uint32_t c = 0; c < kJoinFan; ++c)
                    {
                        if (way + c * ways >= size)
                            ml[j][c].x = kNegInf;
                        x.m = fmaxf(x.m, ml[j][c].x);
                    }
#pragma unroll
                    for (uint32_t c = 0; c < kJoinFan; ++c)
                    {
                        // a part without a largest score counts with 0, which keeps a sum that is not a number one; a part
                        // that is none not at all, whose sums may be infinite
                        const float f = ml[j][c].x == kNegInf ? 0.f : exp2_of(ml[j][c].x - x.m);
                        const f32x4 sums = {o[j][c][0].x, o[j][c][0].y, o[j][c][1].x, o[j][c][1].y};
                        if (way + c * ways < size)
                        {
                            x.l += f * ml[j][c].y;
                            x.o += f * sums;
                        }
                    }
                    r[j] = x;
                }
            };
            auto emit = [&](uint32_t e, const Joined &r) {
                const uint32_t i = e / (HDP / 4), d = e % (HDP / 4) * 4;
                if (e >= fours || (!FULL && d >= hd))
                    return;
                if (n <= fan)
                {
                    store_out(split[which].b, head0 + i, d, r.o[0], r.o[1], r.l);
                    store_out(split[which].b, head0 + i, d + 2, r.o[2], r.o[3], r.l);
                }
                else
                {
                    put2(to + i * hd + d, r.o[0], r.o[1]);
                    put2(to + i * hd + d + 2, r.o[2], r.o[3]);
                    if (d == 0)
                        put2(to + a.tile_heads * hd + 2 * i, r.m, r.l);
                }
            };
            if (fours > 256)
                for (uint32_t e = t; e < fours; e += 512)
                {
                    Joined r[2];
                    gather(std::integral_constant<int, 2>(), r, e, 0);
                    emit(e, r[0]);
                    emit(e + 256, r[1]);
                }
            else
            {
                Joined r;
                gather(std::integral_constant<int, 1>(), &r, t / ways, t % ways);
                for (uint32_t w = 1; w < ways; w *= 2)
                {
                    const float m = __shfl_xor(r.m, w, kWave), l = __shfl_xor(r.l, w, kWave), top = fmaxf(r.m, m);
                    const float f = r.m == kNegInf ? 0.f : exp2_of(r.m - top), h = m == kNegInf ? 0.f : exp2_of(m - top);
                    r.m = top;
                    r.l = f * r.l + h * l;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        r.o[i] = f * r.o[i] + h * __shfl_xor(r.o[i], w, kWave);
                }
                if (t % ways == 0)
                    emit(t / ways, r);
            }
            if (n <= fan)
                break;
            k = group;
            n = (n - 1) / fan + 1;
            stride *= fan;
        }
    }
}

template <bool F16, int HDP, bool FULL>
static hipError_t launch_as(hipStream_t st, PagedAttnArgs &a, size_t work_elems, int cu_count)
{
    using Tile = PagedTile<F16, HDP>;
    const void *fn = (const void *)paged_attn_kernel<F16, HDP, FULL>;
    const size_t lds = (size_t)(a.table.B + 3) / 4 * 16 + Tile::QN * kHeadsPerTile * Tile::QP * (F16 ? 2 : 4) +
                       4 * kHeadsPerTile * 8 + (size_t)4 * a.tile_heads * a.hd * 4;
    static uint64_t done = 0;
    const hipError_t e = lds_attr_once(fn, 128 << 10, done);
    if (e != hipSuccess)
        return e;
    const size_t want = std::min<size_t>((size_t)Tile::PER_CU * cu_count, kPagedMaxWorkgroups);
    const uint32_t grid = (uint32_t)std::min(want, work_elems / (4 * part_floats(a.tile_heads, a.hd)));
    if (grid == 0)
        return hipErrorOutOfMemory;
    paged_attn_kernel<F16, HDP, FULL><<<grid, 256, lds, st>>>(a);
    return hipGetLastError();
}

hipError_t launch_paged_attn(hipStream_t st, const TView &q, const TView &cache, const PageTableView &table,
                             const TView &out, float scale, const PagedRope &rope, float *work, size_t work_elems,
                             uint32_t *arrivals, int cu_count)
{
    const uint32_t KV = cache.n[1] / 2, G = q.n[2] / KV, R = cache.n[2], hd = q.n[3], es = cache.dt == DT_F16 ? 2 : 4;
    PagedAttnArgs a{};
    a.q = q.p;
    a.cache = cache.p;
    a.out = out.p;
    for (int i = 0; i < 3; ++i)
    {
        a.qs[i] = q.s[i + 1];
        a.os[i] = out.s[i + 1];
    }
    a.table = table;
    a.pages = cache.n[0];
    a.KV = KV;
    a.G = G;
    a.hd = hd;
    a.page_tiles = R / 16;
    a.head_bytes = R * hd * es;
    a.page_bytes = 2 * KV * a.head_bytes;
    a.groups = (G - 1) / kHeadsPerTile + 1;
    a.tile_heads = std::min(G, (uint32_t)kHeadsPerTile);
    // 2^28 * (div_magic * d - 2^div_shift) < 2^28 * d <= 2^div_shift, so the quotient of any t < 2^28 is exact
    while ((1u << a.div_shift) < a.page_tiles)
        ++a.div_shift;
    a.div_shift += 28;
    a.div_magic = (uint32_t)((((uint64_t)1 << a.div_shift) + a.page_tiles - 1) / a.page_tiles);
    // the kernel halves rotated fp16 queries
    a.scale_log2 = (es == 2 && rope.style ? 2.f : 1.f) * scale * 1.44269504088896340736f;
    a.rope = rope;
    a.parts = work;
    a.arrivals = arrivals;
    const auto run = [&](auto f16) {
        constexpr bool F16 = decltype(f16)::value;
        return hd == 64    ? launch_as<F16, 64, true>(st, a, work_elems, cu_count)
               : hd < 64   ? launch_as<F16, 64, false>(st, a, work_elems, cu_count)
               : hd == 128 ? launch_as<F16, 128, true>(st, a, work_elems, cu_count)
               : hd < 128  ? launch_as<F16, 128, false>(st, a, work_elems, cu_count)
               : hd == 256 ? launch_as<F16, 256, true>(st, a, work_elems, cu_count)
                           : launch_as<F16, 256, false>(st, a, work_elems, cu_count);
    };
    return cache.dt == DT_F16 ? run(std::true_type()) : run(std::false_type());
}

} // namespace vk
