// VKLLM_OP_PAGED_ATTN: attention of one new token of each sequence over a paged cache. No counterpart in the reference.
//
// For a sequence and a key head, with its queries q_h (up to 16 heads that share the key head), keys k_j and values v_j:
//   out_h = sum_j p_hj v_j / sum_j p_hj,  p_hj = 2^(log2(e) * scale * q_h . k_j - m_h)
// for any m_h, in one pass over the cache: m_h follows the largest score, and sums formed before it rose are scaled down.
// Every byte of keys and values is read once and used for 2 operations per query head, so HBM bounds it.
//
// Work is split without knowing the lengths on the host: a unit is KT consecutive positions of one (sequence, key head),
// all units of the batch are numbered in that order, and each of a fixed number of workgroups (as many as are resident)
// takes an equal run of them. A (sequence, head) that ends up in several workgroups leaves partial sums in the workspace,
// which a second kernel joins. A workgroup finds its units from prefix sums of the lengths, formed in LDS.
//
// Matrix cores do the products although 16 - G of their 16 columns are idle when G heads share a key head: they have 24
// times the rate that the cache arrives at, and the layout spares the shuffles that dot products of single rows need.
// Scores are K Q^T: a wave's 16 keys x 16 heads, of which lane l gets keys 4 (l / 16) + 0..3 of head l % 16. That is, with
// the contraction numbered accordingly, the operand layout of V^T P^T, so probabilities stay in their lanes. V^T
// wants several keys of one dim in a lane: a lane loads HDP / 16 dims of its 4 (8) keys and pairs them up by byte permutes.
#include "device_common.h"
#include "paged_common.h"

namespace vk
{

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kHeadsPerTile = 16;
constexpr float kNegInf = -INFINITY;

struct PagedAttnArgs
{
    TView q, cache, out;
    PageTableView table;
    float scale_log2;  // scale * log2(e)
    uint32_t groups;   // tiles of 16 query heads per key head
    uint32_t tile_heads; // min(16, heads per key head): rows of a partial result
    float *parts;      // [workgroups][2] partial results
    uint32_t *joins;   // [workgroups][4]: what each workgroup leaves to be joined
    PagedRope rope;
};

// a partial result: m [tile_heads], l [tile_heads], o [tile_heads][hd]
__host__ __device__ __forceinline__ size_t part_floats(uint32_t tile_heads, uint32_t hd)
{
    return (size_t)tile_heads * (hd + 2);
}

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
    // and the matrix cores have the time
    static constexpr int QN = F16 ? 2 : 1;
};

__device__ __forceinline__ float exp2_of(float x)
{
    return __builtin_amdgcn_exp2f(x);
}

// dynamic LDS: lengths [B], queries [QN][16][QP], per-wave statistics [4][16][2], per-wave sums [4][tile_heads][hd]
template <bool F16, int HDP> __global__ __launch_bounds__(256) void paged_attn_kernel(PagedAttnArgs a)
{
    using Tile = PagedTile<F16, HDP>;
    using T = typename std::conditional<F16, _Float16, float>::type;
    constexpr int NT = Tile::NT, KW = Tile::KW, KT = Tile::KT, KS = Tile::KS, VD = Tile::VD, VW = Tile::VW,
                  QP = Tile::QP, QN = Tile::QN;
    extern __shared__ uint32_t lds[];
    __shared__ uint64_t scan[4], first_unit;
    __shared__ uint32_t first_row;
    const uint32_t t = threadIdx.x, lane = t % kWave, wave = __builtin_amdgcn_readfirstlane(t / kWave);
    const uint32_t g = lane / 16, c = lane % 16;
    const uint32_t B = a.table.B, KV = a.cache.n[1] / 2, R = a.cache.n[2], hd = a.cache.n[3], H = a.q.n[2], G = H / KV;
    uint32_t *lens = lds;
    T *qs = (T *)(lens + (B + 3) / 4 * 4);
    float *ml = (float *)(qs + QN * kHeadsPerTile * QP), *sums = ml + 4 * kHeadsPerTile * 2;

    // units of every row, and this workgroup's run of them
    const uint32_t per = (B + 255) / 256;
    const uint64_t most = (uint64_t)a.table.P * R;
    uint64_t mine = 0, total;
    for (uint32_t b = t * per; b < t * per + per && b < B; ++b)
    {
        const uint32_t len = a.table.p[(size_t)b * a.table.stride];
        lens[b] = len > most ? (uint32_t)most : len;
        mine += (uint64_t)((lens[b] + (uint64_t)KT - 1) / KT) * KV * a.groups;
    }
    for (uint32_t i = t; i < QN * kHeadsPerTile * QP; i += 256)
        qs[i] = (T)0.f;
    const uint64_t before = block_scan(mine, scan, total);
    const uint64_t share = (total + gridDim.x - 1) / gridDim.x;
    const uint64_t u0 = blockIdx.x * share, u1 = min(u0 + share, total);
    if (u0 >= before && u0 < before + mine)
    {
        uint64_t at = before;
        uint32_t b = t * per;
        for (;; ++b)
        {
            const uint64_t n = (uint64_t)((lens[b] + (uint64_t)KT - 1) / KT) * KV * a.groups;
            if (u0 < at + n)
                break;
            at += n;
        }
        first_unit = at;
        first_row = b;
    }
    __syncthreads();
    // sequences without a token
    for (uint32_t b = blockIdx.x; b < B; b += gridDim.x)
        if (lens[b] == 0)
            for (uint32_t e = t; e < H * hd; e += 256)
                ((T *)a.out.p)[(size_t)b * a.out.s[1] + (size_t)(e / hd) * a.out.s[2] + (size_t)(e % hd) * a.out.s[3]] =
                    (T)0.f;
    if (t == 0)
        a.joins[blockIdx.x * 4] = 0;
    if (u0 >= u1)
        return;

    uint64_t base = first_unit;
    uint32_t b = first_row;
    for (uint64_t u = u0; u < u1;)
    {
        const uint32_t len = lens[b], n_units = (uint32_t)((len + (uint64_t)KT - 1) / KT);
        const uint64_t row_units = (uint64_t)n_units * KV * a.groups;
        if (u >= base + row_units)
        {
            base += row_units;
            ++b;
            continue;
        }
        const uint32_t hg = (uint32_t)((u - base) / n_units), s0 = (uint32_t)((u - base) % n_units);
        const uint32_t s1 = (uint32_t)min((uint64_t)n_units, s0 + (u1 - u));
        const uint32_t h = hg / a.groups, head0 = h * G + hg % a.groups * kHeadsPerTile;
        const uint32_t Gn = min((uint32_t)kHeadsPerTile, (h + 1) * G - head0);

        // queries into LDS, rotated to the last position
        for (uint32_t e = t; e < Gn * (hd / 2); e += 256)
        {
            const uint32_t i = e / (hd / 2), w = e % (hd / 2);
            const uint32_t d0 = a.rope.style == 1 ? 2 * w : w, d1 = a.rope.style == 1 ? 2 * w + 1 : w + hd / 2;
            const T *q = (const T *)a.q.p + (size_t)b * a.q.s[1] + (size_t)(head0 + i) * a.q.s[2];
            const float x = (float)q[(size_t)d0 * a.q.s[3]], y = (float)q[(size_t)d1 * a.q.s[3]];
            float u = x, v = y;
            if (a.rope.style)
            {
                const float2 r = turn_at(len - 1, a.rope.turns[w]);
                u = r.x * x - r.y * y;
                v = r.y * x + r.x * y;
                if constexpr (F16)
                {
                    u *= 0.5f;
                    v *= 0.5f;
                    qs[(kHeadsPerTile + i) * QP + d0] = (T)(u - (float)(T)u);
                    qs[(kHeadsPerTile + i) * QP + d1] = (T)(v - (float)(T)v);
                }
            }
            qs[i * QP + d0] = (T)u;
            qs[i * QP + d1] = (T)v;
        }
        __syncthreads();
        u32x4 qf[QN][KS];
#pragma unroll
        for (int n = 0; n < QN; ++n)
#pragma unroll
            for (int s = 0; s < KS; ++s)
                qf[n][s] = c < Gn ? *(const u32x4 *)(qs + (n * kHeadsPerTile + c) * QP +
                                                     (F16 ? 8 * (g + 4 * s) : 16 * s + 4 * g))
                                  : (u32x4){0, 0, 0, 0};

        float m = kNegInf, l = 0.f;
        f32x4 o[VD];
#pragma unroll
        for (int d = 0; d < VD; ++d)
            o[d] = (f32x4){0.f, 0.f, 0.f, 0.f};
        const uint32_t *row = a.table.p + (size_t)b * a.table.stride + 1;
        uint32_t pid[NT]; // pages of the step after the one that is being loaded
        auto fetch = [&](uint32_t s) {
#pragma unroll
            for (int i = 0; i < NT; ++i)
            {
                const uint32_t key = s * KT + wave * KW + 16 * i;
                pid[i] = s < s1 && key < len ? row[key / R] : kNoPage;
            }
        };
        const T *rows[NT]; // the tiles' first key rows
        uint32_t live[NT]; // their keys
        auto place = [&](uint32_t s) {
#pragma unroll
            for (int i = 0; i < NT; ++i)
            {
                const uint32_t key = s * KT + wave * KW + 16 * i;
                const bool there = pid[i] < a.cache.n[0]; // absent pages: read page 0, use nothing of it
                live[i] = there ? min(16u, len - key) : 0u;
                rows[i] = (const T *)a.cache.p +
                          (there ? (size_t)pid[i] * a.cache.s[0] + (size_t)h * a.cache.s[1] + (size_t)(key % R) * hd : 0);
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
                    const uint32_t d = F16 ? 8 * (g + 4 * s) : 16 * s + 4 * g;
                    kr[i][s] = *(const u32x4 *)(rows[i] + c * hd + (d < hd ? d : 0));
                }
        };
        const T *vrows[NT];
        auto load_v = [&]() {
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                {
                    const T *p = vrows[i] + (4 * g + r) * hd;
                    uint32_t *to = vr[4 * i + r];
                    if constexpr (VW == 2)
                    {
                        const uint2 v = *(const uint2 *)(p + (4 * c < hd ? 4 * c : 0));
                        to[0] = v.x;
                        to[1] = v.y;
                    }
                    else
                    {
#pragma unroll
                        for (int w = 0; w < VW / 4; ++w)
                        {
                            const uint32_t d = VD * c + (F16 ? 8 : 4) * w;
                            const u32x4 v = *(const u32x4 *)(p + (d < hd ? d : 0));
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                to[4 * w + k] = v[k];
                        }
                    }
                }
        };
        auto point_v = [&]() {
#pragma unroll
            for (int i = 0; i < NT; ++i)
                vrows[i] = rows[i] + (size_t)KV * a.cache.s[1];
        };
        fetch(s0);
        place(s0);
        load_k();
        point_v();
        load_v();
        fetch(s0 + 1);
        for (uint32_t s = s0; s < s1; ++s)
        {
            f32x4 x[NT];
#pragma unroll
            for (int i = 0; i < NT; ++i)
            {
                x[i] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < KS; ++k)
                {
                    u32x4 kv = kr[i][k];
                    if (hd != HDP && (F16 ? 8 * (g + 4 * k) : 16 * k + 4 * g) >= hd)
                        kv = (u32x4){0, 0, 0, 0};
                    if constexpr (F16)
                    {
                        x[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                            __builtin_bit_cast(half8, kv), __builtin_bit_cast(half8, qf[0][k]), x[i], 0, 0, 0);
                        if (a.rope.style)
                            x[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                                __builtin_bit_cast(half8, kv), __builtin_bit_cast(half8, qf[1][k]), x[i], 0, 0, 0);
                    }
                    else
                    {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            x[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kv[e]),
                                                                        __uint_as_float(qf[0][k][e]), x[i], 0, 0, 0);
                    }
                }
            }
            uint32_t n[NT];
#pragma unroll
            for (int i = 0; i < NT; ++i)
                n[i] = live[i];
            const bool more = s + 1 < s1;
            if (more)
            {
                place(s + 1);
                load_k();
                fetch(s + 2);
            }
            bool whole = true;
#pragma unroll
            for (int i = 0; i < NT; ++i)
                whole = whole && n[i] == 16;
            float top = kNegInf;
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                {
                    x[i][r] *= a.scale_log2;
                    if (!whole && 4 * g + r >= n[i])
                        x[i][r] = kNegInf;
                    top = fmaxf(top, x[i][r]);
                }
            // m rises when a score passes it by 7: probabilities then stay below 2^15 at the 2^8 that fp16 ones are scaled
            // by, and those down to 2^-32 of the largest still count
            if (__any(top > m + 7.f))
            {
                top = fmaxf(top, __shfl_xor(top, 16, kWave));
                top = fmaxf(top, __shfl_xor(top, 32, kWave));
                const float next = fmaxf(m, top), f = m == kNegInf ? 0.f : exp2_of(m - next);
                m = next;
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
#pragma unroll
                for (int d = 0; d < VD; ++d)
                {
                    u32x4 v; // 8 keys of dim VD * c + d
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        v[j] = __builtin_amdgcn_perm(vr[2 * j + 1][d / 2], vr[2 * j][d / 2],
                                                     d % 2 ? 0x07060302u : 0x05040100u);
                    o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, v), p, o[d], 0, 0, 0);
                    o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, v), q, o[d], 0, 0, 0);
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
            if (more)
            {
                point_v();
                load_v();
            }
        }

        // the four waves' sums
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
                    if (VD * (4 * g + i) + d < hd)
                        to[VD * (4 * g + i) + d] = o[d][i];
        }
        __syncthreads();
        const bool all = s0 == 0 && s1 == n_units;
        float *part = a.parts + (2 * (size_t)blockIdx.x + (u == u0 ? 0 : 1)) * part_floats(a.tile_heads, hd);
        for (uint32_t e = t; e < Gn * hd; e += 256)
        {
            const uint32_t i = e / hd, d = e % hd;
            float mw[4], top = kNegInf, lsum = 0.f, osum = 0.f;
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
                lsum += f * ml[(w * kHeadsPerTile + i) * 2 + 1];
                osum += f * sums[(size_t)(w * a.tile_heads + i) * hd + d];
            }
            if (all)
                ((T *)a.out.p)[(size_t)b * a.out.s[1] + (size_t)(head0 + i) * a.out.s[2] + (size_t)d * a.out.s[3]] =
                    (T)(lsum == 0.f ? 0.f : osum / lsum);
            else
            {
                part[2 * a.tile_heads + i * hd + d] = osum;
                if (d == 0)
                {
                    part[i] = top;
                    part[a.tile_heads + i] = lsum;
                }
            }
        }
        // the workgroup with the first units of a row that goes on has it joined
        if (!all && s0 == 0 && t == 0)
        {
            const uint64_t last = base + (uint64_t)hg * n_units + n_units - 1;
            a.joins[blockIdx.x * 4] = (uint32_t)(last / share) - blockIdx.x + 1;
            a.joins[blockIdx.x * 4 + 1] = b;
            a.joins[blockIdx.x * 4 + 2] = hg;
            a.joins[blockIdx.x * 4 + 3] = u == u0 ? 0 : 1;
        }
        u += s1 - s0;
    }
}

// Joins the partial results of the row that begins in workgroup x of the kernel above and goes on in those after it (its
// first part in slot joins[3], the others in slot 0); workgroup (x, i) has query head i of the tile.
template <bool F16> __global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnArgs a)
{
    using T = typename std::conditional<F16, _Float16, float>::type;
    __shared__ float sums[4][kPagedMaxHd];
    const uint32_t *join = a.joins + blockIdx.x * 4;
    const uint32_t n = join[0], i = blockIdx.y;
    if (n == 0)
        return;
    const uint32_t b = join[1], hg = join[2], slot = join[3];
    const uint32_t KV = a.cache.n[1] / 2, hd = a.cache.n[3], G = a.q.n[2] / KV, h = hg / a.groups;
    const uint32_t head = h * G + hg % a.groups * kHeadsPerTile + i;
    if (head >= (h + 1) * G)
        return;
    const uint32_t t = threadIdx.x, lane = t % kWave, wave = t / kWave;
    const size_t floats = part_floats(a.tile_heads, hd);
    auto part = [&](uint32_t k) { return a.parts + (2 * (size_t)(blockIdx.x + k) + (k == 0 ? slot : 0)) * floats; };
    float top = kNegInf;
    for (uint32_t k = lane; k < n; k += kWave)
        top = fmaxf(top, part(k)[i]);
    top = wave_max(top);
    float lsum = 0.f;
    for (uint32_t k = lane; k < n; k += kWave)
    {
        const float mk = part(k)[i];
        lsum += mk == kNegInf ? 0.f : exp2_of(mk - top) * part(k)[a.tile_heads + i];
    }
    lsum = wave_sum(lsum);
    float o[kPagedMaxHd / kWave] = {};
#pragma unroll 4
    for (uint32_t k = wave; k < n; k += 4)
    {
        const float *p = part(k);
        const float f = p[i] == kNegInf ? 0.f : exp2_of(p[i] - top);
#pragma unroll
        for (int j = 0; j < kPagedMaxHd / kWave; ++j)
            if (lane + j * kWave < hd)
                o[j] += f * p[2 * a.tile_heads + i * hd + lane + j * kWave];
    }
#pragma unroll
    for (int j = 0; j < kPagedMaxHd / kWave; ++j)
        if (lane + j * kWave < hd)
            sums[wave][lane + j * kWave] = o[j];
    __syncthreads();
    if (t < hd)
    {
        const float osum = (sums[0][t] + sums[1][t]) + (sums[2][t] + sums[3][t]);
        ((T *)a.out.p)[(size_t)b * a.out.s[1] + (size_t)head * a.out.s[2] + (size_t)t * a.out.s[3]] =
            (T)(lsum == 0.f ? 0.f : osum / lsum);
    }
}

template <bool F16, int HDP>
static hipError_t launch_as(hipStream_t st, PagedAttnArgs &a, float *work, size_t work_elems, int cu_count)
{
    using Tile = PagedTile<F16, HDP>;
    const void *fn = (const void *)paged_attn_kernel<F16, HDP>;
    const uint32_t hd = a.cache.n[3];
    const size_t lds = (size_t)(a.table.B + 3) / 4 * 16 + Tile::QN * kHeadsPerTile * Tile::QP * (F16 ? 2 : 4) +
                       4 * kHeadsPerTile * 8 + (size_t)4 * a.tile_heads * hd * 4;
    static uint64_t done = 0, memo = 0;
    const hipError_t e = lds_attr_once(fn, 128 << 10, done);
    if (e != hipSuccess)
        return e;
    const int per_cu = occupancy_per_cu(fn, 256, lds, memo);
    if (per_cu <= 0)
        return hipErrorLaunchFailure;
    const size_t each = 4 + 2 * part_floats(a.tile_heads, hd); // words of the workspace per workgroup
    const uint32_t grid = (uint32_t)std::min<size_t>((size_t)per_cu * cu_count, work_elems / each);
    if (grid == 0)
        return hipErrorOutOfMemory;
    a.joins = (uint32_t *)work;
    a.parts = work + 4 * (size_t)grid;
    paged_attn_kernel<F16, HDP><<<grid, 256, lds, st>>>(a);
    paged_join_kernel<F16><<<dim3(grid, a.tile_heads), 256, 0, st>>>(a);
    return hipGetLastError();
}

hipError_t launch_paged_attn(hipStream_t st, const TView &q, const TView &cache, const PageTableView &table,
                             const TView &out, float scale, const PagedRope &rope, float *work, size_t work_elems,
                             int cu_count)
{
    const uint32_t G = q.n[2] / (cache.n[1] / 2), hd = q.n[3];
    const float half = cache.dt == DT_F16 && rope.style ? 2.f : 1.f; // the kernel halves rotated fp16 queries
    PagedAttnArgs a{q, cache, out, table, half * scale * 1.44269504088896340736f, (G - 1) / kHeadsPerTile + 1,
                    std::min(G, (uint32_t)kHeadsPerTile), nullptr, nullptr, rope};
    if (cache.dt == DT_F16)
        return hd <= 64    ? launch_as<true, 64>(st, a, work, work_elems, cu_count)
               : hd <= 128 ? launch_as<true, 128>(st, a, work, work_elems, cu_count)
                           : launch_as<true, 256>(st, a, work, work_elems, cu_count);
    return hd <= 64    ? launch_as<false, 64>(st, a, work, work_elems, cu_count)
           : hd <= 128 ? launch_as<false, 128>(st, a, work, work_elems, cu_count)
                       : launch_as<false, 256>(st, a, work, work_elems, cu_count);
}

} // namespace vk
