// Attention of few rows over a paged cache, and the join of partial results.
//
// o = sum_j 2^(s_j - m) v_j / l, s_j = scale * log2(e) * q . k_j, for few rows of a key head (a row is one new token and one of the query heads
// that read this key head): single tokens and drafts.  Bound by reading the cache once.  A warp takes 16 positions at a time, on its own:
//   S^T = K.Q^T by m16n8k16 products.  The sum over a head's numbers may run in any order, so the lanes load 16-byte pieces of the keys straight
//   into the operand's registers, and the queries lie in shared memory in the order that this gives.
//   O^T = V^T.P^T.  The rows of O^T may stand in any order too: lane (g, t) loads the g-th eighth of the values of its four positions, and pairs
//   of neighbouring positions make the operand.  The weights, which come out position by row, are transposed by movmatrix.
// So nothing of the cache goes through shared memory, and no warp waits for another until the end, where their sums are joined.  Long ranges are
// cut over the CTAs and joined by paged_join_kernel, in the order of the parts.
// Measured: single tokens of 64 sequences of 1000 to 8000 positions, 8 key heads of 128, bf16, 188 us with the join: 1.25 GB at 6.6 TB/s, what a copy
// moves.  One sequence of 16001 positions, 4 key heads of 64, f32: 15 us for 33 MB, where starting, the first loads and the join are most of it.
// (Two CTAs of four warps an SM with up to 255 registers: the loads of a whole step are in flight while the one before is worked on.  Three or four CTAs with fewer
// registers: 191 to 417 us.)
//
// 32 bits: a number is the sum of three bf16 numbers (each the rounded rest of the ones before; what is left is below 2^-24 of it); the six largest
// of the nine products are computed, the largest apart from the others, and a step's results are added in f32 registers.
#include <type_traits>

#include "mma_common.cuh"
#include "paged.cuh"
#include "paged_tc.cuh"

namespace lumen {
namespace {

using tc::ex2;
using tc::kLog2e;
using tc::pack_bf16;
using tc::split3;

constexpr int kWarps = 4, kBlocksPerSm = 2;

template <typename T, int D, int NB>
struct FewGeom {
    static constexpr bool kSplit = sizeof(T) == 4;
    static constexpr int kTerms = kSplit ? 3 : 1;
    static constexpr int kPieces = D * (int)sizeof(T) / 64;       // 16-byte pieces of a key, per lane
    static constexpr int kG = 512 / (D * (int)sizeof(T));         // groups of 16 positions in a step: 256 bytes of keys and of values a lane in flight
    static constexpr int kStep = 16 * kG;
    static constexpr int kTiles = D / 16;                         // of 16 numbers
    static constexpr int kQ = NB * kTiles * 32 * 8 * kTerms;      // bytes: queries in the order of the operand, 8 a lane, tile and term
    static constexpr int kSums = kWarps * NB * 8 * (D + 4) * 4;   // every warp's sums at the end, over the queries
    static constexpr int kSmem = kQ > kSums ? kQ : kSums;
};

template <typename T, int D, int NB>
__global__ void __launch_bounds__(kWarps * 32, kBlocksPerSm) paged_few_kernel(const PagedView p, const PagedAttnArgs a) {
    using G = FewGeom<T, D, NB>;
    constexpr bool kSplit = G::kSplit;
    constexpr int kG = G::kG, kPieces = G::kPieces, kTiles = G::kTiles, kTerms = G::kTerms;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ float m_s[kWarps][NB * 8], l_s[kWarps][NB * 8];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const PagedItem it = a.items[blockIdx.x];
    const PagedSeq sq = it.sq;
    const int *table = p.tables + sq.table;
    const int past = sq.kv_len - sq.q_len;
    const float scale2 = a.scale * kLog2e;
    const int steps = (it.key1 - it.key0 + G::kStep - 1) / G::kStep;

    // rows of the pool of every 8 positions of step i: their page, or -1 behind the end
    auto pages = [&](int i, int (&page)[2 * kG]) {
#pragma unroll
        for (int b = 0; b < 2 * kG; ++b) {
            const int pos = it.key0 + i * G::kStep + 8 * b;
            page[b] = i < steps && pos < it.key1 ? table[pos >> p.page_shift] : -1;
        }
    };
    auto row8 = [&](int i, int b, int page) {  // row of the first of 8 positions
        return (((size_t)page * p.h_kv + it.kvh) << p.page_shift) + ((it.key0 + i * G::kStep + 8 * b) & ((1 << p.page_shift) - 1));
    };
    uint4 k[kG][2][kPieces], v[kG][4][kPieces / 2];  // keys g and g + 8; positions 2t, 2t + 1, 2t + 8, 2t + 9
    static_assert(kPieces % 2 == 0, "an eighth of a row is whole pieces");
    auto load_k = [&](int i, const int (&page)[2 * kG]) {
#pragma unroll
        for (int x = 0; x < kG; ++x)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int pg = page[2 * x + h];
                const uint4 *src = reinterpret_cast<const uint4 *>(static_cast<const T *>(p.k) + (row8(i, 2 * x + h, max(pg, 0)) + g) * D);
#pragma unroll
                for (int c = 0; c < kPieces; ++c) k[x][h][c] = pg >= 0 ? __ldcs(src + 4 * c + t) : make_uint4(0u, 0u, 0u, 0u);
            }
    };
    auto load_v = [&](int i, const int (&page)[2 * kG]) {
#pragma unroll
        for (int x = 0; x < kG; ++x)
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const int b = 2 * x + (y >> 1), in8 = 2 * t + (y & 1), pg = page[b];
                const bool live = pg >= 0 && it.key0 + i * G::kStep + 8 * b + in8 < it.key1;  // (behind the end: zeros, which meet weights of zero)
                const uint4 *src = reinterpret_cast<const uint4 *>(static_cast<const T *>(p.v) + (row8(i, b, max(pg, 0)) + in8) * D) + g * (kPieces / 2);
#pragma unroll
                for (int c = 0; c < kPieces / 2; ++c) v[x][y][c] = live ? __ldcs(src + c) : make_uint4(0u, 0u, 0u, 0u);
            }
    };
    int page[2 * kG];
    pages(warp, page);
    pdl_launch();
    pdl_wait();
    load_k(warp, page);
    load_v(warp, page);

    // queries: row 8 b + g of block b is column g of the operand; lane t has the numbers that its pieces of the keys have
    for (int i = tid; i < NB * kTiles * 32; i += kWarps * 32) {
        const int ln = i & 31, tile = i / 32 % kTiles, row = i / (32 * kTiles) * 8 + (ln >> 2);
        // 32 bits: tile c takes piece c, numbers 16 c + 4 t ..; 16 bits: tiles 2 c and 2 c + 1 the halves of piece c, numbers 32 c + 8 t ..
        const int at = kSplit ? 16 * tile + 4 * (ln & 3) : 32 * (tile / 2) + 8 * (ln & 3) + 4 * (tile & 1);
        const int r = it.row0 + row;
        const T *src = static_cast<const T *>(a.q) + ((size_t)(sq.tok0 + r / p.group) * p.n_head + it.kvh * p.group + r % p.group) * D + at;
        uint2 *dst = reinterpret_cast<uint2 *>(smem) + (size_t)i * kTerms;
        if constexpr (kSplit) {
            const float4 x = row < it.rows ? *reinterpret_cast<const float4 *>(src) : make_float4(0.f, 0.f, 0.f, 0.f);
            uint32_t lo[3], hi[3];
            split3(x.x, x.y, lo);
            split3(x.z, x.w, hi);
#pragma unroll
            for (int n = 0; n < 3; ++n) dst[n] = make_uint2(lo[n], hi[n]);
        } else {
            *dst = row < it.rows ? *reinterpret_cast<const uint2 *>(src) : make_uint2(0u, 0u);
        }
    }
    float o[NB][kTiles][4], m[NB][2], l[NB][2];
    int last[NB][2];  // the last position that the rows 8 b + 2 t + e see
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            m[b][e] = -INFINITY;
            l[b][e] = 0.f;
            const int r = 8 * b + 2 * t + e;
            last[b][e] = r >= it.rows ? -1 : p.causal ? min(it.key1 - 1, past + (it.row0 + r) / p.group) : it.key1 - 1;
        }
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int d = 0; d < kTiles; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[b][d][e] = 0.f;
    __syncthreads();
    const uint2 *q_s = reinterpret_cast<const uint2 *>(smem);

#pragma unroll 1
    for (int i = warp; i < steps; i += kWarps) {
        int next[2 * kG];
        pages(i + kWarps, next);
        float s[kG][NB][4];
#pragma unroll
        for (int x = 0; x < kG; ++x)
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                float sums[4][4] = {};  // (of their own, so that products do not wait for each other; the last the largest)
#pragma unroll
                for (int c = 0; c < kTiles; ++c) {
                    const uint2 *qf = q_s + (size_t)((b * kTiles + c) * 32 + lane) * kTerms;
                    if constexpr (kSplit) {
                        const uint4 k0 = k[x][0][c], k1 = k[x][1][c];
                        uint32_t a0[3], a1[3], a2[3], a3[3];
                        split3(__uint_as_float(k0.x), __uint_as_float(k0.y), a0);
                        split3(__uint_as_float(k1.x), __uint_as_float(k1.y), a1);
                        split3(__uint_as_float(k0.z), __uint_as_float(k0.w), a2);
                        split3(__uint_as_float(k1.z), __uint_as_float(k1.w), a3);
                        const uint2 q0 = qf[0], q1 = qf[1], q2 = qf[2];
                        const uint32_t h[4] = {a0[0], a1[0], a2[0], a3[0]}, md[4] = {a0[1], a1[1], a2[1], a3[1]}, lw[4] = {a0[2], a1[2], a2[2], a3[2]};
                        mma16816(sums[0], lw, q0.x, q0.y);
                        mma16816(sums[1], md, q1.x, q1.y);
                        mma16816(sums[2], h, q1.x, q1.y);
                        mma16816(sums[3], h, q0.x, q0.y);
                        mma16816(sums[0], h, q2.x, q2.y);
                        mma16816(sums[1], md, q0.x, q0.y);
                    } else {
                        const uint4 k0 = k[x][0][c / 2], k1 = k[x][1][c / 2];
                        const uint32_t h[4] = {c & 1 ? k0.z : k0.x, c & 1 ? k1.z : k1.x, c & 1 ? k0.w : k0.y, c & 1 ? k1.w : k1.y};
                        mma16816(sums[c & 3], h, qf->x, qf->y);
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) s[x][b][e] = sums[3][e] + (sums[2][e] + (sums[1][e] + sums[0][e]));
            }
        load_k(i + kWarps, next);
        // weights: lane (g, t) has positions g, g + 8 of the rows 2t, 2t + 1
        const int first = it.key0 + i * G::kStep;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            float f[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float top = -INFINITY;
#pragma unroll
                for (int x = 0; x < kG; ++x)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float &z = s[x][b][2 * h + e];
                        z = first + 16 * x + 8 * h + g <= last[b][e] ? z * scale2 : -INFINITY;
                        top = fmaxf(top, z);
                    }
#pragma unroll
                for (int w = 4; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
                const float now = fmaxf(m[b][e], top), base = now == -INFINITY ? 0.f : now;
                f[e] = ex2(m[b][e] - base);
                m[b][e] = now;
                l[b][e] *= f[e];
#pragma unroll
                for (int x = 0; x < kG; ++x)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float &z = s[x][b][2 * h + e];
                        z = ex2(z - base);
                        l[b][e] += z;
                    }
            }
            if (__any_sync(0xffffffffu, f[0] != 1.f || f[1] != 1.f))
#pragma unroll
                for (int d = 0; d < kTiles; ++d)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[b][d][e] *= f[e & 1];
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            uint32_t w[kG][kTerms][2];  // the weights' terms as the second operand: rows of this block x positions
#pragma unroll
            for (int x = 0; x < kG; ++x)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if constexpr (kSplit) {
                        uint32_t t3[3];
                        split3(s[x][b][2 * h], s[x][b][2 * h + 1], t3);
#pragma unroll
                        for (int n = 0; n < 3; ++n) w[x][n][h] = transpose8x8(t3[n]);
                    } else {
                        w[x][0][h] = transpose8x8(pack_bf16(s[x][b][2 * h], s[x][b][2 * h + 1]));
                    }
                }
#pragma unroll
            for (int d = 0; d < kTiles; ++d) {
                if constexpr (kSplit) {
                    float big[4] = {0.f, 0.f, 0.f, 0.f}, small[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int x = 0; x < kG; ++x) {
                        float n0[4], n1[4];  // numbers 2 d and 2 d + 1 of the lane's eighth, of its four positions
#pragma unroll
                        for (int y = 0; y < 4; ++y) {
                            const uint4 z = v[x][y][d / 2];
                            n0[y] = __uint_as_float(d & 1 ? z.z : z.x);
                            n1[y] = __uint_as_float(d & 1 ? z.w : z.y);
                        }
                        uint32_t a0[3], a1[3], a2[3], a3[3];
                        split3(n0[0], n0[1], a0);
                        split3(n1[0], n1[1], a1);
                        split3(n0[2], n0[3], a2);
                        split3(n1[2], n1[3], a3);
                        const uint32_t h[4] = {a0[0], a1[0], a2[0], a3[0]}, md[4] = {a0[1], a1[1], a2[1], a3[1]}, lw[4] = {a0[2], a1[2], a2[2], a3[2]};
                        mma16816(small, lw, w[x][0][0], w[x][0][1]);
                        mma16816(small, h, w[x][2][0], w[x][2][1]);
                        mma16816(small, md, w[x][1][0], w[x][1][1]);
                        mma16816(small, md, w[x][0][0], w[x][0][1]);
                        mma16816(small, h, w[x][1][0], w[x][1][1]);
                        mma16816(big, h, w[x][0][0], w[x][0][1]);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[b][d][e] += big[e] + small[e];
                } else {
#pragma unroll
                    for (int x = 0; x < kG; ++x) {
                        uint32_t n[4];
#pragma unroll
                        for (int y = 0; y < 4; ++y) {
                            const uint4 z = v[x][y][d / 4];
                            n[y] = d % 4 == 0 ? z.x : d % 4 == 1 ? z.y : d % 4 == 2 ? z.z : z.w;
                        }
                        const uint32_t h[4] = {__byte_perm(n[0], n[1], 0x5410), __byte_perm(n[0], n[1], 0x7632), __byte_perm(n[2], n[3], 0x5410), __byte_perm(n[2], n[3], 0x7632)};
                        mma16816(o[b][d], h, w[x][0][0], w[x][0][1]);
                    }
                }
            }
        }
        load_v(i + kWarps, next);
    }

    // the warps' sums, in their order
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) l[b][e] += __shfl_xor_sync(0xffffffffu, l[b][e], w);
            if (g == 0) {
                m_s[warp][8 * b + 2 * t + e] = m[b][e];
                l_s[warp][8 * b + 2 * t + e] = l[b][e];
            }
        }
    __syncthreads();  // (and every warp is done with the queries)
    float *o_s = reinterpret_cast<float *>(smem);  // [warp][row][D + 4]
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int d = 0; d < kTiles; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) o_s[(size_t)((warp * NB + b) * 8 + 2 * t + (e & 1)) * (D + 4) + g * (D / 8) + 2 * d + (e >> 1)] = o[b][d][e];
    __syncthreads();
    for (int i = tid; i < it.rows * (D / 4); i += kWarps * 32) {
        const int row = i / (D / 4), c = i % (D / 4) * 4;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, m_s[w][row]);
        const float base = top == -INFINITY ? 0.f : top;
        float x[4] = {0.f, 0.f, 0.f, 0.f}, sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float f = ex2(m_s[w][row] - base);
            const float4 y = *reinterpret_cast<const float4 *>(o_s + (size_t)(w * NB * 8 + row) * (D + 4) + c);
            sum = fmaf(l_s[w][row], f, sum);
            x[0] = fmaf(y.x, f, x[0]);
            x[1] = fmaf(y.y, f, x[1]);
            x[2] = fmaf(y.z, f, x[2]);
            x[3] = fmaf(y.w, f, x[3]);
        }
        if (it.part >= 0) {
            const size_t r = (size_t)it.part + row;
            *reinterpret_cast<float4 *>(a.part + r * D + c) = make_float4(x[0], x[1], x[2], x[3]);
            if (c == 0) *reinterpret_cast<float2 *>(a.part + (size_t)a.part_rows * D + 2 * r) = make_float2(top, sum);
            continue;
        }
        const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
        const size_t r = (size_t)(sq.tok0 + (it.row0 + row) / p.group) * p.n_head + it.kvh * p.group + (it.row0 + row) % p.group;
        if (kSplit || a.out_dtype == LUMEN_F32) *reinterpret_cast<float4 *>(static_cast<float *>(a.out) + r * D + c) = make_float4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
        else *reinterpret_cast<uint2 *>(static_cast<__nv_bfloat16 *>(a.out) + r * D + c) = make_uint2(pack_bf16(x[0] * inv, x[1] * inv), pack_bf16(x[2] * inv, x[3] * inv));
        if (c == 0 && a.lse) a.lse[r] = top * 0.6931471805599453f + logf(sum);
    }
}

// Joins the parts of a row, in their order: a warp a row, or (WIDE) eight warps a row whose sums meet in shared memory.
// grid (joins, rows or groups of eight rows)
constexpr int kJoinWarps = 8;
template <int D, bool WIDE>
__global__ void __launch_bounds__(kJoinWarps * 32) paged_join_kernel(const PagedView p, const PagedAttnArgs a) {
    constexpr int E = D / 32;
    using V = typename std::conditional<E == 4, float4, float2>::type;
    __shared__ float o_s[WIDE ? kJoinWarps : 1][D], l_s[kJoinWarps];
    const PagedJoin j = a.joins[blockIdx.x];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = WIDE ? (int)blockIdx.y : (int)(blockIdx.y * kJoinWarps) + warp;
    pdl_launch();
    pdl_wait();
    if (r >= j.rows) return;
    const float2 *ml = reinterpret_cast<const float2 *>(a.part + (size_t)a.part_rows * D);
    float top = -INFINITY;
    for (int i = lane; i < j.splits; i += 32) top = fmaxf(top, ml[(size_t)j.part + (size_t)i * j.rows + r].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float base = top == -INFINITY ? 0.f : top;
    float v[E], l = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = 0.f;
#pragma unroll 8
    for (int i = WIDE ? warp : 0; i < j.splits; i += WIDE ? kJoinWarps : 1) {
        const size_t row = (size_t)j.part + (size_t)i * j.rows + r;
        const float2 x = ml[row];
        float y[E];
        *reinterpret_cast<V *>(y) = *reinterpret_cast<const V *>(a.part + row * D + lane * E);
        const float f = ex2(x.x - base);
        l = fmaf(x.y, f, l);
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = fmaf(y[e], f, v[e]);
    }
    if (WIDE) {
        *reinterpret_cast<V *>(&o_s[warp][lane * E]) = *reinterpret_cast<const V *>(v);
        if (lane == 0) l_s[warp] = l;
        __syncthreads();
        if (warp > 0) return;
#pragma unroll
        for (int w = 1; w < kJoinWarps; ++w) {
            l += l_s[w];
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] += o_s[w][lane * E + e];
        }
    }
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    const size_t o = (size_t)(j.tok0 + (j.row0 + r) / p.group) * p.n_head + j.kvh * p.group + (j.row0 + r) % p.group;
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] *= inv;
    if (a.out_dtype == LUMEN_F32) {
        *reinterpret_cast<V *>(static_cast<float *>(a.out) + o * D + lane * E) = *reinterpret_cast<const V *>(v);
    } else {
#pragma unroll
        for (int e = 0; e < E; e += 2) *reinterpret_cast<uint32_t *>(static_cast<__nv_bfloat16 *>(a.out) + o * D + lane * E + e) = pack_bf16(v[e], v[e + 1]);
    }
    if (lane == 0 && a.lse) a.lse[o] = top * 0.6931471805599453f + logf(l);
}

template <typename T, int D, int NB>
int launch(lumen_ctx *ctx, const PagedView &v, const PagedAttnArgs &a, cudaStream_t s) {
    constexpr size_t bytes = FewGeom<T, D, NB>::kSmem;
    LUMEN_TRY(allow_smem(ctx, paged_few_kernel<T, D, NB>, bytes));
    return launch_paged(ctx, paged_few_kernel<T, D, NB>, dim3((unsigned)a.n_items), kWarps * 32, bytes, s, v, a);
}
template <typename T, int D>
int pick(lumen_ctx *ctx, const PagedView &v, const PagedAttnArgs &a, cudaStream_t s) {
    return a.max_rows <= 8 ? launch<T, D, 1>(ctx, v, a, s) : launch<T, D, 2>(ctx, v, a, s);
}

}  // namespace

// Rows of a sequence and key head up to which this kernel is taken; by events, here and with tensor-core tiles.  8 sequences of 2000 to 8000 positions, 8 key
// heads of 128: 16 bits, 12 rows 47 and 46 us, 16 rows 48 and 48 (32 key heads, 2000 positions: 62 and 67; 20 rows, in blocks of 32: 101 and 61); 32 bits, 32 rows
// (16 at a time) 182 and 188 us.
int paged_few_rows(const PagedGeom &g) { return g.dtype == LUMEN_F32 ? 32 : 16; }

PagedShape paged_few_shape(int num_sms) { return {16, 64, num_sms * kBlocksPerSm}; }

int launch_paged_few(lumen_ctx *ctx, const PagedGeom &g, const PagedView &v, const PagedAttnArgs &a, cudaStream_t s) {
    if (g.dtype == LUMEN_F32) return g.d == 64 ? pick<float, 64>(ctx, v, a, s) : pick<float, 128>(ctx, v, a, s);
    return g.d == 64 ? pick<__nv_bfloat16, 64>(ctx, v, a, s) : pick<__nv_bfloat16, 128>(ctx, v, a, s);
}

int launch_paged_join(lumen_ctx *ctx, const PagedGeom &g, const PagedView &v, const PagedAttnArgs &a, cudaStream_t s) {
    // Many parts of few rows: a row's are read by eight warps (one after another they would wait for each other's latency).
    const bool wide = a.join_splits > 8;
    const dim3 grid((unsigned)a.n_joins, wide ? (unsigned)a.join_rows : ((unsigned)a.join_rows + kJoinWarps - 1) / kJoinWarps);
    auto *kernel = g.d == 64 ? (wide ? paged_join_kernel<64, true> : paged_join_kernel<64, false>) : (wide ? paged_join_kernel<128, true> : paged_join_kernel<128, false>);
    return launch_paged(ctx, kernel, grid, kJoinWarps * 32, 0, s, v, a);
}

}  // namespace lumen
