// Attention of few rows over a paged cache of 32 bits, in 32-bit arithmetic, and the join of partial results.
//
// o = sum_j 2^(s_j - m) v_j / l with s_j = scale * log2(e) * q . k_j, the running maximum m and sum l = sum_j 2^(s_j - m) of every row (a row
// is one new token and one of the query heads of a key head).  A CTA takes an item: up to RT rows of one key head against a range of
// positions, so every key and value is read once for the whole group; long ranges are cut over the CTAs and joined by
// paged_join_kernel, in the order of the parts.
//
// Tiles of kKeys positions come by 16-byte asynchronous copies (the page of every position is looked up), two tiles deep.  A thread computes
// the scores of one key for half of the rows (keys from padded rows of shared memory without bank conflicts, queries broadcast), the
// softmax of a row is shared by 128 / RT threads, and for P.V a warp takes a quarter of the keys and all numbers of a head.
#include <type_traits>

#include "paged.cuh"

namespace lumen {
namespace {

constexpr int kKeys = 64, kThreads = 128;

__device__ __forceinline__ void cp16(void *dst, const void *src, bool live) {
    const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(src), "r"(live ? 16 : 0) : "memory");
}

__device__ __forceinline__ float ex2f(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// four numbers of a row
__device__ __forceinline__ void four(const float *p, float (&v)[4]) {
    const float4 x = *reinterpret_cast<const float4 *>(p);
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
}
template <int D, int RT>
struct RowsSmem {
    static constexpr int kRow = D * 4 + 16;  // bytes between rows of a tile: 8 rows at one column lie in 8 different groups of banks
    static constexpr int kTile = kKeys * kRow;
    static constexpr int kQ = 4 * kTile;                       // f32 queries [RT][D]
    static constexpr int kS = kQ + RT * D * 4;                 // scores [RT][kKeys + 1]
    static constexpr int kP = kS + (RT * (kKeys + 1) * 4 + 15) / 16 * 16;  // weights [kKeys][RT]
    static constexpr int kF = kP + kKeys * RT * 4;             // factor, maximum, sum of every row
    static constexpr int kRowOff = kF + 3 * RT * 4;            // where the tile's positions are: [2][kKeys]
    static constexpr int kBytes = kRowOff + 2 * kKeys * 8;
};

template <int D, int RT>
__global__ void __launch_bounds__(kThreads) paged_rows_kernel(const PagedView p, const PagedAttnArgs a) {
    using G = RowsSmem<D, RT>;
    constexpr int kParts = D * 4 / 16;  // 16-byte pieces of a row
    extern __shared__ __align__(16) unsigned char smem[];
    float *q_s = reinterpret_cast<float *>(smem + G::kQ), *s_s = reinterpret_cast<float *>(smem + G::kS), *p_s = reinterpret_cast<float *>(smem + G::kP);
    float *fac = reinterpret_cast<float *>(smem + G::kF), *mx = fac + RT, *sum = mx + RT;
    long long *at_s = reinterpret_cast<long long *>(smem + G::kRowOff);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const PagedItem it = a.items[blockIdx.x];
    const PagedSeq sq = p.seqs[it.seq];
    const int *table = p.tables + sq.table;
    const int past = sq.kv_len - sq.q_len;
    const float scale2 = a.scale * 1.4426950408889634f;
    auto token = [&](int r) { return sq.tok0 + (it.row0 + r) / p.group; };
    auto head = [&](int r) { return it.kvh * p.group + (it.row0 + r) % p.group; };
    auto last_seen = [&](int r) { return p.causal ? past + (it.row0 + r) / p.group : sq.kv_len - 1; };

    for (int i = tid; i < RT * (D / 4); i += kThreads) {
        const int r = i / (D / 4), e = i % (D / 4) * 4;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        if (r < it.rows) four(static_cast<const float *>(a.q) + ((size_t)token(r) * p.n_head + head(r)) * D + e, v);
        *reinterpret_cast<float4 *>(q_s + r * D + e) = make_float4(v[0], v[1], v[2], v[3]);
    }
    if (tid < RT) mx[tid] = -INFINITY, sum[tid] = 0.f;

    const int tiles = (it.key1 - it.key0 + kKeys - 1) / kKeys;
    auto locate = [&](int j) {
        const int pos = it.key0 + j * kKeys + tid;
        if (tid < kKeys) at_s[(j & 1) * kKeys + tid] = pos < it.key1 ? (long long)paged_row(p, table, it.kvh, pos) : -1;
    };
    auto fetch = [&](int j) {
        unsigned char *kt = smem + (j & 1) * 2 * G::kTile, *vt = kt + G::kTile;
        for (int i = tid; i < kKeys * kParts; i += kThreads) {
            const int r = i / kParts, c = i % kParts * 16;
            const long long at = at_s[(j & 1) * kKeys + r];
            const size_t off = at < 0 ? 0 : (size_t)at * D * 4 + c;
            cp16(kt + r * G::kRow + c, static_cast<const char *>(p.k) + off, at >= 0);  // (behind the end: zeros)
            cp16(vt + r * G::kRow + c, static_cast<const char *>(p.v) + off, at >= 0);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    constexpr int E = D / 32;
    float acc[RT][E];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int e = 0; e < E; ++e) acc[r][e] = 0.f;
    if (tiles > 0) {
        locate(0);
        __syncthreads();
        fetch(0);
    }
#pragma unroll 1
    for (int j = 0; j < tiles; ++j) {
        if (j + 1 < tiles) locate(j + 1);
        __syncthreads();  // positions of the next tile; everyone is done with the tile before this one
        if (j + 1 < tiles) {
            fetch(j + 1);
            asm volatile("cp.async.wait_group 1;" ::: "memory");
        } else {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        }
        __syncthreads();
        const unsigned char *kt = smem + (j & 1) * 2 * G::kTile, *vt = kt + G::kTile;
        const int first = it.key0 + j * kKeys;
        {  // scores: one key, half of the rows
            constexpr int RH = RT / 2;
            const int key = tid % kKeys, r0 = tid / kKeys * RH;
            float s[RH];
#pragma unroll
            for (int r = 0; r < RH; ++r) s[r] = 0.f;
            const float *kr = reinterpret_cast<const float *>(kt + key * G::kRow);
#pragma unroll 4
            for (int e = 0; e < D; e += 4) {
                float k4[4];
                four(kr + e, k4);
#pragma unroll
                for (int r = 0; r < RH; ++r) {
                    const float4 q4 = *reinterpret_cast<const float4 *>(q_s + (r0 + r) * D + e);
                    s[r] = fmaf(q4.x, k4[0], fmaf(q4.y, k4[1], fmaf(q4.z, k4[2], fmaf(q4.w, k4[3], s[r]))));
                }
            }
#pragma unroll
            for (int r = 0; r < RH; ++r) s_s[(r0 + r) * (kKeys + 1) + key] = first + key < it.key1 && first + key <= last_seen(r0 + r) ? s[r] * scale2 : -INFINITY;
        }
        __syncthreads();
        {  // softmax: kThreads / RT threads a row
            constexpr int L = kThreads / RT, N = kKeys / L;
            const int r = tid / L, l = tid % L;
            float s[N], m = -INFINITY, t = 0.f;
#pragma unroll
            for (int i = 0; i < N; ++i) s[i] = s_s[r * (kKeys + 1) + l + L * i], m = fmaxf(m, s[i]);
#pragma unroll
            for (int o = L / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            const float old = mx[r], top = fmaxf(old, m), base = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float w = ex2f(s[i] - base);
                t += w;
                p_s[(l + L * i) * RT + r] = w;
            }
#pragma unroll
            for (int o = L / 2; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
            __syncwarp();
            if (l == 0) {
                const float f = ex2f(old - base);
                fac[r] = f;
                mx[r] = top;
                sum[r] = fmaf(sum[r], f, t);
            }
        }
        __syncthreads();
        {  // P.V: a quarter of the keys
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                const float f = fac[r];
#pragma unroll
                for (int e = 0; e < E; ++e) acc[r][e] *= f;
            }
            const bool hides = first + kKeys > it.key1 || (p.causal && first + kKeys - 1 > past + it.row0 / p.group);
            auto walk = [&](auto guarded) {
#pragma unroll 4
                for (int i = 0; i < kKeys / 4; ++i) {
                    const int key = warp * (kKeys / 4) + i;
                    const float *vr = reinterpret_cast<const float *>(vt + key * G::kRow) + lane * E;
                    float v[E];
                    if constexpr (E == 4) {
                        four(vr, v);
                    } else {
                        const float2 x = *reinterpret_cast<const float2 *>(vr);
                        v[0] = x.x; v[1] = x.y;
                    }
#pragma unroll
                    for (int r = 0; r < RT; r += 4) {
                        const float4 w4 = *reinterpret_cast<const float4 *>(p_s + key * RT + r);
                        const float w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                        for (int x = 0; x < 4; ++x)
                            // a position that the row does not see adds nothing, whatever its value is
                            if (!decltype(guarded)::value || (first + key <= last_seen(r + x) && first + key < it.key1))
#pragma unroll
                                for (int e = 0; e < E; ++e) acc[r + x][e] = fmaf(w[x], v[e], acc[r + x][e]);
                    }
                }
            };
            if (hides) walk(std::true_type());
            else walk(std::false_type());
        }
    }
    // the four warps' sums, in their order
    __syncthreads();
    float *o_s = reinterpret_cast<float *>(smem);  // [4][RT][D], over the tiles
    static_assert(4 * RT * D * 4 <= 4 * G::kTile, "the sums fit the tiles");
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int e = 0; e < E; ++e) o_s[(warp * RT + r) * D + lane * E + e] = acc[r][e];
    __syncthreads();
    for (int i = tid; i < it.rows * (D / 4); i += kThreads) {
        const int r = i / (D / 4), e = i % (D / 4) * 4;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float4 x = *reinterpret_cast<const float4 *>(o_s + (w * RT + r) * D + e);
            v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
        }
        const float m = mx[r], l = sum[r];
        if (it.part >= 0) {
            const size_t row = (size_t)it.part + r;
            *reinterpret_cast<float4 *>(a.part + row * D + e) = make_float4(v[0], v[1], v[2], v[3]);
            if (e == 0) *reinterpret_cast<float2 *>(a.part + (size_t)a.part_rows * D + 2 * row) = make_float2(m, l);
            continue;
        }
        const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
        const size_t o = (size_t)token(r) * p.n_head + head(r);
        *reinterpret_cast<float4 *>(static_cast<float *>(a.out) + o * D + e) = make_float4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
        if (e == 0 && a.lse) a.lse[o] = m * 0.6931471805599453f + logf(l);
    }
}

// Joins the parts of a row: a warp per row, the parts in their order.
template <int D>
__global__ void __launch_bounds__(128) paged_join_kernel(const PagedView p, const PagedAttnArgs a) {
    constexpr int E = D / 32;
    const PagedJoin j = a.joins[blockIdx.x];
    const int r = (int)(blockIdx.y * 4 + (threadIdx.x >> 5)), lane = threadIdx.x & 31;
    if (r >= j.rows) return;
    const PagedSeq sq = p.seqs[j.seq];
    const float2 *ml = reinterpret_cast<const float2 *>(a.part + (size_t)a.part_rows * D);
    float top = -INFINITY;
    for (int i = lane; i < j.splits; i += 32) top = fmaxf(top, ml[(size_t)j.part + (size_t)i * j.rows + r].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float base = top == -INFINITY ? 0.f : top;
    float v[E], l = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = 0.f;
#pragma unroll 4
    for (int i = 0; i < j.splits; ++i) {
        const size_t row = (size_t)j.part + (size_t)i * j.rows + r;
        const float2 x = ml[row];
        const float f = ex2f(x.x - base);
        l = fmaf(x.y, f, l);
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = fmaf(a.part[row * D + lane * E + e], f, v[e]);
    }
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    const size_t o = (size_t)(sq.tok0 + (j.row0 + r) / p.group) * p.n_head + j.kvh * p.group + (j.row0 + r) % p.group;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        if (a.out_dtype == LUMEN_F32) static_cast<float *>(a.out)[o * D + lane * E + e] = v[e] * inv;
        else static_cast<__nv_bfloat16 *>(a.out)[o * D + lane * E + e] = __float2bfloat16_rn(v[e] * inv);
    }
    if (lane == 0 && a.lse) a.lse[o] = top * 0.6931471805599453f + logf(l);
}

template <int D, int RT>
int launch(lumen_ctx *ctx, const PagedView &v, const PagedAttnArgs &a, cudaStream_t s) {
    constexpr size_t bytes = RowsSmem<D, RT>::kBytes;
    LUMEN_TRY(allow_smem(ctx, paged_rows_kernel<D, RT>, bytes));
    paged_rows_kernel<D, RT><<<(unsigned)a.n_items, kThreads, bytes, s>>>(v, a);
    LUMEN_LAUNCHED(ctx);
    return LUMEN_OK;
}
template <int D>
int pick(lumen_ctx *ctx, const PagedView &v, const PagedAttnArgs &a, cudaStream_t s) {
    return a.max_rows <= 4 ? launch<D, 4>(ctx, v, a, s) : a.max_rows <= 8 ? launch<D, 8>(ctx, v, a, s) : launch<D, 16>(ctx, v, a, s);
}

}  // namespace

PagedShape paged_rows_shape(const PagedGeom &g, int num_sms) {
    const int bytes = g.d * 4 * kKeys * 4;  // the tiles: what limits the CTAs of an SM
    return {16, kKeys, num_sms * (bytes > 100 * 1024 ? 1 : 2)};
}

int launch_paged_rows(lumen_ctx *ctx, const PagedGeom &g, const PagedView &v, const PagedAttnArgs &a, cudaStream_t s) {
    return g.d == 64 ? pick<64>(ctx, v, a, s) : pick<128>(ctx, v, a, s);
}

int launch_paged_join(lumen_ctx *ctx, const PagedGeom &g, const PagedView &v, const PagedAttnArgs &a, cudaStream_t s) {
    const dim3 grid((unsigned)a.n_joins, ((unsigned)a.join_rows + 3) / 4);
    if (g.d == 64) paged_join_kernel<64><<<grid, 128, 0, s>>>(v, a);
    else paged_join_kernel<128><<<grid, 128, 0, s>>>(v, a);
    LUMEN_LAUNCHED(ctx);
    return LUMEN_OK;
}

}  // namespace lumen
