// What the cached positions were looked at: mass[j] += sum over the rows that see j of exp(scale * q . k_j - lse).
//
// Every position belongs to one thread, which walks the rows in their order: nothing is exchanged, no atomics, the same sum every time.
#include "paged.cuh"

namespace lumen {
namespace {

constexpr int kKeys = 64, kRows = 16, kThreads = 128;

__device__ __forceinline__ void four(const float *p, float (&v)[4]) {
    const float4 x = *reinterpret_cast<const float4 *>(p);
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
}
__device__ __forceinline__ void four(const __nv_bfloat16 *p, float (&v)[4]) {
    const uint2 x = *reinterpret_cast<const uint2 *>(p);
    v[0] = __uint_as_float(x.x << 16); v[1] = __uint_as_float(x.x & 0xffff0000u);
    v[2] = __uint_as_float(x.y << 16); v[3] = __uint_as_float(x.y & 0xffff0000u);
}

// grid (tiles of the longest sequence, key heads, sequences)
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) paged_mass_kernel(const PagedView p, const T *__restrict__ q, float scale, const float *__restrict__ lse) {
    __shared__ __align__(16) float k_s[kKeys][D + 4];
    __shared__ __align__(16) float q_s[kRows][D];
    __shared__ float l_s[kRows], half_s[kKeys];
    const int tid = threadIdx.x, kvh = blockIdx.y;
    const PagedSeq sq = p.seqs[blockIdx.z];
    const int key0 = blockIdx.x * kKeys, past = sq.kv_len - sq.q_len;
    if (key0 >= sq.kv_len || sq.q_len == 0) return;
    const int *table = p.tables + sq.table;
    for (int i = tid; i < kKeys * (D / 4); i += kThreads) {
        const int r = i / (D / 4), e = i % (D / 4) * 4;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        if (key0 + r < sq.kv_len) four(static_cast<const T *>(p.k) + paged_row(p, table, kvh, key0 + r) * D + e, v);
        *reinterpret_cast<float4 *>(&k_s[r][e]) = make_float4(v[0], v[1], v[2], v[3]);
    }
    const int key = tid % kKeys, half = tid / kKeys, rows = sq.q_len * p.group;
    const int start = p.causal ? max(0, key0 - past) * p.group : 0;  // the first row that sees any of the tile
    float gained = 0.f;
    for (int r0 = start; r0 < rows; r0 += kRows) {
        __syncthreads();
        for (int i = tid; i < kRows * (D / 4); i += kThreads) {
            const int r = i / (D / 4), e = i % (D / 4) * 4, row = r0 + r;
            float v[4] = {0.f, 0.f, 0.f, 0.f};
            if (row < rows) four(q + ((size_t)(sq.tok0 + row / p.group) * p.n_head + kvh * p.group + row % p.group) * D + e, v);
            *reinterpret_cast<float4 *>(&q_s[r][e]) = make_float4(v[0], v[1], v[2], v[3]);
        }
        if (tid < kRows && r0 + tid < rows) l_s[tid] = lse[(size_t)(sq.tok0 + (r0 + tid) / p.group) * p.n_head + kvh * p.group + (r0 + tid) % p.group];
        __syncthreads();
        constexpr int RH = kRows / 2;
        float s[RH];
#pragma unroll
        for (int r = 0; r < RH; ++r) s[r] = 0.f;
#pragma unroll 4
        for (int e = 0; e < D; e += 4) {
            const float4 k4 = *reinterpret_cast<const float4 *>(&k_s[key][e]);
#pragma unroll
            for (int r = 0; r < RH; ++r) {
                const float4 q4 = *reinterpret_cast<const float4 *>(&q_s[half * RH + r][e]);
                s[r] = fmaf(q4.x, k4.x, fmaf(q4.y, k4.y, fmaf(q4.z, k4.z, fmaf(q4.w, k4.w, s[r]))));
            }
        }
#pragma unroll
        for (int r = 0; r < RH; ++r) {
            const int row = r0 + half * RH + r;
            if (row < rows && (!p.causal || key0 + key <= past + row / p.group)) gained += expf(s[r] * scale - l_s[half * RH + r]);
        }
    }
    if (half) half_s[key] = gained;
    __syncthreads();
    if (!half && key0 + key < sq.kv_len) p.mass[paged_row(p, table, kvh, key0 + key)] += gained + half_s[key];
}

template <typename T, int D>
int launch(lumen_ctx *ctx, const PagedView &v, const void *q, float scale, const float *lse, int max_kv, cudaStream_t s) {
    // (sequences beyond the grid's third extent go in further launches)
    for (int s0 = 0; s0 < v.n_seq; s0 += 32768) {
        PagedView w = v;
        w.seqs += s0;
        const dim3 grid((unsigned)((max_kv + kKeys - 1) / kKeys), (unsigned)v.h_kv, (unsigned)std::min(v.n_seq - s0, 32768));
        paged_mass_kernel<T, D><<<grid, kThreads, 0, s>>>(w, static_cast<const T *>(q), scale, lse);
        LUMEN_LAUNCHED(ctx);
    }
    return LUMEN_OK;
}

}  // namespace

int launch_paged_mass(lumen_ctx *ctx, const PagedGeom &g, const PagedView &v, const void *q, float scale, const float *lse, int max_kv, cudaStream_t s) {
    if (g.dtype == LUMEN_F32) return g.d == 64 ? launch<float, 64>(ctx, v, q, scale, lse, max_kv, s) : launch<float, 128>(ctx, v, q, scale, lse, max_kv, s);
    return g.d == 64 ? launch<__nv_bfloat16, 64>(ctx, v, q, scale, lse, max_kv, s) : launch<__nv_bfloat16, 128>(ctx, v, q, scale, lse, max_kv, s);
}

}  // namespace lumen
