// New tokens into a paged cache: norm, rotation, rounding and the write to the slots in one pass over the projections.
//
// y = x / sqrt(mean(x^2) + eps) * w per head, then (a, b) -> (a c - b s, b c + a s) over the pairs (i, i + d/2); values are copied.  A warp
// holds a head vector, d / 32 neighbours a lane, so the partner of a pair is the lane 16 further.  Every number is read once and
// written once: bound by HBM (by the launch for a decode step).  A warp takes kHeads heads whose loads go out together.
#include "paged.cuh"

namespace lumen {
namespace {

constexpr int kWarps = 8, kHeads = 2;

template <int E>
__device__ __forceinline__ void load_row(float (&v)[E], const float *src, bool vec) {
    if (vec) {
        if constexpr (E == 4) {
            const float4 x = __ldcs(reinterpret_cast<const float4 *>(src));
            v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
        } else {
            const float2 x = __ldcs(reinterpret_cast<const float2 *>(src));
            v[0] = x.x; v[1] = x.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = src[i];
    }
}

template <int E>
__device__ __forceinline__ void store_row(float *dst, const float (&v)[E]) {
    if constexpr (E == 4) *reinterpret_cast<float4 *>(dst) = make_float4(v[0], v[1], v[2], v[3]);
    else *reinterpret_cast<float2 *>(dst) = make_float2(v[0], v[1]);
}
template <int E>
__device__ __forceinline__ void store_row(__nv_bfloat16 *dst, const float (&v)[E]) {
#pragma unroll
    for (int i = 0; i < E; i += 2) *reinterpret_cast<__nv_bfloat162 *>(dst + i) = __floats2bfloat162_rn(v[i], v[i + 1]);
}

// grid (heads of q, k and v / 16, tokens): the heads of a token side by side
template <typename T, int D>
__global__ void __launch_bounds__(kWarps * 32) paged_append_kernel(const PagedView p, const PagedAppendArgs a, bool vec) {
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e0 = lane * E, all = p.n_head + 2 * p.h_kv;
    const int h0 = (int)(blockIdx.x * kWarps + warp) * kHeads;
    const size_t t = blockIdx.y + (size_t)gridDim.y * blockIdx.z;
    pdl_launch();
    if (t >= (size_t)p.tokens || h0 >= all) return pdl_wait();
    const int slot = p.tok_slot[t], pos = p.tok_pos[t];
    pdl_wait();
    float v[kHeads][E];
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
        const int h = h0 + i;
        if (h < all) {
            const float *src = h < p.n_head ? a.q + t * a.q_stride + (size_t)h * D
                                            : (h < p.n_head + p.h_kv ? a.k + (size_t)(h - p.n_head) * D : a.v + (size_t)(h - p.n_head - p.h_kv) * D) + t * a.kv_stride;
            load_row<E>(v[i], src + e0, vec);
        }
    }
    float co[E], sn[E];
    const bool rot = a.cos_t != nullptr && h0 < p.n_head + p.h_kv;
    if (rot) {
        const size_t at = (size_t)pos * (D / 2) + (size_t)(e0 & (D / 2 - 1));
#pragma unroll
        for (int i = 0; i < E; ++i) co[i] = a.cos_t[at + i], sn[i] = a.sin_t[at + i];
    }
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
        const int h = h0 + i;
        if (h >= all) break;
        const bool is_q = h < p.n_head, is_k = !is_q && h < p.n_head + p.h_kv;
        const float *gain = is_q ? a.q_norm : is_k ? a.k_norm : nullptr;
        if (gain) {
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) ss = fmaf(v[i][e], v[i][e], ss);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            const float inv = __fdiv_rn(1.0f, sqrtf(ss / (float)D + a.eps));
#pragma unroll
            for (int e = 0; e < E; ++e) v[i][e] = v[i][e] * inv * gain[e0 + e];
        }
        if (rot && (is_q || is_k)) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float other = __shfl_xor_sync(0xffffffffu, v[i][e], 16);
                v[i][e] = v[i][e] * co[e] + (lane < 16 ? -other : other) * sn[e];
            }
        }
        if (is_q) {
            store_row<E>(static_cast<T *>(a.q_out) + (t * p.n_head + h) * D + e0, v[i]);
        } else {
            const int hk = is_k ? h - p.n_head : h - p.n_head - p.h_kv;
            const size_t row = ((((size_t)slot >> p.page_shift) * p.h_kv + hk) << p.page_shift) + (slot & ((1 << p.page_shift) - 1));
            store_row<E>(static_cast<T *>(is_k ? p.k : p.v) + row * D + e0, v[i]);
            if (is_k && lane == 0) p.mass[row] = 0.f;
        }
    }
}

template <typename T, int D>
int launch(lumen_ctx *ctx, const PagedView &v, const PagedAppendArgs &a, cudaStream_t s) {
    constexpr size_t kAlign = D / 32 * 4;  // of the vector that a lane loads
    auto whole = [&](const float *p, size_t stride) { return reinterpret_cast<uintptr_t>(p) % kAlign == 0 && stride * 4 % kAlign == 0; };
    const bool vec = whole(a.q, a.q_stride) && whole(a.k, a.kv_stride) && whole(a.v, a.kv_stride);
    const unsigned y = (unsigned)std::min(v.tokens, 32768), z = ((unsigned)v.tokens + y - 1) / y;
    const dim3 grid(((unsigned)v.n_head + 2u * (unsigned)v.h_kv + kWarps * kHeads - 1) / (kWarps * kHeads), y, z);
    return launch_paged(ctx, paged_append_kernel<T, D>, grid, kWarps * 32, 0, s, v, a, vec);
}

}  // namespace

int launch_paged_append(lumen_ctx *ctx, const PagedGeom &g, const PagedView &v, const PagedAppendArgs &a, cudaStream_t s) {
    if (g.dtype == LUMEN_F32) return g.d == 64 ? launch<float, 64>(ctx, v, a, s) : launch<float, 128>(ctx, v, a, s);
    return g.d == 64 ? launch<__nv_bfloat16, 64>(ctx, v, a, s) : launch<__nv_bfloat16, 128>(ctx, v, a, s);
}

}  // namespace lumen
