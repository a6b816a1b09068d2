// Eviction: the positions of a sequence that received most attention, and its last ones, go to new pages.
//
// paged_select_kernel, a CTA per sequence and key head: the weights as ordered 32-bit integers, in shared memory where they fit; four passes over 8
// bits each narrow the value of the last one that stays, and a last one writes the positions in order, of the equal ones the lowest.  The
// histograms have a column per lane, so that the many equal weights (nothing at all, say) do not queue for one counter: whole numbers, so the
// order of the atomics changes nothing.  paged_move_kernel copies the rows: bound by HBM.
#include "paged.cuh"

namespace lumen {
namespace {

constexpr int kThreads = 1024, kWarps = kThreads / 32;

// Larger weight, larger number; NaN the smallest of all.
__device__ __forceinline__ uint32_t order_of(float x) {
    if (x != x) return 0u;
    const uint32_t u = __float_as_uint(x + 0.f);  // (-0 becomes 0)
    return (u >> 31) ? ~u : u | 0x80000000u;
}

constexpr int kHeld = 40 * 1024;  // weights that shared memory holds

// grid (key heads, sequences); HELD: the weights of every sequence fit (else they are read again in every pass)
template <bool HELD>
__global__ void __launch_bounds__(kThreads) paged_select_kernel(const PagedView from, const PagedSeq *to_seqs, int recent, int *kept, size_t kept_stride) {
    extern __shared__ uint32_t held[];
    __shared__ unsigned hist[256][32], sums[256];
    __shared__ unsigned prefix_s, want_s, above_s[kWarps], equal_s[kWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, kvh = blockIdx.x, s = blockIdx.y;
    const PagedSeq sq = from.seqs[s];
    const int len = sq.kv_len, keep = to_seqs[s].kv_len, last = min(recent, keep), old = len - last, pick = keep - last;
    const int *table = from.tables + sq.table;
    int *out = kept + ((size_t)s * from.h_kv + kvh) * kept_stride;
    pdl_launch();
    pdl_wait();
    for (int i = tid; i < last; i += kThreads) out[pick + i] = old + i;
    if (pick == 0) return;
    auto fetch = [&](int pos) { return order_of(from.mass[paged_row(from, table, kvh, pos)]); };
    auto value = [&](int pos) { return HELD ? held[pos] : fetch(pos); };
    if (HELD)
#pragma unroll 4
        for (int i = tid; i < old; i += kThreads) held[i] = fetch(i);
    // the pick-th largest value: `prefix` are its leading bits, `want` how many of those that share them are still to be taken
    if (tid == 0) prefix_s = 0u, want_s = (unsigned)pick;
    for (int shift = 24; shift >= 0; shift -= 8) {
#pragma unroll
        for (int i = 0; i < 256 * 32 / kThreads; ++i) (&hist[0][0])[tid + i * kThreads] = 0u;
        __syncthreads();
        const unsigned prefix = prefix_s;
        for (int i = tid; i < old; i += kThreads) {
            const uint32_t u = value(i);
            if (shift == 24 || (u >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(u >> shift) & 255u][lane], 1u);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 256 / kWarps; ++i) {
            const int bin = warp * (256 / kWarps) + i;
            const unsigned c = __reduce_add_sync(0xffffffffu, hist[bin][lane]);
            if (lane == 0) sums[bin] = c;
        }
        __syncthreads();
        if (warp == 0) {  // lane l: bins 255 - 8 l down to 248 - 8 l
            unsigned c[8], mine = 0u;
#pragma unroll
            for (int i = 0; i < 8; ++i) c[i] = sums[255 - 8 * lane - i], mine += c[i];
            unsigned incl = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned y = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += y;
            }
            const unsigned want = want_s;
            unsigned before = incl - mine;
            __syncwarp();
            if (before < want && want <= incl)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (before < want && want <= before + c[i]) {
                        prefix_s = prefix | ((unsigned)(255 - 8 * lane - i) << shift);
                        want_s = want - before;
                    }
                    before += c[i];
                }
        }
        __syncthreads();
    }
    const unsigned edge = prefix_s, ties = want_s;  // all above `edge` stay, and the first `ties` equal to it
    // every warp has a run of positions: it counts them, learns what the warps before it have, and writes its own
    const int run = ((old + kWarps - 1) / kWarps + 31) & ~31, lo = min(old, warp * run), hi = min(old, lo + run);
    unsigned above = 0u, equal = 0u;
    for (int i0 = lo; i0 < hi; i0 += 32) {
        const uint32_t u = i0 + lane < hi ? value(i0 + lane) : 0u;
        above += __popc(__ballot_sync(0xffffffffu, i0 + lane < hi && u > edge));
        equal += __popc(__ballot_sync(0xffffffffu, i0 + lane < hi && u == edge));
    }
    if (lane == 0) above_s[warp] = above, equal_s[warp] = equal;
    __syncthreads();
    above = __reduce_add_sync(0xffffffffu, lane < warp ? above_s[lane] : 0u);
    equal = __reduce_add_sync(0xffffffffu, lane < warp ? equal_s[lane] : 0u);
    for (int i0 = lo; i0 < hi; i0 += 32) {
        const int i = i0 + lane;
        const uint32_t u = i < hi ? value(i) : 0u;
        const bool gt = i < hi && u > edge, eq = i < hi && u == edge;
        const unsigned mg = __ballot_sync(0xffffffffu, gt), me = __ballot_sync(0xffffffffu, eq), low = (1u << lane) - 1u;
        const unsigned g = above + (unsigned)__popc(mg & low), e = equal + (unsigned)__popc(me & low);
        if (gt || (eq && e < ties)) out[g + min(e, ties)] = i;
        above += (unsigned)__popc(mg);
        equal += (unsigned)__popc(me);
    }
}

// grid (groups of rows, key heads, sequences): 16 bytes a thread
template <int B>  // bytes of a row
__global__ void __launch_bounds__(256) paged_move_kernel(const PagedView from, const PagedView to, const int *kept, size_t kept_stride) {
    constexpr int kLanes = B / 16, kRowsPer = 256 / kLanes;
    const int kvh = blockIdx.y, s = blockIdx.z, lane = threadIdx.x % kLanes, i = (int)blockIdx.x * kRowsPer + threadIdx.x / kLanes;
    const PagedSeq a = from.seqs[s], b = to.seqs[s];
    pdl_launch();
    pdl_wait();
    if (i >= b.kv_len) return;
    const int pos = kept[((size_t)s * from.h_kv + kvh) * kept_stride + i];
    const size_t src = paged_row(from, from.tables + a.table, kvh, pos), dst = paged_row(to, to.tables + b.table, kvh, i);
    const size_t so = src * B + 16 * lane, d = dst * B + 16 * lane;
    const uint4 k = __ldcs(reinterpret_cast<const uint4 *>(static_cast<const char *>(from.k) + so));
    const uint4 v = __ldcs(reinterpret_cast<const uint4 *>(static_cast<const char *>(from.v) + so));
    *reinterpret_cast<uint4 *>(static_cast<char *>(to.k) + d) = k;
    *reinterpret_cast<uint4 *>(static_cast<char *>(to.v) + d) = v;
    if (lane == 0) to.mass[dst] = from.mass[src];
}

template <int B>
int move(lumen_ctx *ctx, const PagedView &from, const PagedView &to, int n, int max_keep, const int *kept, size_t kept_stride, cudaStream_t s) {
    constexpr int kRowsPer = 256 / (B / 16);
    const dim3 grid((unsigned)((max_keep + kRowsPer - 1) / kRowsPer), (unsigned)from.h_kv, (unsigned)n);
    return launch_paged(ctx, paged_move_kernel<B>, grid, 256, 0, s, from, to, kept, kept_stride);
}

}  // namespace

int launch_paged_evict(lumen_ctx *ctx, const PagedGeom &g, const PagedView &from, const PagedView &to, int recent, int max_len, int max_keep, int *kept,
                       size_t kept_stride, cudaStream_t s) {
    const int bytes = g.d * (g.dtype == LUMEN_F32 ? 4 : 2);
    for (int s0 = 0; s0 < from.n_seq; s0 += 32768) {  // (the grid's extents)
        const int n = std::min(from.n_seq - s0, 32768);
        PagedView f = from, t = to;
        f.seqs += s0;
        t.seqs += s0;
        int *k = kept + (size_t)s0 * from.h_kv * kept_stride;
        const dim3 grid((unsigned)from.h_kv, (unsigned)n);
        if (max_len <= kHeld) {
            LUMEN_TRY(raise_smem_limit(ctx, reinterpret_cast<const void *>(paged_select_kernel<true>), kHeld * 4));
            LUMEN_TRY(launch_paged(ctx, paged_select_kernel<true>, grid, kThreads, (size_t)max_len * 4, s, f, t.seqs, recent, k, kept_stride));
        } else {
            LUMEN_TRY(launch_paged(ctx, paged_select_kernel<false>, grid, kThreads, 0, s, f, t.seqs, recent, k, kept_stride));
        }
        LUMEN_TRY(bytes == 128 ? move<128>(ctx, f, t, n, max_keep, k, kept_stride, s)
                  : bytes == 256 ? move<256>(ctx, f, t, n, max_keep, k, kept_stride, s) : move<512>(ctx, f, t, n, max_keep, k, kept_stride, s));
    }
    return LUMEN_OK;
}

}  // namespace lumen
