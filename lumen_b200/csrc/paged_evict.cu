// Eviction: the positions of a sequence that received most attention, and its last ones, go to new pages.
//
// paged_select_kernel, a CTA or a cluster of CTAs per sequence and key head: the weights as ordered 32-bit integers, in shared memory where they fit;
// up to four passes over 8 bits each narrow the value of the last one that stays (fewer, once all that share the bits found so far stay: three
// for most long caches), and a last one writes the positions in order, of the equal ones the lowest.  The histograms have a column per lane, so that the
// many equal weights (nothing at all, say) do not queue for one counter: whole numbers, so the order of the atomics changes nothing.  Bound by the
// chain of its passes.  paged_move_kernel copies the rows: bound by HBM.
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

constexpr int kHeld = 40 * 1024;  // weights that the shared memory of a CTA holds

// grid (CTAs of a cluster x key heads, sequences); HELD: the weights of every sequence fit (else they are read again in every pass).  Four
// neighbouring positions a thread: bound by the instructions of its SMs.
template <bool HELD>
__global__ void __launch_bounds__(kThreads) paged_select_kernel(const PagedView from, const PagedSeq *to_seqs, int recent, int *kept, size_t kept_stride, int ctas) {
    extern __shared__ uint4 held[];
    __shared__ __align__(16) unsigned hist[256][32];
    __shared__ unsigned own[2][256], sums[256], prefix_s, want_s, whole_s, above_s[kWarps], equal_s[kWarps], counts_s[2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = (int)blockIdx.x % ctas, kvh = (int)blockIdx.x / ctas, s = blockIdx.y;
    const PagedSeq sq = from.seqs[s];
    const int len = sq.kv_len, keep = to_seqs[s].kv_len, last = min(recent, keep), old = len - last, pick = keep - last;
    const int all_groups = (old + 3) / 4, share = (all_groups + ctas - 1) / ctas, first = min(all_groups, rank * share), groups = min(all_groups, first + share) - first;
    const int *table = from.tables + sq.table;
    int *out = kept + ((size_t)s * from.h_kv + kvh) * kept_stride;
    pdl_launch();
    pdl_wait();
    for (int i = rank * kThreads + tid; i < last; i += ctas * kThreads) out[pick + i] = old + i;
    if (pick == 0) return;  // (of the whole cluster)
    auto fetch = [&](int group) {  // (a page holds whole groups; what of the last group lies behind `old` is left out where it is used)
        const float4 m = *reinterpret_cast<const float4 *>(from.mass + paged_row(from, table, kvh, 4 * (first + group)));
        return make_uint4(order_of(m.x), order_of(m.y), order_of(m.z), order_of(m.w));
    };
    auto value = [&](int group) { return HELD ? held[group] : fetch(group); };
    auto rest = [&](int group) { return old - 4 * (first + group); };  // positions from the group's first on
    // the pick-th largest value: `prefix` are its leading bits, `want` how many of those that share them are still to be taken
    uint32_t prefix = 0u;
    unsigned want = (unsigned)pick;
    for (int shift = 24; shift >= 0; shift -= 8) {
#pragma unroll
        for (int i = 0; i < 256 * 8 / kThreads; ++i) reinterpret_cast<uint4 *>(&hist[0][0])[tid + i * kThreads] = make_uint4(0u, 0u, 0u, 0u);
        __syncthreads();
        const uint32_t mask = shift == 24 ? 0u : ~0u << (shift + 8);
        auto count = [&](uint32_t u, bool live) {
            if (live && (u & mask) == prefix) atomicAdd(&hist[(u >> shift) & 255u][lane], 1u);
        };
        if (HELD && shift == 24) {
#pragma unroll 4
            for (int i = tid; i < groups; i += kThreads) held[i] = fetch(i);  // (a thread reads back what it wrote itself)
        }
#pragma unroll 2
        for (int i = tid; i < groups; i += kThreads) {
            const uint4 u = value(i);
            const int n = rest(i);
            count(u.x, true);
            count(u.y, n > 1);
            count(u.z, n > 2);
            count(u.w, n > 3);
        }
        __syncthreads();
        unsigned *mine_s = ctas > 1 ? own[(shift >> 3) & 1] : sums;
        {  // four threads a counter
            const uint4 *row = reinterpret_cast<const uint4 *>(&hist[tid >> 2][(tid & 3) * 8]);
            const uint4 x = row[0], y = row[1];
            unsigned c = x.x + x.y + x.z + x.w + y.x + y.y + y.z + y.w;
            c += __shfl_xor_sync(0xffffffffu, c, 1);
            c += __shfl_xor_sync(0xffffffffu, c, 2);
            if ((tid & 3) == 0) mine_s[tid >> 2] = c;
        }
        if (ctas > 1) {  // (two sets in turn: the one of the pass before may still be read)
            cluster_meet();
            if (tid < 256) {
                unsigned c = 0u;
                for (int r = 0; r < ctas; ++r) c += there(&mine_s[tid], (unsigned)r);
                sums[tid] = c;
            }
        }
        __syncthreads();
        if (warp == 0) {  // lane l has the bins 255 - 8 l down to 248 - 8 l
            unsigned c[8], mine = 0u;
#pragma unroll
            for (int i = 0; i < 8; ++i) c[i] = sums[255 - 8 * lane - i], mine += c[i];
            unsigned incl = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned y = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += y;
            }
            unsigned before = incl - mine;
            if (before < want && want <= incl) {  // (of exactly one lane)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (before < want && want <= before + c[i]) {
                        prefix_s = prefix | (unsigned)(255 - 8 * lane - i) << shift;
                        want_s = want - before;
                        whole_s = want - before == c[i];
                    }
                    before += c[i];
                }
            }
        }
        __syncthreads();
        prefix = prefix_s;
        want = want_s;
        if (whole_s && prefix) {  // all that share these bits stay: the last of them need not be found
            --prefix;
            want = 0u;
            break;
        }
    }
    const uint32_t edge = prefix;  // all above it stay, and the first `want` equal to it
    // every warp has a run of groups: it counts them, learns what the warps and CTAs before it have, and writes its own
    const int run = ((groups + kWarps - 1) / kWarps + 31) & ~31, lo = min(groups, warp * run), hi = min(groups, lo + run);
    auto kinds = [&](int i, unsigned &gt, unsigned &eq) {  // a bit for each of the four positions
        gt = eq = 0u;
        if (i >= hi) return;
        const uint4 u = value(i);
        const unsigned live = rest(i) >= 4 ? 15u : (1u << rest(i)) - 1u;
        gt = ((u.x > edge) | (u.y > edge) << 1 | (u.z > edge) << 2 | (u.w > edge) << 3) & live;
        eq = ((u.x == edge) | (u.y == edge) << 1 | (u.z == edge) << 2 | (u.w == edge) << 3) & live;
    };
    unsigned above = 0u, equal = 0u, gt, eq;
    for (int i0 = lo; i0 < hi; i0 += 32) {
        kinds(i0 + lane, gt, eq);
        above += __popc(gt);
        equal += __popc(eq);
    }
    above = __reduce_add_sync(0xffffffffu, above);
    equal = __reduce_add_sync(0xffffffffu, equal);
    if (lane == 0) above_s[warp] = above, equal_s[warp] = equal;
    __syncthreads();
    const unsigned before_above = __reduce_add_sync(0xffffffffu, lane < warp ? above_s[lane] : 0u), before_equal = __reduce_add_sync(0xffffffffu, lane < warp ? equal_s[lane] : 0u);
    if (ctas > 1) {
        if (warp == kWarps - 1 && lane == 0) counts_s[0] = before_above + above, counts_s[1] = before_equal + equal;
        cluster_meet();
    }
    above = before_above;
    equal = before_equal;
    for (int r = 0; r < rank; ++r) above += there(&counts_s[0], (unsigned)r), equal += there(&counts_s[1], (unsigned)r);
    for (int i0 = lo; i0 < hi; i0 += 32) {
        const int i = i0 + lane;
        kinds(i, gt, eq);
        const unsigned mine = (unsigned)__popc(gt) | (unsigned)__popc(eq) << 16;  // (at most 128 of each)
        unsigned incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
        }
        unsigned g = above + ((incl - mine) & 0xffffu), e = equal + ((incl - mine) >> 16);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const bool is_gt = (gt >> x) & 1u, is_eq = (eq >> x) & 1u;
            if (is_gt || (is_eq && e < want)) out[g + min(e, want)] = 4 * (first + i) + x;
            g += is_gt;
            e += is_eq;
        }
        const unsigned all = __shfl_sync(0xffffffffu, incl, 31);
        above += all & 0xffffu;
        equal += all >> 16;
    }
    if (ctas > 1) cluster_meet();  // (the counts may still be read by the CTAs behind)
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
        // Long sequences, where there are SMs for it: four each (with the copy, 32 rows of 16384 positions 32 us, with one SM each 35, with eight, two
        // CTAs an SM, 59); short ones: the cluster's meetings cost what they save.
        const int ctas = max_len > 4096 && 4LL * from.h_kv * n <= 2LL * ctx->num_sms ? 4 : 1, held = ((max_len + 3) / 4 + ctas - 1) / ctas;
        const dim3 grid((unsigned)(ctas * from.h_kv), (unsigned)n);
        auto *kernel = held * 4 <= kHeld ? paged_select_kernel<true> : paged_select_kernel<false>;
        const size_t smem = held * 4 <= kHeld ? (size_t)held * 16 : 0;
        if (smem) LUMEN_TRY(raise_smem_limit(ctx, reinterpret_cast<const void *>(kernel), kHeld * 4));
        LUMEN_TRY(launch_paged(ctx, kernel, (unsigned)ctas, grid, kThreads, smem, s, f, t.seqs, recent, k, kept_stride, ctas));
        LUMEN_TRY(bytes == 128 ? move<128>(ctx, f, t, n, max_keep, k, kept_stride, s)
                  : bytes == 256 ? move<256>(ctx, f, t, n, max_keep, k, kept_stride, s) : move<512>(ctx, f, t, n, max_keep, k, kept_stride, s));
    }
    return LUMEN_OK;
}

}  // namespace lumen
