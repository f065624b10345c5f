// lalb_kv_evict.cu -- eviction from a batch's KV cache by accumulated
// attention weight (lalb_kv_evict): per sequence and KV head the `keep` rows
// that stay, and the copies that bring them below `keep`.
//
// Attention does not care about the order of a cache's rows (their keys are
// rotated already), so nothing is compacted in order: the kept rows below
// `keep` stay, and the i-th kept row above takes the i-th place given up
// below.  That is the least that can move (each kept row above the limit once),
// and since every source lies at or above `keep` and every destination below
// it, the copies need no order among themselves.
//
// evict_select_kernel, one cluster of 1, 2 or 4 CTAs per (sequence, KV
// head): a 32-bit key per row (protected rows the largest, weights in their
// order, NaN 0) kept in the shared memory of the CTA that owns the row, the
// keep-th largest key by up to three counting passes of 11, 11 and 10 bits
// whose counts the CTAs add up over distributed shared memory, then the two
// lists by ballots: CTA, warp and lane own rows in row order, so that ranks
// follow it.  With one CTA it is bound by instructions (30 per 32 rows and
// pass: 42 us for 32768 rows), hence the cluster.
// Its six walks over the rows (three counts, ties, two for the lists) are most
// of a call on long rows: 23 us of 40 for 16 pairs of 32768 rows, 64 CTAs.
// evict_move_kernel copies the rows, 4 head_dim elements per moved row, and
// their positions and weights.  Latency bounds it: each 16-byte piece loads two
// indices before its data, and 19 us for 32 sequences of 1500 to 4095 bf16 rows
// cut to 2000 are 26 % of the DRAM's rate and 24 % of L2's.
#include <cooperative_groups.h>

#include <algorithm>

#include "lalb_batch.cuh"

using namespace lalb;
namespace cg = cooperative_groups;

namespace {

constexpr int kSelThreads = 1024;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kBins = 2048;
constexpr size_t kKeyBytesMax = 180 * 1024;   // keys of up to 46080 rows of a CTA stay in shared memory
constexpr int kMaxCluster = 4;
constexpr int kRowsPerCta = 8192;             // fewer are not worth another CTA
constexpr int kMoveThreads = 256;
constexpr int kMoveUnroll = 2;                // 16-byte pieces in flight per thread (4 and 8: 2 and 6 us more of 31)
constexpr int kMoveFill = 16;                 // blocks per SM

struct EvictArgs {
    int *lens;
    int *row_pos;
    float *row_weight;
    uint8_t *k, *v;
    int2 *count;           // [n_seq * n_kv] (rows that move, length; 0, 0: nothing to do)
    int *dst, *src;        // [n_seq * n_kv][list] places below keep, rows above it
    unsigned int *status;
    int n_seq, max_ctx, n_kv, keep, n_sink, n_recent, list;
    int shift;             // log2 of the 16-byte pieces of one row of one KV head
};

__device__ __forceinline__ uint32_t weight_key(float w) {
    return w != w ? 0u : ordered_key(w + 0.0f);   // -0 counts as 0
}
__device__ __forceinline__ bool evict_safe(const EvictArgs &a, int p, int newest) {
    return p < a.n_sink || (long long)p > (long long)newest - a.n_recent;
}

// Rows i = t, t + 1024, .. below n, eight at a time: load(i, u) for all of a
// batch, then use(i, u).
template <class LOAD, class USE>
__device__ __forceinline__ void rows8(int t, int n, LOAD load, USE use) {
    for (int i0 = t; i0 < n; i0 += 8 * kSelThreads) {
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (i0 + u * kSelThreads < n) load(i0 + u * kSelThreads, u);
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (i0 + u * kSelThreads < n) use(i0 + u * kSelThreads, u);
    }
}

struct SelShared {
    uint32_t hist[3][kBins];        // one per pass: a CTA may still read one when the next is filled
    int wsum[3][kSelWarps];
    int newest;                     // read by the cluster's other CTAs: newest, ties, places, movers
    int ties, places, movers;
    uint32_t digit, above, count;
};

// kCached: every key in shared memory; otherwise each pass forms it again
// from row_pos and row_weight.  kCluster: more than one CTA.
template <bool kCached, bool kCluster>
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const EvictArgs a) {
    extern __shared__ uint32_t keys[];
    __shared__ SelShared sh;
    int rank = 0, size = 1;
    if constexpr (kCluster) {
        rank = (int)cg::this_cluster().block_rank();
        size = (int)cg::this_cluster().num_blocks();
    }
    auto sync = [&]() {
        if constexpr (kCluster)
            cg::this_cluster().sync();
        else
            __syncthreads();
    };
    auto peer = [&](int r) -> const SelShared * {
        if constexpr (kCluster) return cg::this_cluster().map_shared_rank(&sh, r);
        return &sh;
    };
    const int bg = blockIdx.x / size, b = bg / a.n_kv;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_wait();
    pdl_launch_dependents();
    const int n = a.lens[b];        // the same for every CTA of the cluster
    if (n < 0 || n > a.max_ctx) {
        if (tid == 0 && rank == 0) {
            a.count[bg] = make_int2(0, 0);
            atomicOr(a.status, LALB_STATUS_BAD_POSITION);
        }
        return;
    }
    if (n <= a.keep) {
        if (tid == 0 && rank == 0) a.count[bg] = make_int2(0, 0);
        return;
    }
    // this CTA's rows: [c0, c0 + nc), whole warps' worth but for the last
    const int chunk = ((n + size - 1) / size + 31) & ~31;
    const int c0 = min(n, rank * chunk), nc = min(n - c0, chunk);
    const int *pos = a.row_pos + (size_t)bg * a.max_ctx + c0;
    float *weight = a.row_weight + (size_t)bg * a.max_ctx + c0;

    // ---- the newest position, and the weights' keys -------------------------------
    int newest = INT_MIN;
    {
        int p[8];
        float w[8];
        rows8(
            tid, nc,
            [&](int i, int u) {
                p[u] = pos[i];
                if (kCached) w[u] = weight[i];
            },
            [&](int i, int u) {
                newest = max(newest, p[u]);
                if (kCached) keys[i] = weight_key(w[u]);
            });
    }
    for (int i = tid; i < 3 * kBins; i += kSelThreads) sh.hist[0][i] = 0;
    newest = __reduce_max_sync(0xffffffffu, newest);
    if (lane == 0) sh.wsum[0][warp] = newest;
    __syncthreads();
    newest = __reduce_max_sync(0xffffffffu, sh.wsum[0][lane]);
    if constexpr (kCluster) {
        if (tid == 0) sh.newest = newest;
        sync();
        newest = __reduce_max_sync(0xffffffffu, lane < size ? peer(lane)->newest : INT_MIN);
    }

    auto fresh_key = [&](int i) {
        return evict_safe(a, pos[i], newest) ? 0xffffffffu : weight_key(weight[i]);
    };
    auto key_of = [&](int i) -> uint32_t { return kCached ? keys[i] : fresh_key(i); };

    // ---- the keep-th largest key ----------------------------------------------------
    uint32_t prefix = 0, mask = 0;
    int need = a.keep;          // rows still to take among those that match the prefix
    bool all = false;           // every one of them is taken: no need to look closer
    for (int pass = 0; pass < 3 && !all; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const int bins = pass == 2 ? 1024 : 2048;
        uint32_t *hist = sh.hist[pass];
        // one atomic for the digit of the warp's first such lane (the weights'
        // leading bits agree for many rows), one each for the rest
        auto count_digit = [&](bool in, uint32_t d) {
            const uint32_t who = __ballot_sync(0xffffffffu, in);
            if (!who) return;
            const int lead = __ffs(who) - 1;
            const uint32_t dl = __shfl_sync(0xffffffffu, d, lead);
            const uint32_t same = __ballot_sync(0xffffffffu, in && d == dl);
            if (lane == lead)
                atomicAdd(&hist[d], (uint32_t)__popc(same));
            else if (in && d != dl)
                atomicAdd(&hist[d], 1u);
        };
        const int n32 = (nc + 31) & ~31;      // whole warps: ballots
        if (kCached && pass == 0) {
            int p[8];
            rows8(
                tid, n32, [&](int i, int u) { p[u] = i < nc ? pos[i] : 0; },
                [&](int i, int u) {
                    const bool in = i < nc;
                    uint32_t key = in ? keys[i] : 0u;
                    if (in && evict_safe(a, p[u], newest)) keys[i] = key = 0xffffffffu;
                    count_digit(in, key >> 21);
                });
        } else {
            uint32_t key[8];
            rows8(
                tid, n32, [&](int i, int u) { key[u] = i < nc ? key_of(i) : 0u; },
                [&](int i, int u) {
                    count_digit(i < nc && (key[u] & mask) == prefix, (key[u] >> shift) & (bins - 1));
                });
        }
        sync();
        // the digit whose rows straddle `need`, counted from the largest; every
        // CTA of the cluster finds the same
        const int per = bins / kSelThreads;
        const int hi = bins - 1 - tid * per;
        uint32_t top = 0, own = 0;
        for (int r = 0; r < size; ++r) {
            const uint32_t *h = peer(r)->hist[pass];
            top += h[hi];
            own += per == 2 ? h[hi] + h[hi - 1] : h[hi];
        }
        uint32_t incl = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t x = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += x;
        }
        if (lane == 31) sh.wsum[1][warp] = (int)incl;
        __syncthreads();
        const uint32_t before =
            incl - own + (uint32_t)__reduce_add_sync(0xffffffffu, lane < warp ? sh.wsum[1][lane] : 0);
        if (before < (uint32_t)need && (uint32_t)need <= before + own) {
            const bool second = per == 2 && before + top < (uint32_t)need;
            sh.digit = second ? hi - 1 : hi;
            sh.above = second ? before + top : before;
            sh.count = second ? own - top : top;
        }
        __syncthreads();
        prefix |= sh.digit << shift;
        mask |= (uint32_t)(bins - 1) << shift;
        need -= (int)sh.above;
        all = sh.count == (uint32_t)need;
        __syncthreads();
    }

    // ---- the lists: warp w owns rows [r0, r1) -----------------------------------------
    const int run = ((nc + kSelWarps - 1) / kSelWarps + 31) & ~31;
    const int r0 = min(nc, warp * run), r1 = min(nc, r0 + run);
    auto scan = [&](int which) -> int {   // sum of the earlier warps' wsum[which]
        return __reduce_add_sync(0xffffffffu, lane < warp ? sh.wsum[which][lane] : 0);
    };
    auto total = [&](int which) -> int { return __reduce_add_sync(0xffffffffu, sh.wsum[which][lane]); };
    // rows of the keep-th key: all of them are kept, or the first `need` in row order
    int ties0 = 0;
    if (!all) {
        int ties = 0;
        for (int i0 = r0; i0 < r1; i0 += 32) {
            const int i = i0 + lane;
            ties += __popc(__ballot_sync(0xffffffffu, i < r1 && key_of(i) == prefix));
        }
        if (lane == 0) sh.wsum[0][warp] = ties;
        __syncthreads();
        ties0 = scan(0);
        if constexpr (kCluster) {
            const int t = total(0);
            if (tid == 0) sh.ties = t;
            sync();
            ties0 += __reduce_add_sync(0xffffffffu, lane < rank ? peer(lane)->ties : 0);
        }
    }
    // pass 0 counts the warp's places and movers, pass 1 writes them at their
    // ranks and clears the weights of the rows that go
    int place = 0, mover = 0;
    const uint32_t lower = (1u << lane) - 1;
    for (int pass = 0; pass < 2; ++pass) {
        int tie = ties0;
        for (int i0 = r0; i0 < r1; i0 += 32) {
            const int i = i0 + lane;
            const bool live = i < r1;
            const uint32_t key = live ? key_of(i) : 0u;
            bool kept;
            if (all) {
                kept = live && key >= prefix;
            } else {
                const uint32_t eq = __ballot_sync(0xffffffffu, live && key == prefix);
                kept = live && (key > prefix || (key == prefix && tie + __popc(eq & lower) < need));
                tie += __popc(eq);
            }
            const bool low = c0 + i < a.keep;
            const bool is_place = live && !kept && low, is_mover = kept && !low;
            const uint32_t bp = __ballot_sync(0xffffffffu, is_place), bm = __ballot_sync(0xffffffffu, is_mover);
            if (pass == 1) {
                if (is_place) a.dst[(size_t)bg * a.list + place + __popc(bp & lower)] = c0 + i;
                if (is_mover) a.src[(size_t)bg * a.list + mover + __popc(bm & lower)] = c0 + i;
                if (live && !kept && !low) weight[i] = 0.0f;
            }
            place += __popc(bp);
            mover += __popc(bm);
        }
        if (pass == 0) {
            if (lane == 0) {
                sh.wsum[1][warp] = place;
                sh.wsum[2][warp] = mover;
            }
            __syncthreads();
            place = scan(1);
            mover = scan(2);
            int moved = total(1);
            if constexpr (kCluster) {
                const int m = total(2);
                if (tid == 0) {
                    sh.places = moved;
                    sh.movers = m;
                }
                sync();
                const int p = lane < size ? peer(lane)->places : 0, q = lane < rank ? peer(lane)->movers : 0;
                moved = __reduce_add_sync(0xffffffffu, p);
                place += __reduce_add_sync(0xffffffffu, lane < rank ? p : 0);
                mover += __reduce_add_sync(0xffffffffu, q);
            }
            // as many places as movers: exactly `keep` rows are kept
            if (tid == 0 && rank == 0) a.count[bg] = make_int2(moved, n);
        }
    }
    if constexpr (kCluster) sync();   // no CTA ends while another may read its shared memory
}

__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const EvictArgs a) {
    const int bg = blockIdx.y, b = bg / a.n_kv, g = bg % a.n_kv;
    pdl_wait();
    pdl_launch_dependents();
    const int2 c = __ldcg(a.count + bg);
    const int moved = c.x, n = c.y;
    if (n == 0) return;
    const int *dst = a.dst + (size_t)bg * a.list, *src = a.src + (size_t)bg * a.list;
    const size_t rows0 = (size_t)b * a.max_ctx;
    // positions and weights: the rows' new places get theirs, the old ones 0
    int *pos = a.row_pos + (size_t)bg * a.max_ctx;
    float *weight = a.row_weight + (size_t)bg * a.max_ctx;
    for (int i = blockIdx.x * kMoveThreads + threadIdx.x; i < moved; i += gridDim.x * kMoveThreads) {
        const int from = __ldcg(src + i), to = __ldcg(dst + i);
        pos[to] = pos[from];
        weight[to] = weight[from];
        weight[from] = 0.0f;
    }
    if (g == 0 && blockIdx.x == 0 && threadIdx.x == 0) a.lens[b] = a.keep;
    // piece p: 16 bytes of K (even rows of pieces) or V (odd) of move p >> (shift + 1)
    const long long pieces = (long long)moved << (a.shift + 1);
    const long long stride = (long long)gridDim.x * kMoveThreads;
    for (long long p0 = blockIdx.x * kMoveThreads + threadIdx.x; p0 < pieces; p0 += kMoveUnroll * stride) {
        uint4 x[kMoveUnroll];
        uint4 *to[kMoveUnroll];
#pragma unroll
        for (int u = 0; u < kMoveUnroll; ++u) {
            const long long p = p0 + u * stride;
            to[u] = nullptr;
            if (p < pieces) {
                const uint32_t row = (uint32_t)(p >> a.shift), c16 = (uint32_t)p & ((1u << a.shift) - 1), m = row >> 1;
                uint4 *t = reinterpret_cast<uint4 *>((row & 1) ? a.v : a.k);
                const size_t s = (rows0 + __ldcg(src + m)) * a.n_kv + g, d = (rows0 + __ldcg(dst + m)) * a.n_kv + g;
                x[u] = __ldcs(t + (s << a.shift) + c16);
                to[u] = t + (d << a.shift) + c16;
            }
        }
#pragma unroll
        for (int u = 0; u < kMoveUnroll; ++u)
            if (to[u]) *to[u] = x[u];
    }
}

size_t up256(size_t n) { return (n + 255) / 256 * 256; }
int list_len(const lalb_kv_batch *c, int keep) { return std::min(keep, c->max_ctx - keep); }

}  // namespace

extern "C" int lalb_kv_evict_ws_bytes(const lalb_kv_batch *cache, int keep, size_t *bytes) {
    if (!bytes) return LALB_ERR_INVALID;
    if (int st = kv_batch_shape(cache)) return st;
    if (keep < 1 || keep > cache->max_ctx) return LALB_ERR_INVALID;
    const size_t bg = (size_t)cache->n_seq * cache->n_kv_head;
    *bytes = up256(bg * sizeof(int2)) + 2 * up256(bg * list_len(cache, keep) * sizeof(int));
    return LALB_OK;
}

extern "C" int lalb_kv_evict(lalb_ctx *ctx, const lalb_kv_batch *cache, int32_t *lens, int keep, int n_sink,
                             int n_recent, void *ws, lalb_stream stream) try {
    if (!ctx) return LALB_ERR_INVALID;
    if (!cache || !lens || !ws) return lalb_fail(ctx, LALB_ERR_INVALID, "kv_evict: null pointer");
    if (int st = kv_batch_check(ctx, cache, "kv_evict")) return st;
    if (!cache->row_pos || !cache->row_weight)
        return lalb_fail(ctx, LALB_ERR_INVALID, "kv_evict: the cache needs row_pos and row_weight");
    if (keep < 1 || keep > cache->max_ctx || n_sink < 0 || n_recent < 0 || (long long)n_sink + n_recent > keep)
        return lalb_fail(ctx, LALB_ERR_INVALID, "kv_evict: keep %d of %d rows, n_sink %d, n_recent %d", keep,
                         cache->max_ctx, n_sink, n_recent);
    if (((uintptr_t)ws & 255u) || ((uintptr_t)lens & 3u))
        return lalb_fail(ctx, LALB_ERR_INVALID, "kv_evict: misaligned buffer");
    const long long bg = (long long)cache->n_seq * cache->n_kv_head;
    if (bg > 65535) return lalb_fail(ctx, LALB_ERR_UNSUPPORTED, "kv_evict: %lld sequences x KV heads", bg);
    EvictArgs a = {};
    a.lens = lens;
    a.row_pos = cache->row_pos;
    a.row_weight = cache->row_weight;
    a.k = static_cast<uint8_t *>(cache->k);
    a.v = static_cast<uint8_t *>(cache->v);
    a.list = list_len(cache, keep);
    uint8_t *w = static_cast<uint8_t *>(ws);
    a.count = reinterpret_cast<int2 *>(w);
    w += up256(bg * sizeof(int2));
    a.dst = reinterpret_cast<int *>(w);
    w += up256((size_t)bg * a.list * sizeof(int));
    a.src = reinterpret_cast<int *>(w);
    a.status = &ctx->scratch->status;
    a.n_seq = cache->n_seq;
    a.max_ctx = cache->max_ctx;
    a.n_kv = cache->n_kv_head;
    a.keep = keep;
    a.n_sink = n_sink;
    a.n_recent = n_recent;
    const int row16 = cache->head_dim * dtype_size(cache->dtype) / 16;   // 4 .. 64: a power of two
    while ((1 << a.shift) < row16) ++a.shift;
    DeviceGuard guard(ctx->device);
    if (!guard.ok()) return lalb_fail(ctx, LALB_ERR_CUDA, "kv_evict: device %d", ctx->device);
    // CTAs per (sequence, KV head): while each still has kRowsPerCta rows and
    // all of them run at once (one of 1024 threads on an SM).  A call of 16
    // (sequence, KV head) with 32768 rows each took 53 / 39 / 33 / 56 us with
    // 1 / 2 / 4 / 8 (clusters of 8 whole SMs do not all fit at once), with 8192
    // rows 26 / 27 / 27 / 51, with 2048 rows 17 / 21 / 23 / 44.
    int size = 1;
    while (size < kMaxCluster && cache->max_ctx / (2 * size) >= kRowsPerCta && bg * 2 * size <= ctx->sm_count)
        size *= 2;
    // a CTA's rows at most: the chunk the kernel computes for max_ctx
    const size_t key_bytes = ((((size_t)cache->max_ctx + size - 1) / size + 31) & ~(size_t)31) * sizeof(uint32_t);
    const bool cached = key_bytes <= kKeyBytesMax;
    const void *select = size == 1 ? (cached ? (const void *)evict_select_kernel<true, false>
                                             : (const void *)evict_select_kernel<false, false>)
                                   : (cached ? (const void *)evict_select_kernel<true, true>
                                             : (const void *)evict_select_kernel<false, true>);
    if (cached)
        if (int st = lalb_set_smem_attr(ctx, select, (int)key_bytes)) return st;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(bg * size));
    cfg.blockDim = dim3(kSelThreads);
    cfg.dynamicSmemBytes = cached ? key_bytes : 0;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = size;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = size > 1 ? 2 : 1;
    void *params[] = {&a};
    LALB_CUDA_TRY(ctx, cudaLaunchKernelExC(&cfg, select, params));
    LALB_LAUNCH_CHECK(ctx, "evict_select_kernel");
    const long long most = 2ll * a.list * row16;   // pieces of one (sequence, KV head)
    const long long fill = ((long long)ctx->sm_count * kMoveFill + bg - 1) / bg;
    const long long per = (most + kMoveThreads * kMoveUnroll - 1) / (kMoveThreads * kMoveUnroll);
    const dim3 grid((unsigned)std::max(1ll, std::min(fill, per)), (unsigned)bg);
    if (int st = launch_pdl(ctx, (const void *)evict_move_kernel, grid, dim3(kMoveThreads), 0,
                            (cudaStream_t)stream, {&a}))
        return st;
    LALB_LAUNCH_CHECK(ctx, "evict_move_kernel");
    return LALB_OK;
} catch (...) {   // out of host memory: no exception leaves a C entry point
    return LALB_ERR_NOMEM;
}
