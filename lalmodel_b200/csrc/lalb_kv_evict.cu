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
// evict_select_kernel, one CTA per (sequence, KV head): a 32-bit key per row
// (protected rows the largest, weights in their order, NaN 0) kept in shared
// memory, the keep-th largest key by three counting passes of 11, 11 and 10
// bits, then the two lists by ballots: each warp owns a run of neighbouring
// rows, so that ranks follow the row order.  It is bound by latency: its
// passes over at most a few hundred KB in one SM.  evict_move_kernel copies
// the rows and is memory bound: 4 head_dim elements per moved row.
#include <algorithm>

#include "lalb_batch.cuh"

using namespace lalb;

namespace {

constexpr int kSelThreads = 1024;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kBins = 2048;
constexpr size_t kKeyBytesMax = 200 * 1024;   // keys of up to 51200 rows stay in shared memory
constexpr int kMoveThreads = 256;
constexpr int kMoveUnroll = 4;

struct EvictArgs {
    int *lens;
    int *row_pos;
    float *row_weight;
    uint8_t *k, *v;
    int *count;            // [n_seq * n_kv] rows that move
    int *dst, *src;        // [n_seq * n_kv][list] places below keep, rows above it
    unsigned int *status;
    int n_seq, max_ctx, n_kv, keep, n_sink, n_recent, list;
    int row16;             // 16-byte pieces of one row of one KV head
};

__device__ __forceinline__ uint32_t evict_key(const EvictArgs &a, size_t m, int newest) {
    const int p = __ldcg(a.row_pos + m);
    const float w = __ldcg(a.row_weight + m);
    if (p < a.n_sink || (long long)p > (long long)newest - a.n_recent) return 0xffffffffu;
    if (w != w) return 0u;
    return ordered_key(w + 0.0f);   // -0 counts as 0
}

// kCached: every key in shared memory; otherwise each pass forms it again
// from row_pos and row_weight (which change only after the last pass).
template <bool kCached>
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const EvictArgs a) {
    extern __shared__ uint32_t keys[];
    __shared__ uint32_t hist[kBins];
    __shared__ int wsum[3][kSelWarps];
    __shared__ int newest_s;
    __shared__ uint32_t digit_s, above_s;
    const int bg = blockIdx.x, b = bg / a.n_kv;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_wait();
    pdl_launch_dependents();
    const int n = a.lens[b];
    if (n < 0 || n > a.max_ctx) {
        if (tid == 0) {
            a.count[bg] = 0;
            atomicOr(a.status, LALB_STATUS_BAD_POSITION);
        }
        return;
    }
    if (n <= a.keep) {
        if (tid == 0) a.count[bg] = 0;
        return;
    }
    const size_t base = (size_t)bg * a.max_ctx;

    // ---- the newest position ------------------------------------------------------
    int newest = INT_MIN;
    for (int i = tid; i < n; i += kSelThreads) newest = max(newest, __ldcg(a.row_pos + base + i));
    newest = __reduce_max_sync(0xffffffffu, newest);
    if (lane == 0) wsum[0][warp] = newest;
    __syncthreads();
    if (warp == 0) {
        newest = __reduce_max_sync(0xffffffffu, wsum[0][lane]);
        if (lane == 0) newest_s = newest;
    }
    __syncthreads();
    newest = newest_s;

    auto key_of = [&](int i) -> uint32_t { return kCached ? keys[i] : evict_key(a, base + i, newest); };

    // ---- the keep-th largest key ----------------------------------------------------
    uint32_t prefix = 0, mask = 0;
    int need = a.keep;          // rows still to take among those that match the prefix
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const int bins = pass == 2 ? 1024 : 2048;
        for (int i = tid; i < bins; i += kSelThreads) hist[i] = 0;
        __syncthreads();
        for (int i0 = warp * 32; i0 < n; i0 += kSelThreads) {
            const int i = i0 + lane;
            uint32_t key = 0;
            bool in = i < n;
            if (in) {
                key = (kCached && pass > 0) ? keys[i] : evict_key(a, base + i, newest);
                if (kCached && pass == 0) keys[i] = key;
                in = (key & mask) == prefix;
            }
            // one addition per distinct digit of the warp: the weights' leading
            // bits agree for most rows
            const uint32_t d = in ? (key >> shift) & (bins - 1) : 0xffffffffu;
            const uint32_t same = __match_any_sync(0xffffffffu, d);
            if (in && lane == __ffs(same) - 1) atomicAdd(&hist[d], (uint32_t)__popc(same));
        }
        __syncthreads();
        // the digit whose rows straddle `need`, counted from the largest
        const int per = bins / kSelThreads;
        const int hi = bins - 1 - tid * per;
        uint32_t own = hist[hi];
        if (per == 2) own += hist[hi - 1];
        uint32_t incl = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t x = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += x;
        }
        if (lane == 31) wsum[0][warp] = (int)incl;
        __syncthreads();
        uint32_t before = incl - own;
        for (int w = 0; w < warp; ++w) before += (uint32_t)wsum[0][w];
        if (before < (uint32_t)need && (uint32_t)need <= before + own) {
            const uint32_t top = hist[hi];
            const bool second = per == 2 && before + top < (uint32_t)need;
            digit_s = second ? hi - 1 : hi;
            above_s = second ? before + top : before;
        }
        __syncthreads();
        prefix |= digit_s << shift;
        mask |= (uint32_t)(bins - 1) << shift;
        need -= (int)above_s;
    }

    // ---- the lists: warp w owns rows [r0, r1) -----------------------------------------
    const int run = ((n + kSelWarps - 1) / kSelWarps + 31) & ~31;
    const int r0 = min(n, warp * run), r1 = min(n, r0 + run);
    auto scan = [&](int which) -> int {   // sum of the earlier warps' wsum[which]
        const int x = lane < warp ? wsum[which][lane] : 0;
        return __reduce_add_sync(0xffffffffu, x);
    };
    int ties = 0;
    for (int i0 = r0; i0 < r1; i0 += 32) {
        const int i = i0 + lane;
        ties += __popc(__ballot_sync(0xffffffffu, i < r1 && key_of(i) == prefix));
    }
    if (lane == 0) wsum[0][warp] = ties;
    __syncthreads();
    const int ties0 = scan(0);
    // pass 0 counts the warp's places and movers, pass 1 writes them at their ranks
    int place = 0, mover = 0;
    const uint32_t lower = (1u << lane) - 1;
    for (int pass = 0; pass < 2; ++pass) {
        int tie = ties0;
        for (int i0 = r0; i0 < r1; i0 += 32) {
            const int i = i0 + lane;
            const bool live = i < r1;
            const uint32_t key = live ? key_of(i) : 0u;
            const uint32_t eq = __ballot_sync(0xffffffffu, live && key == prefix);
            const bool kept = live && (key > prefix || (key == prefix && tie + __popc(eq & lower) < need));
            tie += __popc(eq);
            const bool is_place = live && !kept && i < a.keep, is_mover = kept && i >= a.keep;
            const uint32_t bp = __ballot_sync(0xffffffffu, is_place), bm = __ballot_sync(0xffffffffu, is_mover);
            if (pass == 1) {
                if (is_place) a.dst[(size_t)bg * a.list + place + __popc(bp & lower)] = i;
                if (is_mover) a.src[(size_t)bg * a.list + mover + __popc(bm & lower)] = i;
            }
            place += __popc(bp);
            mover += __popc(bm);
        }
        if (pass == 0) {
            if (lane == 0) {
                wsum[1][warp] = place;
                wsum[2][warp] = mover;
            }
            __syncthreads();
            place = scan(1);
            mover = scan(2);
        }
    }
    // as many places as movers: exactly `keep` rows are kept
    int moved = 0;
    for (int w = 0; w < kSelWarps; ++w) moved += wsum[1][w];
    if (tid == 0) a.count[bg] = moved;
    __syncthreads();
    for (int i = tid; i < moved; i += kSelThreads) {
        const size_t d = base + __ldcg(a.dst + (size_t)bg * a.list + i);
        const size_t s = base + __ldcg(a.src + (size_t)bg * a.list + i);
        a.row_pos[d] = __ldcg(a.row_pos + s);
        a.row_weight[d] = __ldcg(a.row_weight + s);
    }
    __syncthreads();
    for (int i = a.keep + tid; i < n; i += kSelThreads) a.row_weight[base + i] = 0.0f;
}

__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const EvictArgs a) {
    const int bg = blockIdx.y, b = bg / a.n_kv, g = bg % a.n_kv;
    pdl_wait();
    pdl_launch_dependents();
    const int moved = a.count[bg];
    if (g == 0 && blockIdx.x == 0 && threadIdx.x == 0) {
        const int n = a.lens[b];
        if (n > a.keep && n <= a.max_ctx) a.lens[b] = a.keep;
    }
    const int *dst = a.dst + (size_t)bg * a.list, *src = a.src + (size_t)bg * a.list;
    const size_t rows0 = (size_t)b * a.max_ctx;
    // piece p: 16 bytes of K (even rows of pieces) or V of move p / (2 row16)
    const long long pieces = (long long)moved * 2 * a.row16;
    const long long stride = (long long)gridDim.x * kMoveThreads;
    for (long long p0 = (long long)blockIdx.x * kMoveThreads + threadIdx.x; p0 < pieces;
         p0 += kMoveUnroll * stride) {
        uint4 x[kMoveUnroll];
        uint4 *to[kMoveUnroll];
#pragma unroll
        for (int u = 0; u < kMoveUnroll; ++u) {
            const long long p = p0 + u * stride;
            to[u] = nullptr;
            if (p < pieces) {
                const int row = (int)(p / a.row16), c = (int)(p % a.row16), m = row >> 1;
                uint8_t *t = (row & 1) ? a.v : a.k;
                const size_t s = (((rows0 + __ldcg(src + m)) * a.n_kv + g) * a.row16 + c) * 16;
                const size_t d = (((rows0 + __ldcg(dst + m)) * a.n_kv + g) * a.row16 + c) * 16;
                x[u] = *reinterpret_cast<const uint4 *>(t + s);
                to[u] = reinterpret_cast<uint4 *>(t + d);
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
    *bytes = up256(bg * sizeof(int)) + 2 * up256(bg * list_len(cache, keep) * sizeof(int));
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
    if (keep == cache->max_ctx) return LALB_OK;   // nothing can be longer
    EvictArgs a = {};
    a.lens = lens;
    a.row_pos = cache->row_pos;
    a.row_weight = cache->row_weight;
    a.k = static_cast<uint8_t *>(cache->k);
    a.v = static_cast<uint8_t *>(cache->v);
    a.list = list_len(cache, keep);
    uint8_t *w = static_cast<uint8_t *>(ws);
    a.count = reinterpret_cast<int *>(w);
    w += up256(bg * sizeof(int));
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
    a.row16 = cache->head_dim * dtype_size(cache->dtype) / 16;
    DeviceGuard guard(ctx->device);
    if (!guard.ok()) return lalb_fail(ctx, LALB_ERR_CUDA, "kv_evict: device %d", ctx->device);
    const size_t key_bytes = (size_t)cache->max_ctx * sizeof(uint32_t);
    const bool cached = key_bytes <= kKeyBytesMax;
    const void *select = cached ? (const void *)evict_select_kernel<true> : (const void *)evict_select_kernel<false>;
    if (cached)
        if (int st = lalb_set_smem_attr(ctx, select, (int)key_bytes)) return st;
    if (int st = launch_pdl(ctx, select, dim3((unsigned)bg), dim3(kSelThreads), cached ? key_bytes : 0,
                            (cudaStream_t)stream, {&a}))
        return st;
    LALB_LAUNCH_CHECK(ctx, "evict_select_kernel");
    const long long most = 2ll * a.list * a.row16;   // pieces of one (sequence, KV head)
    const long long fill = ((long long)ctx->sm_count * 8 + bg - 1) / bg;
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
