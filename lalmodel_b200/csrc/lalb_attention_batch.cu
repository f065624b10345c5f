// lalb_attention_batch.cu -- one decode step of attention for a batch of
// sequences that share a prefix (lalb_attention_batch), attention_forward
// (runtime/lal_runtime.c:833-882) for many sequences at once.
//
// One CTA per (sequence, KV head), one warp per q head in turn: an online
// softmax (running maximum and sum) over the prefix rows and the sequence's
// own, fp32 throughout.
#include <math.h>

#include <algorithm>

#include "lalb_batch.cuh"

using namespace lalb;

namespace {

constexpr int kAbWarps = 8;

struct AbArgs {
    const void *q, *pk, *pv, *k, *v;
    const int *lens;
    float *row_weight;
    float2 *stat;                // [n_seq][n_head] (max, 1 / sum)
    void *out;
    unsigned int *status;
    long long q_stride;
    int n_seq, n_head, n_kv, max_ctx, prefix, add_weights;
    float scale, decay;
};

template <class T, int HD>
__device__ __forceinline__ float ab_score(const float (&q)[HD / 32], const T *row, int lane) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) s = fmaf(q[i], to_f32<T>(row[lane + 32 * i]), s);
    return warp_sum(s);
}

template <class T, int HD>
__global__ void __launch_bounds__(32 * kAbWarps) attention_batch_kernel(const AbArgs a) {
    __shared__ float2 stat[1024];
    const int g = blockIdx.x, b = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group = a.n_head / a.n_kv;
    int n = a.lens[b];
    if (n < 0 || n > a.max_ctx) {
        if (threadIdx.x == 0) atomicOr(a.status, LALB_STATUS_BAD_POSITION);
        n = 0;
    }
    const size_t kvr = (size_t)a.n_kv * HD;
    const T *pk = static_cast<const T *>(a.pk), *pv = static_cast<const T *>(a.pv);
    const T *k = static_cast<const T *>(a.k) + (size_t)b * a.max_ctx * kvr;
    const T *v = static_cast<const T *>(a.v) + (size_t)b * a.max_ctx * kvr;
    for (int hh = warp; hh < group; hh += kAbWarps) {
        const int h = g * group + hh;
        const T *qp = static_cast<const T *>(a.q) + (size_t)b * a.q_stride + (size_t)h * HD;
        float q[HD / 32], acc[HD / 32];
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) {
            q[i] = to_f32<T>(qp[lane + 32 * i]) * a.scale;
            acc[i] = 0.0f;
        }
        float m = -INFINITY, l = 0.0f;
        for (int j = 0; j < a.prefix + n; ++j) {
            const size_t off = (size_t)(j < a.prefix ? j : j - a.prefix) * kvr + (size_t)g * HD;
            const float s = ab_score<T, HD>(q, (j < a.prefix ? pk : k) + off, lane);
            const T *vr = (j < a.prefix ? pv : v) + off;
            const float mn = fmaxf(m, s), c = expf(m - mn), p = expf(s - mn);
            m = mn;
            l = fmaf(l, c, p);
#pragma unroll
            for (int i = 0; i < HD / 32; ++i) acc[i] = fmaf(acc[i], c, p * to_f32<T>(vr[lane + 32 * i]));
        }
        T *o = static_cast<T *>(a.out) + (size_t)b * a.n_head * HD + (size_t)h * HD;
        const float inv = l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) o[lane + 32 * i] = from_f32<T>(acc[i] * inv);
        if (lane == 0 && hh < 1024) stat[hh] = make_float2(m, inv);
    }
    if (!a.add_weights) return;
    __syncthreads();
    for (int j = warp; j < n; j += kAbWarps) {
        float w = 0.0f;
        for (int hh = 0; hh < group; ++hh) {
            const T *qp = static_cast<const T *>(a.q) + (size_t)b * a.q_stride + (size_t)(g * group + hh) * HD;
            float q[HD / 32];
#pragma unroll
            for (int i = 0; i < HD / 32; ++i) q[i] = to_f32<T>(qp[lane + 32 * i]) * a.scale;
            w += expf(ab_score<T, HD>(q, k + (size_t)j * kvr + (size_t)g * HD, lane) - stat[hh].x) * stat[hh].y;
        }
        if (lane == 0) {
            float *r = a.row_weight + ((size_t)b * a.n_kv + g) * a.max_ctx + j;
            *r = a.decay == 0.0f ? w : fmaf(a.decay, *r, w);
        }
    }
}

template <class T>
const void *ab_kernel(int hd) {
    switch (hd) {
        case 32: return (const void *)attention_batch_kernel<T, 32>;
        case 64: return (const void *)attention_batch_kernel<T, 64>;
        case 128: return (const void *)attention_batch_kernel<T, 128>;
        default: return (const void *)attention_batch_kernel<T, 256>;
    }
}

// Shapes, without pointers.
int ab_shape(const lalb_kv_batch *c, const lalb_attn_batch *p) {
    if (int st = kv_batch_shape(c)) return st;
    if (!p || p->prefix_len < 0) return LALB_ERR_INVALID;
    if (int st = lalb_attention_check(p->n_head, c->n_kv_head, c->head_dim)) return st;
    if (p->n_head / c->n_kv_head > 1024 || (long long)p->n_head * c->head_dim > (1 << 24) || c->n_seq > 65535)
        return LALB_ERR_UNSUPPORTED;
    return LALB_OK;
}

}  // namespace

extern "C" int lalb_attention_batch_ws_bytes(const lalb_kv_batch *cache, const lalb_attn_batch *attn,
                                             size_t *bytes) {
    if (!bytes) return LALB_ERR_INVALID;
    if (int st = ab_shape(cache, attn)) return st;
    *bytes = 256;
    return LALB_OK;
}

extern "C" int lalb_attention_batch(lalb_ctx *ctx, const lalb_kv_batch *cache, const lalb_attn_batch *attn,
                                    const void *q, long long q_stride, const int32_t *lens, void *ws, void *out,
                                    lalb_stream stream) try {
    if (!ctx) return LALB_ERR_INVALID;
    if (!cache || !attn || !q || !lens || !ws || !out)
        return lalb_fail(ctx, LALB_ERR_INVALID, "attention_batch: null pointer");
    if (int st = kv_batch_check(ctx, cache, "attention_batch")) return st;
    if (int st = ab_shape(cache, attn))
        return lalb_fail(ctx, st, "attention_batch: n_head %d over %d KV heads (at most 1024 each), prefix_len %d",
                         attn->n_head, cache->n_kv_head, attn->prefix_len);
    const int es = dtype_size(cache->dtype);
    if (attn->prefix_len > 0 && (!attn->prefix_k || !attn->prefix_v ||
                                 (((uintptr_t)attn->prefix_k | (uintptr_t)attn->prefix_v) & 15u)))
        return lalb_fail(ctx, LALB_ERR_INVALID, "attention_batch: prefix_k and prefix_v must be 16-byte aligned");
    if (q_stride < (long long)attn->n_head * cache->head_dim || q_stride * es % 16 || ((uintptr_t)q & 15u) ||
        ((uintptr_t)out & 15u) || ((uintptr_t)lens & 3u) || ((uintptr_t)ws & 255u))
        return lalb_fail(ctx, LALB_ERR_INVALID, "attention_batch: q_stride %lld, or a misaligned buffer", q_stride);
    if (!std::isfinite(attn->scale) || (attn->add_weights && !std::isfinite(attn->decay)))
        return lalb_fail(ctx, LALB_ERR_INVALID, "attention_batch: scale and decay must be finite");
    if (attn->add_weights && !cache->row_weight)
        return lalb_fail(ctx, LALB_ERR_INVALID, "attention_batch: add_weights needs the cache's row_weight");
    AbArgs a = {};
    a.q = q;
    a.pk = attn->prefix_k;
    a.pv = attn->prefix_v;
    a.k = cache->k;
    a.v = cache->v;
    a.lens = lens;
    a.row_weight = cache->row_weight;
    a.out = out;
    a.status = &ctx->scratch->status;
    a.q_stride = q_stride;
    a.n_seq = cache->n_seq;
    a.n_head = attn->n_head;
    a.n_kv = cache->n_kv_head;
    a.max_ctx = cache->max_ctx;
    a.prefix = attn->prefix_len;
    a.add_weights = attn->add_weights;
    a.scale = attn->scale == 0.0f ? (float)(1.0 / sqrt((double)cache->head_dim)) : attn->scale;
    a.decay = attn->decay;
    DeviceGuard guard(ctx->device);
    if (!guard.ok()) return lalb_fail(ctx, LALB_ERR_CUDA, "attention_batch: device %d", ctx->device);
    const void *fn = cache->dtype == LALB_DT_F32   ? ab_kernel<float>(cache->head_dim)
                     : cache->dtype == LALB_DT_F16 ? ab_kernel<__half>(cache->head_dim)
                                                   : ab_kernel<__nv_bfloat16>(cache->head_dim);
    void *params[] = {&a};
    LALB_CUDA_TRY(ctx, cudaLaunchKernel(fn, dim3(cache->n_kv_head, cache->n_seq), dim3(32 * kAbWarps), params, 0,
                                        (cudaStream_t)stream));
    return LALB_OK;
} catch (...) {   // out of host memory: no exception leaves a C entry point
    return LALB_ERR_NOMEM;
}
