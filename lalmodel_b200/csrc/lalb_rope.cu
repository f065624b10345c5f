// lalb_rope.cu -- rotary positions for T tokens, straight into the cache of
// a batch of sequences (lalb_rope_append): apply_rope
// (runtime/lal_runtime.c:137-153) with both pair layouts, a rotated part of
// the head and the two ways of stretching a context.
//
// Every pair (x0, x1) of a q or k head becomes m (x0 c - x1 s, x0 s + x1 c),
// c and s the cosine and sine of pos * f_d.  The frequencies come from the
// host in turns (f_d / 2 pi, double): pos * f_d / 2 pi loses its whole turns
// in double, where they are exact, and the remainder r in [-1/2, 1/2] goes
// on in fp32 as hi + lo, sincospi(2 hi) corrected to first order by lo.  A
// plain fp32 angle would be off by 2^-24 pos: 1e-2 at position 2^17.
//
// Memory bound: 4 + 2 or 4 + 4 bytes per element, no reuse but the angles,
// which the heads of a token share through shared memory (rot_dim / 2 of
// them per token; computing them per head would cost more instructions than
// the rotation).  A CTA takes kTok tokens or, when the call has fewer tokens
// than the GPU has SMs, a part of the heads of one.
#include <math.h>

#include <algorithm>

#include "lalb_batch.cuh"

using namespace lalb;

namespace {

constexpr int kRopeThreads = 256;
constexpr int kMaxPairs = 128;   // head_dim 256, all of it rotated
constexpr int kTok = 2;          // tokens per CTA of a long call

struct RopeArgs {
    const void *qkv;
    long long stride;            // elements between tokens
    const int *positions, *slots;
    void *q_out, *k, *v;
    int *row_pos;
    float *row_weight;
    unsigned int *status;
    int T, n_head, n_kv, hd, rot, layout, max_ctx, n_rows;
    float mscale;
    double turns[kMaxPairs];     // f_d / 2 pi
};

// (cos, sin) of pos * 2 pi * turns, times m.
__device__ __forceinline__ float2 rope_angle(int pos, double turns, float m) {
    double t = (double)pos * turns;
    t = 2.0 * (t - rint(t));                    // the angle in units of pi, [-1, 1]
    const float hi = (float)t;
    const float lo = (float)((t - (double)hi) * 3.14159265358979323846);
    float s, c;
    sincospif(hi, &s, &c);
    return make_float2(m * fmaf(-s, lo, c), m * fmaf(c, lo, s));
}

// One unit of work is 8 elements of a head: in the HALF layout 4 pairs' first
// and 4 pairs' second elements, else 8 neighbours.
template <class TI, class TO>
__global__ void __launch_bounds__(kRopeThreads) rope_append_kernel(const __grid_constant__ RopeArgs a) {
    __shared__ float2 cs[kTok][kMaxPairs];
    // gridDim.y > 1: one token, its units split over the CTAs
    const int t0 = gridDim.y > 1 ? blockIdx.x : blockIdx.x * kTok;
    const int nt = gridDim.y > 1 ? 1 : min(kTok, a.T - t0);
    const int pairs = a.rot >> 1;
    pdl_wait();                 // qkv is the matmul's output
    pdl_launch_dependents();
    for (int i = threadIdx.x; i < nt * pairs; i += kRopeThreads)
        cs[i / pairs][i % pairs] = rope_angle(__ldg(a.positions + t0 + i / pairs), a.turns[i % pairs], a.mscale);
    __syncthreads();
    const TI *qkv = static_cast<const TI *>(a.qkv);
    const int per_head = a.hd >> 3;
    const int heads = a.n_head + (a.slots ? 2 * a.n_kv : 0);
    const int units = heads * per_head;
    const int step = kRopeThreads * gridDim.y;
    for (int i = blockIdx.y * kRopeThreads + threadIdx.x; i < nt * units; i += step) {
        const int tt = i / units, u = i % units, t = t0 + tt;
        const int h = u / per_head, e = u % per_head;
        const bool is_v = h >= a.n_head + a.n_kv;
        TO *dst;
        if (h < a.n_head) {
            dst = static_cast<TO *>(a.q_out) + (size_t)t * a.n_head * a.hd + (size_t)h * a.hd;
        } else {
            const int slot = __ldg(a.slots + t);
            const int g = is_v ? h - a.n_head - a.n_kv : h - a.n_head;
            if (slot < 0) continue;
            if (slot >= a.n_rows) {
                if (e == 0) atomicOr(a.status, LALB_STATUS_BAD_POSITION);
                continue;
            }
            dst = static_cast<TO *>(is_v ? a.v : a.k) + ((size_t)slot * a.n_kv + g) * a.hd;
            if (!is_v && e == 0) {
                const int b = slot / a.max_ctx;
                const size_t m = ((size_t)b * a.n_kv + g) * a.max_ctx + (slot - b * a.max_ctx);
                if (a.row_pos) a.row_pos[m] = __ldg(a.positions + t);
                if (a.row_weight) a.row_weight[m] = 0.0f;
            }
        }
        const TI *src = qkv + (size_t)t * a.stride + (size_t)h * a.hd;
        const int half_units = a.rot >> 3;   // HALF: units that hold 4 pairs each
        float x[4], y[4];
        int d0, d1;
        if (a.layout == LALB_ROPE_HALF && e < half_units) {
            d0 = 4 * e;
            d1 = d0 + pairs;
        } else {
            d0 = 8 * e;
            d1 = d0 + 4;
        }
        load4<TI>(src + d0, x);
        load4<TI>(src + d1, y);
        if (!is_v && 8 * e < a.rot) {
            if (a.layout == LALB_ROPE_HALF) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 w = cs[tt][d0 + j];
                    const float p = x[j], q = y[j];
                    x[j] = fmaf(p, w.x, -(q * w.y));
                    y[j] = fmaf(p, w.y, q * w.x);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; j += 2) {
                    const float2 w0 = cs[tt][4 * e + (j >> 1)], w1 = cs[tt][4 * e + 2 + (j >> 1)];
                    const float p = x[j], q = x[j + 1], r = y[j], s = y[j + 1];
                    x[j] = fmaf(p, w0.x, -(q * w0.y));
                    x[j + 1] = fmaf(p, w0.y, q * w0.x);
                    y[j] = fmaf(r, w1.x, -(s * w1.y));
                    y[j + 1] = fmaf(r, w1.y, s * w1.x);
                }
            }
        }
        store4<TO>(dst + d0, x);
        store4<TO>(dst + d1, y);
    }
}

// f_d / 2 pi of every pair; false on a parameter that has no meaning.
bool rope_turns(const lalb_rope *r, int rot, double *turns) {
    const double two_pi = 6.283185307179586476925;
    const double theta = r->theta == 0.0f ? 10000.0 : (double)r->theta;
    if (!(theta > 1.0) || std::isinf(theta)) return false;
    if (r->scaling != LALB_ROPE_UNSCALED && r->scaling != LALB_ROPE_LINEAR && r->scaling != LALB_ROPE_PARTS)
        return false;
    if (r->scaling != LALB_ROPE_UNSCALED && !(r->factor > 0.0f && std::isfinite(r->factor))) return false;
    if (r->scaling == LALB_ROPE_PARTS &&
        !(r->orig_ctx > 0.0f && std::isfinite(r->orig_ctx) && std::isfinite(r->turns_fast) &&
          std::isfinite(r->turns_slow) && r->turns_fast > r->turns_slow))
        return false;
    // eight pow calls at most take as long as the rest of the call on the host:
    // between them the frequencies go on by multiplication (15 roundings, 2^-49)
    const double step = pow(theta, -2.0 / rot);
    double power = 1.0;
    for (int d = 0; d < rot / 2; ++d) {
        power = d % 16 ? power * step : pow(theta, -2.0 * d / rot);
        double f = power;
        if (r->scaling == LALB_ROPE_LINEAR) f /= (double)r->factor;
        if (r->scaling == LALB_ROPE_PARTS) {
            const double t = (double)r->orig_ctx * f / two_pi;
            const double lo = r->turns_slow, hi = r->turns_fast;
            const double g = std::min(1.0, std::max(0.0, (t - lo) / (hi - lo)));
            f *= g + (1.0 - g) / (double)r->factor;
        }
        turns[d] = f / two_pi;
    }
    return true;
}

const void *rope_kernel(int in, int out) {
    if (out == LALB_DT_F32) return (const void *)rope_append_kernel<float, float>;
    if (out == LALB_DT_F16)
        return in == LALB_DT_F32 ? (const void *)rope_append_kernel<float, __half>
                                 : (const void *)rope_append_kernel<__half, __half>;
    return in == LALB_DT_F32 ? (const void *)rope_append_kernel<float, __nv_bfloat16>
                             : (const void *)rope_append_kernel<__nv_bfloat16, __nv_bfloat16>;
}

}  // namespace

extern "C" int lalb_rope_append(lalb_ctx *ctx, const lalb_rope *rope, const lalb_kv_batch *cache, int n_head,
                                const void *qkv, int qkv_dtype, long long qkv_stride, int T,
                                const int32_t *positions, const int32_t *slots, void *q_out,
                                lalb_stream stream) try {
    if (!ctx) return LALB_ERR_INVALID;
    if (!rope || !cache || !qkv || !positions || !q_out)
        return lalb_fail(ctx, LALB_ERR_INVALID, "rope_append: null pointer");
    if (int st = kv_batch_check(ctx, cache, "rope_append")) return st;
    if (int st = lalb_attention_check(n_head, cache->n_kv_head, cache->head_dim))
        return lalb_fail(ctx, st, "rope_append: n_head %d over %d KV heads", n_head, cache->n_kv_head);
    if (T < 0) return lalb_fail(ctx, LALB_ERR_INVALID, "rope_append: T %d", T);
    if (qkv_dtype != LALB_DT_F32 && qkv_dtype != cache->dtype)
        return lalb_fail(ctx, LALB_ERR_UNSUPPORTED, "rope_append: qkv is F32 or of the cache's type");
    const long long row = ((long long)n_head + (slots ? 2ll * cache->n_kv_head : 0)) * cache->head_dim;
    if (row > (1 << 24)) return lalb_fail(ctx, LALB_ERR_UNSUPPORTED, "rope_append: %lld elements a token", row);
    if (qkv_stride < row || qkv_stride * dtype_size(qkv_dtype) % 16 || ((uintptr_t)qkv & 15u) ||
        ((uintptr_t)q_out & 15u) || ((uintptr_t)positions & 3u) || ((uintptr_t)slots & 3u))
        return lalb_fail(ctx, LALB_ERR_INVALID, "rope_append: qkv_stride %lld, or a misaligned buffer", qkv_stride);
    RopeArgs a = {};
    a.rot = rope->rot_dim ? rope->rot_dim : cache->head_dim;
    if (a.rot < 0 || a.rot > cache->head_dim || a.rot % 8)
        return lalb_fail(ctx, LALB_ERR_UNSUPPORTED, "rope_append: rot_dim %d (a multiple of 8 up to head_dim)",
                         rope->rot_dim);
    if (rope->layout != LALB_ROPE_HALF && rope->layout != LALB_ROPE_INTERLEAVED)
        return lalb_fail(ctx, LALB_ERR_INVALID, "rope_append: layout %d", rope->layout);
    if (!std::isfinite(rope->mscale) || !rope_turns(rope, a.rot, a.turns))
        return lalb_fail(ctx, LALB_ERR_INVALID, "rope_append: theta, scaling or mscale");
    if (T == 0) return LALB_OK;
    a.qkv = qkv;
    a.stride = qkv_stride;
    a.positions = positions;
    a.slots = slots;
    a.q_out = q_out;
    a.k = cache->k;
    a.v = cache->v;
    a.row_pos = cache->row_pos;
    a.row_weight = cache->row_weight;
    a.status = &ctx->scratch->status;
    a.T = T;
    a.n_head = n_head;
    a.n_kv = cache->n_kv_head;
    a.hd = cache->head_dim;
    a.layout = rope->layout;
    a.max_ctx = cache->max_ctx;
    a.n_rows = cache->n_seq * cache->max_ctx;
    a.mscale = rope->mscale == 0.0f ? 1.0f : rope->mscale;
    DeviceGuard guard(ctx->device);
    if (!guard.ok()) return lalb_fail(ctx, LALB_ERR_CUDA, "rope_append: device %d", ctx->device);
    // fewer tokens than SMs: a token's units over as many CTAs as give every thread one
    const int units = (int)(row / 8);
    dim3 grid((T + kTok - 1) / kTok, 1);
    if (T <= ctx->sm_count) grid = dim3(T, std::min(64, (units + kRopeThreads - 1) / kRopeThreads));
    if (grid.y == 1) grid.x = (T + kTok - 1) / kTok;
    if (int st = launch_pdl(ctx, rope_kernel(qkv_dtype, cache->dtype), grid, dim3(kRopeThreads), 0,
                            (cudaStream_t)stream, {&a}))
        return st;
    LALB_LAUNCH_CHECK(ctx, "rope_append_kernel");
    return LALB_OK;
} catch (...) {   // out of host memory: no exception leaves a C entry point
    return LALB_ERR_NOMEM;
}
