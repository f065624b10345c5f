// lalb_batch.cuh -- what the batched-decode operators (lalb_rope.cu,
// lalb_attention_batch.cu, lalb_kv_evict.cu) share: the check of a
// lalb_kv_batch, element types, and a guard that makes the context's device
// current for the length of a call.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "lalb_internal.cuh"

int lalb_attention_check(int n_head, int n_kv, int hd);   // lalb_attention.cu

namespace lalb {

// The calling thread's device is the context's while this lives, and the one
// it was before afterwards.
class DeviceGuard {
  public:
    explicit DeviceGuard(int device) {
        ok_ = cudaGetDevice(&old_) == cudaSuccess && (old_ == device || cudaSetDevice(device) == cudaSuccess);
        changed_ = ok_ && old_ != device;
    }
    ~DeviceGuard() {
        if (changed_) cudaSetDevice(old_);
    }
    bool ok() const { return ok_; }

  private:
    int old_ = 0;
    bool ok_ = false, changed_ = false;
};

inline int dtype_size(int dtype) {
    return dtype == LALB_DT_F32 ? 4 : dtype == LALB_DT_F16 || dtype == LALB_DT_BF16 ? 2 : 0;
}

// Shape and type of a cache (no pointers): LALB_OK or the reason's status.
inline int kv_batch_shape(const lalb_kv_batch *c) {
    if (!c || c->n_seq <= 0 || c->max_ctx <= 0 || c->n_kv_head <= 0) return LALB_ERR_INVALID;
    // row numbers, and those of a tile that begins at the last row, fit 31 bits
    if ((long long)c->n_seq * c->max_ctx > 0x7fffff00ll) return LALB_ERR_UNSUPPORTED;
    if (!dtype_size(c->dtype)) return LALB_ERR_UNSUPPORTED;
    if (int st = lalb_attention_check(c->n_kv_head, c->n_kv_head, c->head_dim)) return st;
    // a row's elements, and so every index within one, fit 31 bits
    if ((long long)c->n_kv_head * c->head_dim > (1 << 24)) return LALB_ERR_UNSUPPORTED;
    return LALB_OK;
}

inline int kv_batch_check(lalb_ctx *ctx, const lalb_kv_batch *c, const char *who) {
    if (int st = kv_batch_shape(c))
        return lalb_fail(ctx, st, "%s: cache (dtype F32, F16 or BF16; head_dim 32, 64, 128 or 256; positive "
                                  "sizes, n_seq*max_ctx <= 2^31 - 256)", who);
    if (!c->k || !c->v || (((uintptr_t)c->k | (uintptr_t)c->v) & 15u))
        return lalb_fail(ctx, LALB_ERR_INVALID, "%s: k and v must be 16-byte aligned device buffers", who);
    if ((((uintptr_t)c->row_pos | (uintptr_t)c->row_weight) & 3u))
        return lalb_fail(ctx, LALB_ERR_INVALID, "%s: row_pos and row_weight must be 4-byte aligned", who);
    return LALB_OK;
}

// ---- elements ----------------------------------------------------------------
template <class T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Four consecutive elements, aligned to their own size.
template <class T>
__device__ __forceinline__ void load4(const T *p, float (&v)[4]) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = *reinterpret_cast<const float4 *>(p);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    } else {
        const uint2 a = *reinterpret_cast<const uint2 *>(p);
        const T *h = reinterpret_cast<const T *>(&a);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = to_f32<T>(h[i]);
    }
}

template <class T>
__device__ __forceinline__ void store4(T *p, const float (&v)[4]) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
        __align__(8) T h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = from_f32<T>(v[i]);
        *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<const uint2 *>(h);
    }
}

}  // namespace lalb
