// Reading and writing the caller's matrices 8 elements at a time (ns_gather.cu, ns_small.cu).
#pragma once

#include <cuda_bf16.h>

#include "ns_plan.h"

namespace vb {
namespace {

template <typename T> __device__ __forceinline__ float to_f32(T x);
template <> __device__ __forceinline__ float to_f32(float x) { return x; }
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f32(float x) { return __float2half_rn(x); }

// 8 elements along one direction (`step` apart in memory); the first `count` exist, the rest read as zero
template <typename T>
__device__ __forceinline__ void load8_as(const T *p, int64_t step, int count, bool vec, float (&v)[8])
{
    if (vec && count == 8) {
        constexpr int kWords = (int)sizeof(T) * 8 / 16;
        uint4 q[kWords];
#pragma unroll
        for (int w = 0; w < kWords; ++w) q[w] = reinterpret_cast<const uint4 *>(p)[w];
        const T *e = reinterpret_cast<const T *>(q);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = to_f32(e[k]);
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = k < count ? to_f32(p[k * step]) : 0.0f;
    }
}
template <typename T>
__device__ __forceinline__ void store8_as(T *p, int64_t step, int count, bool vec, const float (&v)[8])
{
    if (vec && count == 8) {
        constexpr int kWords = (int)sizeof(T) * 8 / 16;
        uint4 q[kWords];
        T *e = reinterpret_cast<T *>(q);
#pragma unroll
        for (int k = 0; k < 8; ++k) e[k] = from_f32<T>(v[k]);
#pragma unroll
        for (int w = 0; w < kWords; ++w) reinterpret_cast<uint4 *>(p)[w] = q[w];
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k < count) p[k * step] = from_f32<T>(v[k]);
    }
}
__device__ __forceinline__ void load8(int type, const void *base, int64_t at, int64_t step, int count, bool vec, float (&v)[8])
{
    if (type == VB_DTYPE_F32) load8_as(static_cast<const float *>(base) + at, step, count, vec, v);
    else if (type == VB_DTYPE_BF16) load8_as(static_cast<const __nv_bfloat16 *>(base) + at, step, count, vec, v);
    else load8_as(static_cast<const __half *>(base) + at, step, count, vec, v);
}
__device__ __forceinline__ void store8(int type, void *base, int64_t at, int64_t step, int count, bool vec, const float (&v)[8])
{
    if (type == VB_DTYPE_F32) store8_as(static_cast<float *>(base) + at, step, count, vec, v);
    else if (type == VB_DTYPE_BF16) store8_as(static_cast<__nv_bfloat16 *>(base) + at, step, count, vec, v);
    else store8_as(static_cast<__half *>(base) + at, step, count, vec, v);
}

__device__ __forceinline__ float2 unpack_half(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2 *>(&w)); }

// 8 elements as they lie in memory (whole and aligned octets; others are read when they are asked for): loads first,
// conversions later, so that a thread has several octets on their way.
struct Raw {
    uint4 q[2];
    bool packed;
    __device__ __forceinline__ void load(int type, const void *base, int64_t at, int count, bool vec)
    {
        packed = vec && count == 8;
        if (packed) {
            const char *p = static_cast<const char *>(base) + at * (type == VB_DTYPE_F32 ? 4 : 2);
            q[0] = *reinterpret_cast<const uint4 *>(p);
            if (type == VB_DTYPE_F32) q[1] = reinterpret_cast<const uint4 *>(p)[1];
        }
    }
    __device__ __forceinline__ void get(int type, const void *base, int64_t at, int64_t step, int count, float (&v)[8]) const
    {
        if (!packed) {
            load8(type, base, at, step, count, false, v);
            return;
        }
        if (type == VB_DTYPE_F32) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                v[4 * k] = __uint_as_float(q[k].x), v[4 * k + 1] = __uint_as_float(q[k].y);
                v[4 * k + 2] = __uint_as_float(q[k].z), v[4 * k + 3] = __uint_as_float(q[k].w);
            }
        } else {
            const uint32_t h[4] = {q[0].x, q[0].y, q[0].z, q[0].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (type == VB_DTYPE_BF16) {
                    v[2 * k] = __uint_as_float(h[k] << 16);
                    v[2 * k + 1] = __uint_as_float(h[k] & 0xffff0000u);
                } else {
                    const float2 x = unpack_half(h[k]);
                    v[2 * k] = x.x, v[2 * k + 1] = x.y;
                }
            }
        }
    }
};

// along i where that is the contiguous direction and j is not
__device__ __forceinline__ bool walks_i(const NsArray &a) { return a.si == 1 && a.sj != 1; }
// U of one octet in the velocity's direction: new velocity in v, U in u.
__device__ __forceinline__ void momentum8(const NsElementwise &w, const float (&g)[8], float (&v)[8], float (&u)[8])
{
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        v[e] = fmaf(w.momentum, v[e], g[e]);
        u[e] = w.nesterov ? fmaf(w.momentum, v[e], g[e]) : v[e];
    }
}

}  // namespace
}  // namespace vb
