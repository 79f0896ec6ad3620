// Element-wise passes of Newton-Schulz on caller-owned matrices (ns_plan.cu):
//   norm    sum of squares of every matrix's U (f64 partial sums per tile, no atomics)
//   gather  U times a power of two -> the f16 working matrix; step: also v <- mu v + g
//   finish  the last iterate -> the caller's output, or  p <- p (1 - lr wd) - lr s O
// with U the input (orthogonalize) or g + mu v' / v' of the new velocity v' (step).
//
// Bound by HBM traffic.  U is needed twice (the norm is a property of the whole matrix) and is
// computed twice instead of being stored: with bf16 gradients and f32 velocities that moves 18
// bytes per element where storing an f32 U would move 20.  The planner launches norm and gather
// alternately over groups of matrices that fit the L2 cache, so the second read mostly stays on chip.
//
// The norm is accumulated in f64: squares of the whole f32 range neither overflow nor vanish.  The
// power of two brings the working matrix's norm into (2^12, 2^13]: inputs with 11 significand bits or
// fewer enter the iteration unrounded; the remaining factor is applied by the first products.
//
// A tile is 64 x 128 of the working matrix (short side x long side).  Where an array's contiguous
// direction is the tile's other one, the tile is turned in shared memory, so global accesses run
// along memory for row-major and transposed arrays alike (any other strides: along j, element by element).
#include "ns_elementwise.h"

namespace vb {

namespace {

constexpr int kThreads = 256;
constexpr int kPitch = kNsTileJ + 1;

// The tile's pass `k` (0..3) in one direction: this thread's 8 elements start at (i, j).
struct Octet {
    int i, j;
};
__device__ __forceinline__ Octet octet_along_j(int k)
{
    return {k * 16 + (int)(threadIdx.x >> 4), (int)(threadIdx.x & 15) * 8};
}
__device__ __forceinline__ Octet octet_along_i(int k)
{
    return {(int)(threadIdx.x & 7) * 8, k * 32 + (int)(threadIdx.x >> 3)};
}
__device__ __forceinline__ Octet octet(bool along_i, int k) { return along_i ? octet_along_i(k) : octet_along_j(k); }

// Where the tile lies and which direction an array is walked in.
struct TileView {
    int i0, j0, n, m;
    __device__ __forceinline__ int count(bool along_i, Octet o) const
    {
        const int i = i0 + o.i, j = j0 + o.j;
        if (i >= n || j >= m) return 0;
        const int left = along_i ? n - i : m - j;
        return left < 8 ? left : 8;
    }
};
__device__ __forceinline__ int64_t offset(const NsArray &a, const TileView &t, Octet o)
{
    return (int64_t)(t.i0 + o.i) * a.si + (int64_t)(t.j0 + o.j) * a.sj;
}
__device__ __forceinline__ void read8(int type, const NsArray &a, bool vec, bool along_i, const TileView &t, Octet o,
                                      float (&v)[8])
{
    load8(type, a.ptr, offset(a, t, o), along_i ? a.si : a.sj, t.count(along_i, o), vec, v);
}
__device__ __forceinline__ void write8(int type, const NsArray &a, bool vec, bool along_i, const TileView &t, Octet o,
                                       const float (&v)[8])
{
    store8(type, a.ptr, offset(a, t, o), along_i ? a.si : a.sj, t.count(along_i, o), vec, v);
}
__device__ __forceinline__ float &at(float *tile, bool along_i, Octet o, int e)
{
    return along_i ? tile[(o.i + e) * kPitch + o.j] : tile[o.i * kPitch + o.j + e];
}

__device__ __forceinline__ double block_sum(double v, double *warp_sums)
{
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
    if ((threadIdx.x & 31) == 0) warp_sums[threadIdx.x >> 5] = v;
    __syncthreads();
    double total = 0.0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) total += warp_sums[w];
    return total;
}

__device__ __forceinline__ TileView tile_view(const NsMatrixDims &d, int tile)
{
    const int per_row = d.mp / kNsTileJ, local = tile - d.tile0;
    return {(local / per_row) * kNsTileI, (local % per_row) * kNsTileJ, d.n, d.m};
}

// The gradient goes through shared memory where its direction is not the velocity's.
__device__ __forceinline__ void stage_gradient(const NsElementwise &w, const NsMatrixArg &a, const TileView &t, float *tile)
{
    const bool gi = walks_i(a.a[0]);
    for (int k = 0; k < 4; ++k) {
        const Octet o = octet(gi, k);
        float g[8];
        read8(w.types[0], a.a[0], a.direct & 1u, gi, t, o, g);
#pragma unroll
        for (int e = 0; e < 8; ++e) at(tile, gi, o, e) = g[e];
    }
    __syncthreads();
}

template <bool kStep>
__global__ void __launch_bounds__(kThreads)
ns_norm_kernel(const NsElementwise w, const __grid_constant__ NsBatchArgs b, const int32_t *__restrict__ tile_matrix)
{
    __shared__ float tile[kStep ? kNsTileI * kPitch : 1];
    __shared__ double warp_sums[kThreads / 32];
    if (*w.error != 0u) return;
    const int index = b.tile0 + (int)blockIdx.x;
    const int matrix = tile_matrix[index];
    const NsMatrixArg &a = b.m[matrix - b.first];
    if (a.live == 0u) return;
    const TileView t = tile_view(w.dims[matrix], index);
    double sum = 0.0;
    if (kStep) {
        const bool vi = walks_i(a.a[1]), turned = walks_i(a.a[0]) != vi;
        if (turned) stage_gradient(w, a, t, tile);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const Octet o = octet(vi, k);
            float g[8], v[8], u[8];
            if (turned) {
#pragma unroll
                for (int e = 0; e < 8; ++e) g[e] = at(tile, vi, o, e);
            } else {
                read8(w.types[0], a.a[0], a.direct & 1u, vi, t, o, g);
            }
            read8(w.types[1], a.a[1], a.direct & 2u, vi, t, o, v);
            momentum8(w, g, v, u);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum = fma((double)u[e], (double)u[e], sum);
        }
    } else {
        const bool along_i = walks_i(a.a[0]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const Octet o = octet(along_i, k);
            float u[8];
            read8(w.types[0], a.a[0], a.direct & 1u, along_i, t, o, u);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum = fma((double)u[e], (double)u[e], sum);
        }
    }
    sum = block_sum(sum, warp_sums);
    if (threadIdx.x == 0) w.partials[index] = sum;
}

// 8 values of the working matrix (j contiguous): one f16 plane, or the value's two
__device__ __forceinline__ void store_working(__half *x, int64_t plane, int planes, const float (&v)[8])
{
    __half h[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = __float2half_rn(v[e]);
    *reinterpret_cast<uint4 *>(x) = *reinterpret_cast<const uint4 *>(h);
    if (planes == 2) {
        __half l[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) l[e] = __float2half_rn(v[e] - __half2float(h[e]));
        *reinterpret_cast<uint4 *>(x + plane) = *reinterpret_cast<const uint4 *>(l);
    }
}

template <bool kStep>
__global__ void __launch_bounds__(kThreads)
ns_gather_kernel(const NsElementwise w, const __grid_constant__ NsBatchArgs b, const int32_t *__restrict__ tile_matrix)
{
    __shared__ float tile[kNsTileI * kPitch];
    __shared__ double warp_sums[kThreads / 32];
    if (*w.error != 0u) return;
    const int index = b.tile0 + (int)blockIdx.x;
    const int matrix = tile_matrix[index];
    const NsMatrixArg &a = b.m[matrix - b.first];
    const NsMatrixDims d = w.dims[matrix];
    if (index == d.tile0 && threadIdx.x == 0) {
        w.active[matrix] = a.live;
        w.stored[matrix] = 0u;
    }
    if (a.live == 0u) return;
    const TileView t = tile_view(d, index);

    double sum = 0.0;  // the same order in every block and call
    for (int k = threadIdx.x; k < d.n_tiles; k += kThreads) sum += w.partials[d.tile0 + k];
    const double norm = sqrt(block_sum(sum, warp_sums));
    int ex = 13;
    if (norm > 0.0 && isfinite(norm)) (void)frexp(norm, &ex);
    const int shift = 13 - ex;  // norm * 2^shift in [2^12, 2^13)
    // two factors, each a normal power of two: |shift| may pass f32's exponent range
    const float up0 = ldexpf(1.0f, shift / 2), up1 = ldexpf(1.0f, shift - shift / 2);
    if (index == d.tile0 && threadIdx.x == 0)
        // an infinite or undefined norm makes the whole result undefined, as the formula does
        w.scale[matrix] = isfinite(norm) ? (float)(ldexp(1.0, -shift) / (norm + (double)w.eps)) : nanf("");

    __half *x = w.x + d.x_off;
    const int64_t plane = (int64_t)d.np * d.mp;
    const bool ui = walks_i(a.a[kStep ? 1 : 0]);
    const bool turned = kStep && walks_i(a.a[0]) != ui;
    if (turned) stage_gradient(w, a, t, tile);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const Octet o = octet(ui, k);
        float u[8];
        if (kStep) {
            float g[8], v[8];
            if (turned) {
#pragma unroll
                for (int e = 0; e < 8; ++e) g[e] = at(tile, ui, o, e);
            } else {
                read8(w.types[0], a.a[0], a.direct & 1u, ui, t, o, g);
            }
            read8(w.types[1], a.a[1], a.direct & 2u, ui, t, o, v);
            momentum8(w, g, v, u);
            write8(w.types[1], a.a[1], a.direct & 2u, ui, t, o, v);
        } else {
            read8(w.types[0], a.a[0], a.direct & 1u, ui, t, o, u);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] = u[e] * up0 * up1;
        if (ui) {  // this thread alone read these elements of the tile
#pragma unroll
            for (int e = 0; e < 8; ++e) at(tile, true, o, e) = u[e];
        } else {
            store_working(x + (int64_t)(t.i0 + o.i) * d.mp + t.j0 + o.j, plane, w.planes, u);
        }
    }
    if (ui) {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const Octet o = octet(false, k);
            float u[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) u[e] = at(tile, false, o, e);
            store_working(x + (int64_t)(t.i0 + o.i) * d.mp + t.j0 + o.j, plane, w.planes, u);
        }
    }
}

template <bool kStep>
__global__ void __launch_bounds__(kThreads)
ns_finish_kernel(const NsElementwise w, const __grid_constant__ NsBatchArgs b, const int32_t *__restrict__ tile_matrix)
{
    __shared__ float tile[kNsTileI * kPitch];
    if (*w.error != 0u) return;
    const int index = b.tile0 + (int)blockIdx.x;
    const int matrix = tile_matrix[index];
    const NsMatrixArg &a = b.m[matrix - b.first];
    if (a.live == 0u) return;
    const NsMatrixDims d = w.dims[matrix];
    const TileView t = tile_view(d, index);
    const __half *x = w.x + d.final_off;
    const int64_t plane = (int64_t)d.np * d.mp;
    constexpr int kOut = kStep ? 2 : 1;
    const NsArray &out = a.a[kOut];
    const bool vec = (a.direct >> kOut) & 1u;
    const bool oi = walks_i(out);
    const float rate = w.rate * a.scale;
#pragma unroll
    for (int pass = 0; pass < 2; ++pass) {
        // pass 0: the iterate, along j; pass 1: from the turned tile, along i
        if (pass == 1 && !oi) break;
        if (pass == 1) __syncthreads();
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const Octet o = octet(pass == 1, k);
            float u[8];
            if (pass == 0) {
                const int64_t pos = (int64_t)(t.i0 + o.i) * d.mp + t.j0 + o.j;
                load8_as(x + pos, 1, 8, true, u);
                if (w.planes == 2) {
                    float l[8];
                    load8_as(x + plane + pos, 1, 8, true, l);
#pragma unroll
                    for (int e = 0; e < 8; ++e) u[e] += l[e];
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) u[e] *= d.final_scale;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) u[e] = at(tile, true, o, e);
            }
            if (pass == 0 && oi) {
#pragma unroll
                for (int e = 0; e < 8; ++e) at(tile, false, o, e) = u[e];
                continue;
            }
            if (kStep) {
                float p[8];
                read8(w.types[kOut], out, vec, oi, t, o, p);
#pragma unroll
                for (int e = 0; e < 8; ++e) u[e] = fmaf(-rate, u[e], p[e] * w.decay);
            }
            write8(w.types[kOut], out, vec, oi, t, o, u);
        }
    }
}

}  // namespace

int launch_ns_norm(const NsElementwise &w, const NsBatchArgs &b, const int32_t *d_tile_matrix, bool step, cudaStream_t stream)
{
    if (b.n_tiles <= 0) return VB_OK;
    if (step) ns_norm_kernel<true><<<b.n_tiles, kThreads, 0, stream>>>(w, b, d_tile_matrix);
    else ns_norm_kernel<false><<<b.n_tiles, kThreads, 0, stream>>>(w, b, d_tile_matrix);
    VB_CUDA(cudaGetLastError());
    return VB_OK;
}

int launch_ns_gather(const NsElementwise &w, const NsBatchArgs &b, const int32_t *d_tile_matrix, bool step, cudaStream_t stream)
{
    if (b.n_tiles <= 0) return VB_OK;
    if (step) ns_gather_kernel<true><<<b.n_tiles, kThreads, 0, stream>>>(w, b, d_tile_matrix);
    else ns_gather_kernel<false><<<b.n_tiles, kThreads, 0, stream>>>(w, b, d_tile_matrix);
    VB_CUDA(cudaGetLastError());
    return VB_OK;
}

int launch_ns_finish(const NsElementwise &w, const NsBatchArgs &b, const int32_t *d_tile_matrix, bool step, cudaStream_t stream)
{
    if (b.n_tiles <= 0) return VB_OK;
    if (step) ns_finish_kernel<true><<<b.n_tiles, kThreads, 0, stream>>>(w, b, d_tile_matrix);
    else ns_finish_kernel<false><<<b.n_tiles, kThreads, 0, stream>>>(w, b, d_tile_matrix);
    VB_CUDA(cudaGetLastError());
    return VB_OK;
}

}  // namespace vb
