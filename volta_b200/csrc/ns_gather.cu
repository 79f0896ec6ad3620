// Element-wise passes of Newton-Schulz on caller-owned matrices (ns_plan.cu):
//   norm    sum of squares of every matrix's U (f64 partial sums per tile, no atomics)
//   gather  U times a power of two -> the f16 working matrix; step: also v <- mu v + g
//   finish  the last iterate -> the caller's output, or  p <- p (1 - lr wd) - lr s O
// with U the input (orthogonalize) or g + mu v' / v' of the new velocity v' (step).
//
// Bound by HBM traffic.  U is needed twice (the norm is a property of the whole matrix) and is
// computed twice instead of being stored: with bf16 gradients and f32 velocities that moves 18
// bytes per element where storing an f32 U would move 20.  The planner launches norm and gather
// alternately over groups of matrices that fit the L2 cache, so the second read of small ones stays on chip.
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
// Two of the tile's four octets of one array in one direction, on their way or as f32 (more of them cost
// occupancy, which this needs more: four at 128 registers were a quarter slower).
struct Octets {
    Raw raw[2];
    __device__ __forceinline__ void load(int k0, int type, const NsArray &a, bool vec, bool along_i, const TileView &t)
    {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const Octet o = octet(along_i, k0 + k);
            raw[k].load(type, a.ptr, offset(a, t, o), t.count(along_i, o), vec);
        }
    }
    __device__ __forceinline__ void get(int k, int type, const NsArray &a, bool along_i, const TileView &t, float (&v)[8]) const
    {
        const Octet o = octet(along_i, k);
        raw[k & 1].get(type, a.ptr, offset(a, t, o), along_i ? a.si : a.sj, t.count(along_i, o), v);
    }
};
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

// U of a tile: the gradient (or input), the velocity, and how they are walked.  Where the gradient's direction is
// not the velocity's it goes through shared memory.
template <bool kStep, bool kTurned>
struct Source {
    Octets g, v;
    bool along_i, turned;
    __device__ __forceinline__ Source(const NsMatrixArg &a)
    {
        along_i = kTurned && walks_i(a.a[kStep ? 1 : 0]);
        turned = kTurned && kStep && walks_i(a.a[0]) != along_i;
    }
    __device__ __forceinline__ void stage(const NsElementwise &w, const NsMatrixArg &a, const TileView &t, float *tile)
    {
        if (!turned) return;
#pragma unroll
        for (int k0 = 0; k0 < 4; k0 += 2) {
            g.load(k0, w.types[0], a.a[0], a.direct & 1u, !along_i, t);
#pragma unroll
            for (int k = k0; k < k0 + 2; ++k) {
                const Octet o = octet(!along_i, k);
                float x[8];
                g.get(k, w.types[0], a.a[0], !along_i, t, x);
#pragma unroll
                for (int e = 0; e < 8; ++e) at(tile, !along_i, o, e) = x[e];
            }
        }
        __syncthreads();
    }
    __device__ __forceinline__ void load(int k0, const NsElementwise &w, const NsMatrixArg &a, const TileView &t)
    {
        if (!turned) g.load(k0, w.types[0], a.a[0], a.direct & 1u, along_i, t);
        if (kStep) v.load(k0, w.types[1], a.a[1], a.direct & 2u, along_i, t);
    }
    // octet k, along along_i; vv: the new velocity
    __device__ __forceinline__ void get(int k, const NsElementwise &w, const NsMatrixArg &a, const TileView &t, float *tile,
                                        float (&vv)[8], float (&u)[8]) const
    {
        const Octet o = octet(along_i, k);
        float x[8];
        if (turned) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = at(tile, along_i, o, e);
        } else {
            g.get(k, w.types[0], a.a[0], along_i, t, x);
        }
        if (kStep) {
            v.get(k, w.types[1], a.a[1], along_i, t, vv);
            momentum8(w, x, vv, u);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) u[e] = x[e];
        }
    }
};

// The kernels come in two forms: kTurned has the shared memory to turn tiles in, the other one, for lists whose
// arrays are all contiguous along the long side (or neither way), keeps the SM's threads instead.
template <bool kStep, bool kTurned>
__global__ void __launch_bounds__(kThreads, 4)
ns_norm_kernel(const NsElementwise w, const __grid_constant__ NsBatchArgs b, const int32_t *__restrict__ tile_matrix)
{
    __shared__ float tile[kStep && kTurned ? kNsTileI * kPitch : 1];
    __shared__ double warp_sums[kThreads / 32];
    const int index = b.tile0 + (int)blockIdx.x;
    const int matrix = tile_matrix[index];
    const NsMatrixArg &a = b.m[matrix - b.first];
    if (a.live == 0u) return;
    const TileView t = tile_view(a.d, index);
    Source<kStep, kTurned> s(a);
    s.stage(w, a, t, tile);
    double sum = 0.0;
#pragma unroll
    for (int k0 = 0; k0 < 4; k0 += 2) {
        s.load(k0, w, a, t);
#pragma unroll
        for (int k = k0; k < k0 + 2; ++k) {
            float v[8], u[8];
            s.get(k, w, a, t, tile, v, u);
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

template <bool kStep, bool kTurned>
__global__ void __launch_bounds__(kThreads, 4)
ns_gather_kernel(const NsElementwise w, const __grid_constant__ NsBatchArgs b, const int32_t *__restrict__ tile_matrix)
{
    __shared__ float tile[kTurned ? kNsTileI * kPitch : 1];
    __shared__ double warp_sums[kThreads / 32];
    const int index = b.tile0 + (int)blockIdx.x;
    const int matrix = tile_matrix[index];
    const NsMatrixArg &a = b.m[matrix - b.first];
    const NsMatrixDims &d = a.d;
    if (index == d.tile0 && threadIdx.x == 0) {
        w.active[matrix] = a.live;
        w.stored[matrix] = 0u;
    }
    if (a.live == 0u || *w.error != 0u) return;
    const TileView t = tile_view(d, index);
    Source<kStep, kTurned> s(a);
    s.stage(w, a, t, tile);
    s.load(0, w, a, t);  // on their way while the norm is summed

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
#pragma unroll
    for (int k0 = 0; k0 < 4; k0 += 2) {
        if (k0 > 0) s.load(k0, w, a, t);
#pragma unroll
        for (int k = k0; k < k0 + 2; ++k) {
            const Octet o = octet(s.along_i, k);
            float v[8], u[8];
            s.get(k, w, a, t, tile, v, u);
            if (kStep) write8(w.types[1], a.a[1], a.direct & 2u, s.along_i, t, o, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) u[e] = u[e] * up0 * up1;
            if (s.along_i) {  // this thread alone read these elements of the tile
#pragma unroll
                for (int e = 0; e < 8; ++e) at(tile, true, o, e) = u[e];
            } else {
                store_working(x + (int64_t)(t.i0 + o.i) * d.mp + t.j0 + o.j, plane, w.planes, u);
            }
        }
    }
    if (s.along_i) {
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

template <bool kStep, bool kTurned>
__global__ void __launch_bounds__(kThreads, 4)
ns_finish_kernel(const NsElementwise w, const __grid_constant__ NsBatchArgs b, const int32_t *__restrict__ tile_matrix)
{
    __shared__ float tile[kTurned ? kNsTileI * kPitch : 1];
    const int index = b.tile0 + (int)blockIdx.x;
    const int matrix = tile_matrix[index];
    const NsMatrixArg &a = b.m[matrix - b.first];
    if (a.live == 0u || *w.error != 0u) return;
    const NsMatrixDims &d = a.d;
    const TileView t = tile_view(d, index);
    const __half *x = w.x + d.final_off;
    const int64_t plane = (int64_t)d.np * d.mp;
    constexpr int kOut = kStep ? 2 : 1;
    const NsArray &out = a.a[kOut];
    const bool vec = (a.direct >> kOut) & 1u;
    const bool oi = kTurned && walks_i(out);
    const float rate = w.rate * a.scale;
    Octets p;  // the parameters, along their own direction
    auto finish = [&](int k, float (&u)[8]) {
        if (kStep) {
            float x8[8];
            p.get(k, w.types[kOut], out, oi, t, x8);
#pragma unroll
            for (int e = 0; e < 8; ++e) u[e] = fmaf(-rate, u[e], x8[e] * w.decay);
        }
        write8(w.types[kOut], out, vec, oi, t, octet(oi, k), u);
    };
#pragma unroll
    for (int k0 = 0; k0 < 4; k0 += 2) {
        uint4 high[2], low[2];  // the iterate, along j
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const Octet o = octet(false, k0 + k);
            const int64_t pos = (int64_t)(t.i0 + o.i) * d.mp + t.j0 + o.j;
            high[k] = *reinterpret_cast<const uint4 *>(x + pos);
            if (w.planes == 2) low[k] = *reinterpret_cast<const uint4 *>(x + plane + pos);
        }
        if (kStep && !oi) p.load(k0, w.types[kOut], out, vec, oi, t);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            float u[8];
            const uint32_t h[4] = {high[k].x, high[k].y, high[k].z, high[k].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 z = unpack_half(h[e]);
                u[2 * e] = z.x, u[2 * e + 1] = z.y;
            }
            if (w.planes == 2) {
                const uint32_t l[4] = {low[k].x, low[k].y, low[k].z, low[k].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 z = unpack_half(l[e]);
                    u[2 * e] += z.x, u[2 * e + 1] += z.y;
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) u[e] *= d.final_scale;
            if (oi) {  // turned in shared memory
#pragma unroll
                for (int e = 0; e < 8; ++e) at(tile, false, octet(false, k0 + k), e) = u[e];
            } else {
                finish(k0 + k, u);
            }
        }
    }
    if (!oi) return;
    __syncthreads();
#pragma unroll
    for (int k0 = 0; k0 < 4; k0 += 2) {
        if (kStep) p.load(k0, w.types[kOut], out, vec, oi, t);
#pragma unroll
        for (int k = k0; k < k0 + 2; ++k) {
            float u[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) u[e] = at(tile, true, octet(true, k), e);
            finish(k, u);
        }
    }
}

}  // namespace

int launch_ns_norm(const NsElementwise &w, const NsBatchArgs &b, const int32_t *d_tile_matrix, bool step, bool turned, cudaStream_t stream)
{
    if (b.n_tiles <= 0) return VB_OK;
    auto *kernel = step ? (turned ? ns_norm_kernel<true, true> : ns_norm_kernel<true, false>)
                        : (turned ? ns_norm_kernel<false, true> : ns_norm_kernel<false, false>);
    kernel<<<b.n_tiles, kThreads, 0, stream>>>(w, b, d_tile_matrix);
    VB_CUDA(cudaGetLastError());
    return VB_OK;
}

int launch_ns_gather(const NsElementwise &w, const NsBatchArgs &b, const int32_t *d_tile_matrix, bool step, bool turned, cudaStream_t stream)
{
    if (b.n_tiles <= 0) return VB_OK;
    auto *kernel = step ? (turned ? ns_gather_kernel<true, true> : ns_gather_kernel<true, false>)
                        : (turned ? ns_gather_kernel<false, true> : ns_gather_kernel<false, false>);
    kernel<<<b.n_tiles, kThreads, 0, stream>>>(w, b, d_tile_matrix);
    VB_CUDA(cudaGetLastError());
    return VB_OK;
}

int launch_ns_finish(const NsElementwise &w, const NsBatchArgs &b, const int32_t *d_tile_matrix, bool step, bool turned, cudaStream_t stream)
{
    if (b.n_tiles <= 0) return VB_OK;
    auto *kernel = step ? (turned ? ns_finish_kernel<true, true> : ns_finish_kernel<true, false>)
                        : (turned ? ns_finish_kernel<false, true> : ns_finish_kernel<false, false>);
    kernel<<<b.n_tiles, kThreads, 0, stream>>>(w, b, d_tile_matrix);
    VB_CUDA(cudaGetLastError());
    return VB_OK;
}

}  // namespace vb
