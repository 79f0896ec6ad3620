// Newton-Schulz of matrices with a short side of at most 64 (convolution filters, single attention heads,
// narrow output layers) in one launch: a cluster of 1 to 8 CTAs per matrix does everything, from the
// caller's arrays to the caller's arrays.
//
// Such a matrix is a handful of 64 x 64 x 64 products: what costs is latency.  The stages of the general path
// (ns_products.cu) take 8 us each for it, 17 of them for a quintic; here a stage is a tcgen05.mma group, a
// pass of four warps from tensor memory to shared memory, and a __syncthreads.
//
// X (n x m) is cut by columns over the cluster; a CTA's share is read once for the norm, once more (from L2) to
// be scaled by a power of two into f16 planes in shared memory, and stays there: 64 columns are an 8 KiB block
// that serves as K-major operand of the Gram and as MN-major operand of the update alike.  The Gram's
// partial sums are added over the cluster through distributed shared memory in rank order, so all CTAs hold the
// same bits and run the same short-side program, the planner's products (ns_plan.cu), with all of its matrices
// in shared memory as two f16 planes.  With 22 bits on the short side the groups of steps can be long: in
// VB_NS_F16 the five steps of a quintic are one group, so X is read twice and never rewritten.
//
// Shared memory: five squares of 16 KiB, the share of X, and 8 KiB that M = 128 operands run over into (rows
// 64 .. 127 of A are whatever lies there; they only reach rows of the accumulator that nobody reads).
#include <algorithm>

#include "ns_elementwise.h"
#include "tc_ptx.h"

namespace vb {

namespace {

constexpr int kThreads = 256;
constexpr int kSide = kNsSmallSide;
constexpr int kBlockBytes = kSide * 128;          // 64 rows x 64 f16
constexpr int kSquareBytes = 2 * kBlockBytes;     // two planes
constexpr int kSquaresBytes = kNsSmallSquares * kSquareBytes;
constexpr int kTmemCols = 256;
constexpr int kSumSquare = kNsSmallSquares - 1;   // the square whose memory holds partial Grams (f32) between stages

struct alignas(8) Shared {
    uint64_t done;
    double warp_sums[kThreads / 32];
    double cta_sum;
    uint32_t tmem_base;
    uint32_t abort;
    NsSmallOp ops[kNsSmallOps];
};

size_t smem_bytes(int columns, int planes)
{
    return 1024 + kSquaresBytes + (size_t)(columns / 64) * planes * kBlockBytes + kBlockBytes + sizeof(Shared);
}

__device__ __forceinline__ uint32_t pack_half(float a, float b)
{
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 unpack_half(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2 *>(&w)); }

// f += c * (32 values of one row of a block, columns col .. col + 31, all planes)
template <int kPlanes>
__device__ __forceinline__ void add_row(float (&f)[32], float c, uint32_t block, int row, int col)
{
#pragma unroll
    for (int pl = 0; pl < kPlanes; ++pl) {
        const uint32_t at = block + (uint32_t)(pl * kBlockBytes + row * 128);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            uint32_t v[4];
            ld_shared_128(at + (uint32_t)((((col >> 3) + q) ^ (row & 7)) << 4), v[0], v[1], v[2], v[3]);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 x = unpack_half(v[k]);
                f[q * 8 + 2 * k] = fmaf(c, x.x, f[q * 8 + 2 * k]);
                f[q * 8 + 2 * k + 1] = fmaf(c, x.y, f[q * 8 + 2 * k + 1]);
            }
        }
    }
}
template <int kPlanes>
__device__ __forceinline__ void put_row(float (&f)[32], uint32_t block, int row, int col)
{
#pragma unroll
    for (int pl = 0; pl < kPlanes; ++pl) {
        const uint32_t at = block + (uint32_t)(pl * kBlockBytes + row * 128);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            uint32_t h[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                h[k] = pack_half(f[q * 8 + 2 * k], f[q * 8 + 2 * k + 1]);
                if (pl + 1 < kPlanes) {  // what the rounding left over (the difference is exact)
                    const float2 x = unpack_half(h[k]);
                    f[q * 8 + 2 * k] -= x.x;
                    f[q * 8 + 2 * k + 1] -= x.y;
                }
            }
            st_shared_128(at + (uint32_t)((((col >> 3) + q) ^ (row & 7)) << 4), h[0], h[1], h[2], h[3]);
        }
    }
}

// A (128 x 64, rows from 64 on unused) times B (64 x 64) into 64 accumulator columns; operands are blocks of
// kA and kB planes, the products of their planes smallest first.
template <int kA, int kB>
__device__ __forceinline__ void issue_product(uint32_t tmem, uint32_t a, uint32_t b, bool b_mn, bool accumulate)
{
    // f32 accumulator, f16 operands, A K-major, M = 128, N = 64
    const uint32_t idesc = (1u << 4) | ((uint32_t)b_mn << 16) | ((uint32_t)(kSide >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
    bool first = !accumulate;
#pragma unroll
    for (int t = kA + kB - 2; t >= 0; --t) {  // plane of A + plane of B; low x low is dropped
        if (kA == 2 && kB == 2 && t == 2) continue;
#pragma unroll
        for (int pa = 0; pa < kA; ++pa) {
            const int pb = t - pa;
            if (pb < 0 || pb >= kB) continue;
#pragma unroll
            for (int kk = 0; kk < kSide / 16; ++kk) {
                const uint32_t at_b = b + (uint32_t)(pb * kBlockBytes);
                tcgen05_mma_bf16<1>(tmem, make_smem_desc(a + (uint32_t)(pa * kBlockBytes + kk * 32), 16, 1024),
                                    b_mn ? make_smem_desc(at_b + kk * 2048, kBlockBytes, 1024)
                                         : make_smem_desc(at_b + kk * 32, 16, 1024),
                                    idesc, first ? 0u : 1u);
                first = false;
            }
        }
    }
}

__device__ __forceinline__ double warp_sum(double v)
{
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
    return v;
}
__device__ __forceinline__ double ld_cluster_f64(uint32_t addr)
{
    double v;
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr)
{
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}

// The CTA's columns [j0, j1) of the caller's arrays, 8 elements at a time along the first array's direction.
struct Share {
    int n, m, j0, columns;  // columns: padded to 64
    bool along_i;
    __device__ __forceinline__ int octets() const { return columns * (kSide / 8); }
    __device__ __forceinline__ void locate(int o, int &i, int &j, int &count) const
    {
        if (along_i) {
            i = (o & 7) * 8;
            j = o >> 3;
        } else {
            const int per_row = columns / 8;
            i = o / per_row;
            j = (o % per_row) * 8;
        }
        const int left = (j0 + j < m && i < n) ? (along_i ? n - i : m - j0 - j) : 0;
        count = left < 0 ? 0 : left < 8 ? left : 8;
    }
    __device__ __forceinline__ void read(int type, const NsArray &a, bool vec, int i, int j, int count, float (&v)[8]) const
    {
        // a vector access runs along the array's own direction
        load8(type, a.ptr, (int64_t)i * a.si + (int64_t)(j0 + j) * a.sj, along_i ? a.si : a.sj, count,
              vec && walks_i(a) == along_i, v);
    }
    __device__ __forceinline__ void write(int type, const NsArray &a, bool vec, int i, int j, int count, const float (&v)[8]) const
    {
        store8(type, a.ptr, (int64_t)i * a.si + (int64_t)(j0 + j) * a.sj, along_i ? a.si : a.sj, count,
               vec && walks_i(a) == along_i, v);
    }
};

template <bool kStep>
__device__ __forceinline__ void read_u(const NsElementwise &w, const NsMatrixArg &a, const Share &s, int i, int j, int count,
                                       float (&v)[8], float (&u)[8])
{
    if (kStep) {
        float g[8];
        s.read(w.types[0], a.a[0], a.direct & 1u, i, j, count, g);
        s.read(w.types[1], a.a[1], a.direct & 2u, i, j, count, v);
        momentum8(w, g, v, u);
    } else {
        s.read(w.types[0], a.a[0], a.direct & 1u, i, j, count, u);
    }
}

__device__ __forceinline__ void report(const NsError &error)
{
    atomicExch(error.device, 4u);
    *reinterpret_cast<volatile uint32_t *>(error.host) = 4u;
    __threadfence_system();
}

template <int kPlanes, bool kStep>
__global__ void __launch_bounds__(kThreads)
ns_small_kernel(const NsElementwise w, const NsSmall small, const __grid_constant__ NsBatchArgs b, const NsError error,
                uint32_t wait_limit, int withhold)
{
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *x_bytes = smem + kSquaresBytes;
    const int blocks = small.columns / 64;
    Shared &sh = *reinterpret_cast<Shared *>(x_bytes + (size_t)blocks * kPlanes * kBlockBytes + kBlockBytes);
    const uint32_t squares = smem_u32(smem), x_base = smem_u32(x_bytes);

    const int clusters = small.cluster, rank = (int)blockIdx.x % clusters;
    const int index = (int)blockIdx.x / clusters;
    const NsMatrixArg &a = b.m[index];
    const NsSmallMatrix d = small.matrices[b.first + index];
    if (a.live == 0u) return;  // the whole cluster
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool worker = (warp & 3) < 2;  // TMEM lanes 0 .. 63
    const int row = (warp & 3) * 32 + lane, col = (warp >> 2) * 32;

    if (threadIdx.x == 0) {
        mbar_init(&sh.done, 1);
        sh.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    for (int k = threadIdx.x; k < d.n_ops; k += kThreads) sh.ops[k] = small.ops[d.op0 + k];
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem_base)),
                     "r"((uint32_t)kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }

    // ---- the norm: every CTA of the cluster its columns, then all sums in rank order ----
    const Share s{d.n, d.m, rank * small.columns, small.columns, walks_i(a.a[kStep ? 1 : 0])};
    double sum = 0.0;
#pragma unroll 4
    for (int o = threadIdx.x; o < s.octets(); o += kThreads) {
        int i, j, count;
        s.locate(o, i, j, count);
        float v[8], u[8];
        read_u<kStep>(w, a, s, i, j, count, v, u);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fma((double)u[e], (double)u[e], sum);
    }
    sum = warp_sum(sum);
    if (lane == 0) sh.warp_sums[warp] = sum;
    tcgen05_fence_before();
    // dead: nothing is stored.  The control flow goes on all the same, the cluster counts on it.
    bool dead = __syncthreads_or(*reinterpret_cast<const volatile uint32_t *>(error.device) != 0u) != 0;
    tcgen05_fence_after();
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int k = 0; k < kThreads / 32; ++k) t += sh.warp_sums[k];
        sh.cta_sum = t;
    }
    cluster_sync_all();
    double total = 0.0;
    for (int r = 0; r < clusters; ++r) total += ld_cluster_f64(map_to_cta(smem_u32(&sh.cta_sum), (uint32_t)r));
    const double norm = sqrt(total);
    int ex = 13;
    if (norm > 0.0 && isfinite(norm)) (void)frexp(norm, &ex);
    const int shift = 13 - ex;  // norm * 2^shift in [2^12, 2^13)
    const float up0 = ldexpf(1.0f, shift / 2), up1 = ldexpf(1.0f, shift - shift / 2);
    // an infinite or undefined norm makes the whole result undefined, as the formula does
    const float scale = isfinite(norm) ? (float)(ldexp(1.0, -shift) / (norm + (double)w.eps)) : nanf("");

    // ---- the share of X as f16 planes, blocks of 64 columns; step: the new velocity ----
#pragma unroll 2
    for (int o = threadIdx.x; o < s.octets(); o += kThreads) {
        int i, j, count;
        s.locate(o, i, j, count);
        float v[8], u[8];
        read_u<kStep>(w, a, s, i, j, count, v, u);
        if (kStep && !dead) s.write(w.types[1], a.a[1], a.direct & 2u, i, j, count, v);
        const uint32_t block = x_base + (uint32_t)((j >> 6) * kPlanes * kBlockBytes);
        __half h[8], l[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float x = e < count ? u[e] * up0 * up1 : 0.0f;
            h[e] = __float2half_rn(x);
            l[e] = __float2half_rn(x - __half2float(h[e]));
        }
        if (s.along_i) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {  // i is a multiple of 8: row & 7 == e
                const uint32_t at = block + (uint32_t)((i + e) * 128 + ((((j & 63) >> 3) ^ e) << 4) + (j & 7) * 2);
                asm volatile("st.shared.b16 [%0], %1;" ::"r"(at), "h"(__half_as_ushort(h[e])) : "memory");
                if (kPlanes == 2) asm volatile("st.shared.b16 [%0], %1;" ::"r"(at + kBlockBytes), "h"(__half_as_ushort(l[e])) : "memory");
            }
        } else {
            const uint32_t at = block + (uint32_t)(i * 128 + ((((j & 63) >> 3) ^ (i & 7)) << 4));
            const uint4 qh = *reinterpret_cast<const uint4 *>(h), ql = *reinterpret_cast<const uint4 *>(l);
            st_shared_128(at, qh.x, qh.y, qh.z, qh.w);
            if (kPlanes == 2) st_shared_128(at + kBlockBytes, ql.x, ql.y, ql.z, ql.w);
        }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();

    const uint32_t tmem = sh.tmem_base, my_tmem = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)col;
    uint32_t phase = 0;
    auto wait_done = [&] {
        if (!dead) {
            if (!mbar_wait(&sh.done, phase, &sh.abort, wait_limit)) {
                dead = true;
                if (threadIdx.x == 0) report(error);
            }
            phase ^= 1u;
        }
        dead = __syncthreads_or(dead) != 0;
        tcgen05_fence_after();
    };
    // after the accumulators were read and shared memory was written: the tensor core may go on
    auto release = [&] {
        tcgen05_fence_before();
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();
        tcgen05_fence_after();
    };
    auto square = [&](int k) { return squares + (uint32_t)(k * kSquareBytes); };

    for (int op0 = 0; op0 < d.n_ops;) {
        const NsSmallOp first = sh.ops[op0];
        if (first.kind == 1) {
            // ---- Gram: this CTA's columns, then the cluster's sum ----
            float g[32];
#pragma unroll
            for (int k = 0; k < 32; ++k) g[k] = 0.0f;
            // two planes: an accumulator takes 128 columns (its additions truncate, see ns_products.cu)
            const int chunk = kPlanes == 2 ? 2 : blocks;
            for (int b0 = 0; b0 < blocks; b0 += chunk) {
                if (threadIdx.x == 0 && !dead && !withhold) {
                    for (int k = b0; k < min(b0 + chunk, blocks); ++k) {
                        const uint32_t x = x_base + (uint32_t)(k * kPlanes * kBlockBytes);
                        issue_product<kPlanes, kPlanes>(tmem, x, x, false, k > b0);
                    }
                    tcgen05_commit<1>(&sh.done);
                }
                wait_done();
                if (worker) {
                    uint32_t v[32];
                    tmem_ld_32x32_sync(my_tmem, v);
#pragma unroll
                    for (int k = 0; k < 32; ++k) g[k] += __uint_as_float(v[k]);
                }
                release();
            }
            if (clusters > 1) {
                const uint32_t sums = square(kSumSquare);
                const uint32_t mine = (uint32_t)(row * 64 + col) * 4;  // f32 [64][64]
                if (worker) {
#pragma unroll
                    for (int q = 0; q < 8; ++q)
                        st_shared_128(sums + mine + (uint32_t)((q ^ (lane & 7)) << 4), __float_as_uint(g[4 * q]), __float_as_uint(g[4 * q + 1]),
                                      __float_as_uint(g[4 * q + 2]), __float_as_uint(g[4 * q + 3]));
                }
                cluster_sync_all();
                if (worker) {
#pragma unroll
                    for (int k = 0; k < 32; ++k) g[k] = 0.0f;
                    for (int r = 0; r < clusters; ++r) {
                        const uint32_t from = map_to_cta(sums + mine, (uint32_t)r);
#pragma unroll
                        for (int q = 0; q < 8; ++q) {
                            const float4 v = ld_cluster_f32x4(from + (uint32_t)((q ^ (lane & 7)) << 4));
                            g[4 * q] += v.x;
                            g[4 * q + 1] += v.y;
                            g[4 * q + 2] += v.z;
                            g[4 * q + 3] += v.w;
                        }
                    }
                }
                cluster_sync_all();  // the sums' memory is a square again
            }
            if (worker) {
                const float c = first.g * (first.scale_power == 2 ? scale * scale : 1.0f);
#pragma unroll
                for (int k = 0; k < 32; ++k) g[k] *= c;
                put_row<2>(g, square(first.D), row, col);
            }
            release();
            op0 += 1;
        } else if (first.kind == 0) {
            // ---- one stage: one or two independent products ----
            int op1 = op0 + 1;
            while (!sh.ops[op1 - 1].stage_end) ++op1;
            if (threadIdx.x == 0 && !dead) {
                for (int k = op0; k < op1; ++k)
                    issue_product<2, 2>(tmem + (uint32_t)((k - op0) * 64), square(sh.ops[k].A), square(sh.ops[k].B), false, false);
                tcgen05_commit<1>(&sh.done);
            }
            wait_done();
            if (worker) {
                for (int k = op0; k < op1; ++k) {
                    const NsSmallOp op = sh.ops[k];
                    uint32_t v[32];
                    tmem_ld_32x32_sync(my_tmem + (uint32_t)((k - op0) * 64), v);
                    float f[32];
#pragma unroll
                    for (int j = 0; j < 32; ++j) f[j] = op.g * __uint_as_float(v[j]);
                    if (op.E >= 0) add_row<2>(f, op.e, square(op.E), row, col);
                    if (op.F >= 0) add_row<2>(f, op.f, square(op.F), row, col);
                    put_row<2>(f, square(op.D), row, col);
                }
            }
            release();
            op0 = op1;
        } else {
            // ---- update of X, four blocks of 64 columns at a time; the last one goes to the caller ----
            const bool last = op0 + 1 == d.n_ops;
            const float mult = first.scale_power == 1 ? scale : 1.0f;
            const float out_scale = last ? d.final_scale : 1.0f;
            const float ce = first.e * mult * out_scale, cg = first.g * mult * out_scale;
            for (int b0 = 0; b0 < blocks; b0 += 4) {
                const int b1 = min(b0 + 4, blocks);
                if (threadIdx.x == 0 && !dead) {
                    for (int k = b0; k < b1; ++k)
                        issue_product<2, kPlanes>(tmem + (uint32_t)((k - b0) * 64), square(first.A),
                                                  x_base + (uint32_t)(k * kPlanes * kBlockBytes), true, false);
                    tcgen05_commit<1>(&sh.done);
                }
                wait_done();
                if (worker) {
                    for (int k = b0; k < b1; ++k) {
                        const uint32_t block = x_base + (uint32_t)(k * kPlanes * kBlockBytes);
                        uint32_t v[32];
                        tmem_ld_32x32_sync(my_tmem + (uint32_t)((k - b0) * 64), v);
                        float f[32];
#pragma unroll
                        for (int j = 0; j < 32; ++j) f[j] = cg * __uint_as_float(v[j]);
                        add_row<kPlanes>(f, ce, block, row, col);
                        if (!last) {
                            put_row<kPlanes>(f, block, row, col);
                            continue;
                        }
                        if (dead || row >= d.n) continue;
                        constexpr int kOut = kStep ? 2 : 1;
                        const NsArray &dst = a.a[kOut];
                        const int type = w.types[kOut];
                        const bool vec = (a.direct >> kOut) & 1u, by_i = walks_i(dst);
                        const float rate = w.rate * a.scale;
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const int j = s.j0 + k * 64 + col + q * 8;
                            const int count = min(8, d.m - j);
                            if (count <= 0) break;
                            const int64_t at = (int64_t)row * dst.si + (int64_t)j * dst.sj;
                            float o[8];
                            if (kStep) {
                                float p[8];
                                load8(type, dst.ptr, at, dst.sj, count, vec && !by_i, p);
#pragma unroll
                                for (int e = 0; e < 8; ++e) o[e] = fmaf(-rate, f[q * 8 + e], p[e] * w.decay);
                            } else {
#pragma unroll
                                for (int e = 0; e < 8; ++e) o[e] = f[q * 8 + e];
                            }
                            store8(type, dst.ptr, at, dst.sj, count, vec && !by_i, o);
                        }
                    }
                }
                release();
            }
            op0 += 1;
        }
    }

    tcgen05_fence_before();
    __syncthreads();
    cluster_sync_all();  // nobody leaves while its shared memory may be read
    if (warp == 1) {
        tcgen05_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)kTmemCols) : "memory");
    }
}

template <int kPlanes, bool kStep>
int launch_variant(const NsElementwise &w, const NsSmall &s, const NsBatchArgs &b, NsError error, cudaStream_t stream,
                   uint32_t wait_limit, bool withhold)
{
    const size_t smem = smem_bytes(s.columns, kPlanes);
    VB_CUDA(cudaFuncSetAttribute(ns_small_kernel<kPlanes, kStep>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(kThreads);
    cfg.gridDim = dim3((unsigned)(b.count * s.cluster));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)s.cluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    VB_CUDA(cudaLaunchKernelEx(&cfg, ns_small_kernel<kPlanes, kStep>, w, s, b, error, wait_limit, withhold ? 1 : 0));
    return VB_OK;
}

}  // namespace

int ns_small_columns(int planes)
{
    const int room = 232448 - (int)smem_bytes(0, planes);
    return room / (planes * kBlockBytes) * 64;
}

int launch_ns_small(const NsElementwise &w, const NsSmall &s, const NsBatchArgs &b, NsError error, bool step, cudaStream_t stream,
                    uint32_t wait_limit, bool withhold)
{
    if (b.count <= 0) return VB_OK;
    if (w.planes == 2)
        return step ? launch_variant<2, true>(w, s, b, error, stream, wait_limit, withhold)
                    : launch_variant<2, false>(w, s, b, error, stream, wait_limit, withhold);
    return step ? launch_variant<1, true>(w, s, b, error, stream, wait_limit, withhold)
                : launch_variant<1, false>(w, s, b, error, stream, wait_limit, withhold);
}

}  // namespace vb
