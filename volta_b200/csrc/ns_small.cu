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
// that serves, along one direction or the other, as operand of the Gram and of the update alike.  The Gram's
// partial sums are added over the cluster through distributed shared memory in rank order, so all CTAs hold the
// same bits and run the same short-side program, the planner's products (ns_plan.cu), with all of its matrices
// in shared memory as two f16 planes.  With 22 bits on the short side the groups of steps can be long: in
// VB_NS_F16 the five steps of a quintic are one group, so X is read twice and never rewritten.
//
// What a stage of short-side products costs (cycles, 64 x 288 to f32 accuracy): issuing 12 MMAs 1000, their completion 300
// to 500, tensor memory to shared memory 900, barriers 200; a Gram over a cluster of 8 takes 6500, 4300 of them the sum.
// The whole call takes 39 us with a 32 x 9 matrix beside it; 192 bf16 heads of 1024 x 64 take 107 us, two rounds of one
// head per SM.
//
// A short side of at most 16 to f32 accuracy (tiny) is worked on in f64 on the CUDA cores instead: planes of 22
// bits, amplified by steep coefficients, left errors of 1e-5 to 2e-5 at 8 x 3000, and 16 x 16 products are nothing.
// U stays in shared memory in f32; G, the polynomial of G and its product with U are f64.
//
// Shared memory: five squares of 16 KiB, the share of X, and 8 KiB that M = 128 operands run over into (rows
// 64 .. 127 of A are whatever lies there; they only reach rows of the accumulator that nobody reads).
#include <algorithm>

#include "ns_elementwise.h"
#include "tc_ptx.h"

namespace vb {

namespace {

constexpr int kThreads = 512;
constexpr int kCols = 16;  // columns of a worker warp: 8 of the 16 warps reach TMEM lanes 0 .. 63
constexpr int kSide = kNsSmallSide;
constexpr int kBlockBytes = kSide * 128;          // 64 rows x 64 f16
constexpr int kSquareBytes = 2 * kBlockBytes;     // two planes
constexpr int kSquaresBytes = kNsSmallSquares * kSquareBytes;
constexpr int kTmemCols = 256;
constexpr int kSumSquare = kNsSmallSquares - 1;   // the square whose memory holds partial Grams (f32) between stages

constexpr int kTiny = kNsTinySide;
struct TinySquares {  // in the squares' memory
    double g[kTiny][kTiny + 1], q[kTiny][kTiny + 1], t[kTiny][kTiny + 1], p[kTiny][kTiny + 1];
    double part[2][kTiny * kTiny];  // this CTA's Gram, by halves of its columns
};
static_assert(sizeof(TinySquares) <= kSquaresBytes, "they share memory");

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

// f += c * (16 values of one row of a block, columns col .. col + 15, all planes)
template <int kPlanes>
__device__ __forceinline__ void add_row(float (&f)[kCols], float c, uint32_t block, uint32_t plane, int row, int col)
{
#pragma unroll
    for (int pl = 0; pl < kPlanes; ++pl) {
        const uint32_t at = block + pl * plane + (uint32_t)(row * 128);
#pragma unroll
        for (int q = 0; q < kCols / 8; ++q) {
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
__device__ __forceinline__ void put_row(float (&f)[kCols], uint32_t block, uint32_t plane, int row, int col)
{
#pragma unroll
    for (int pl = 0; pl < kPlanes; ++pl) {
        const uint32_t at = block + pl * plane + (uint32_t)(row * 128);
#pragma unroll
        for (int q = 0; q < kCols / 8; ++q) {
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

// An operand of M (or N) x 64: the descriptor of its plane 0, what to add to its address field for the next plane
// and for the next 16 of the contraction, and which way it lies.
struct Operand {
    uint64_t desc;
    uint32_t plane, step;
    bool mn_major;
};
// A (M = 128) times B (N = 64) into 64 accumulator columns, the products of their planes smallest first.  The whole
// warp runs this, its elected lane issues.  k_slices: 16 each.
template <int kA, int kB>
__device__ __forceinline__ void issue_product(uint32_t tmem, const Operand &a, const Operand &b, bool accumulate, int k_slices,
                                              bool elected)
{
    // f32 accumulator, f16 operands, M = 128, N = 64
    const uint32_t idesc = (1u << 4) | ((uint32_t)a.mn_major << 15) | ((uint32_t)b.mn_major << 16) |
                           ((uint32_t)(kSide >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
    bool first = true;
#pragma unroll
    for (int t = kA + kB - 2; t >= 0; --t) {  // plane of A + plane of B; low x low is dropped
        if (kA == 2 && kB == 2 && t == 2) continue;
#pragma unroll
        for (int pa = 0; pa < kA; ++pa) {
            const int pb = t - pa;
            if (pb < 0 || pb >= kB) continue;
#pragma unroll
            for (int kk = 0; kk < kSide / 16; ++kk) {
                if (elected && kk < k_slices)
                    tcgen05_mma_bf16<1>(tmem, a.desc + pa * a.plane + kk * a.step, b.desc + pb * b.plane + kk * b.step, idesc,
                                        (first && kk == 0) ? (accumulate ? 1u : 0u) : 1u);
            }
            first = false;
        }
    }
}
// Descriptors of an operand block in shared memory: everything but the address is the same for all blocks.
struct Descriptors {
    uint64_t k_major, mn_major;  // of address 0
    __device__ __forceinline__ Descriptors() : k_major(make_smem_desc(0, 16, 1024)), mn_major(make_smem_desc(0, kBlockBytes, 1024)) {}
    // `addr` holds rows of 64 along the contraction, or 64 rows of the contraction
    __device__ __forceinline__ Operand operand(uint32_t addr, uint32_t plane, bool mn) const
    {
        return {(mn ? mn_major : k_major) + (addr >> 4), plane >> 4, mn ? 2048u >> 4 : 32u >> 4, mn};
    }
};
__device__ __forceinline__ void tmem_ld_16_sync(uint32_t taddr, float (&f)[kCols])
{
    uint32_t v[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr)
        : "memory");
#pragma unroll
    for (int k = 0; k < 16; ++k) f[k] = __uint_as_float(v[k]);
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
// volatile, so after the barrier before it; no memory clobber, so that several are in flight
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr)
{
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ void st_cluster_f32x4(uint32_t addr, float4 v)
{
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
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
    __device__ __forceinline__ int64_t offset(const NsArray &a, int i, int j) const { return (int64_t)i * a.si + (int64_t)(j0 + j) * a.sj; }
    __device__ __forceinline__ int64_t step(const NsArray &a) const { return along_i ? a.si : a.sj; }
    // a vector access runs along the array's own direction
    __device__ __forceinline__ bool vec(const NsArray &a, bool aligned) const { return aligned && walks_i(a) == along_i; }
    __device__ __forceinline__ void write(int type, const NsArray &a, bool aligned, int i, int j, int count, const float (&v)[8]) const
    {
        store8(type, a.ptr, offset(a, i, j), along_i ? a.si : a.sj, count, vec(a, aligned), v);
    }
};

// Calls fn(i, j, count, v, u) for this thread's octets of U (and, step, of the new velocity).
constexpr int kInFlight = 4;
template <bool kStep, typename Fn>
__device__ __forceinline__ void for_u(const NsElementwise &w, const NsMatrixArg &a, const Share &s, Fn &&fn)
{
    for (int o0 = threadIdx.x; o0 < s.octets(); o0 += kThreads * kInFlight) {
        Raw g[kInFlight], v[kStep ? kInFlight : 1];
#pragma unroll
        for (int k = 0; k < kInFlight; ++k) {
            const int o = o0 + k * kThreads;
            if (o >= s.octets()) break;
            int i, j, count;
            s.locate(o, i, j, count);
            g[k].load(w.types[0], a.a[0].ptr, s.offset(a.a[0], i, j), count, s.vec(a.a[0], a.direct & 1u));
            if (kStep) v[kStep ? k : 0].load(w.types[1], a.a[1].ptr, s.offset(a.a[1], i, j), count, s.vec(a.a[1], a.direct & 2u));
        }
#pragma unroll
        for (int k = 0; k < kInFlight; ++k) {
            const int o = o0 + k * kThreads;
            if (o >= s.octets()) break;
            int i, j, count;
            s.locate(o, i, j, count);
            float gg[8], vv[8], u[8];
            g[k].get(w.types[0], a.a[0].ptr, s.offset(a.a[0], i, j), s.step(a.a[0]), count, gg);
            if (kStep) {
                v[kStep ? k : 0].get(w.types[1], a.a[1].ptr, s.offset(a.a[1], i, j), s.step(a.a[1]), count, vv);
                momentum8(w, gg, vv, u);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) u[e] = gg[e];
            }
            fn(i, j, count, vv, u);
        }
    }
}

// X in shared memory: plane p's block b (64 columns of X) at (p blocks + b) 8 KiB, as 64 rows of 128 bytes; a row is
// a row of X, or (turned) a column.
struct Image {
    uint32_t base, plane;
    bool turned;
    __device__ __forceinline__ uint32_t block(int b) const { return base + (uint32_t)(b * kBlockBytes); }
    __device__ __forceinline__ uint32_t at(int i, int j) const
    {
        const int r = turned ? j & 63 : i, c = turned ? i : j & 63;
        return block(j >> 6) + (uint32_t)(r * 128 + (((c >> 3) ^ (r & 7)) << 4) + (c & 7) * 2);
    }
};

// 8 elements of the input that lie in the image as they were
template <int kPlanes>
__device__ __forceinline__ void read_copied(int type, const Image &x, int i, int j, float (&u)[8])
{
    uint32_t q[kPlanes][4];
#pragma unroll
    for (int pl = 0; pl < kPlanes; ++pl) ld_shared_128(x.at(i, j) + pl * x.plane, q[pl][0], q[pl][1], q[pl][2], q[pl][3]);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (kPlanes == 2) {
#pragma unroll
            for (int pl = 0; pl < kPlanes; ++pl) u[4 * pl + k] = __uint_as_float(q[pl][k]);
        } else if (type == VB_DTYPE_BF16) {
            u[2 * k] = __uint_as_float(q[0][k] << 16);
            u[2 * k + 1] = __uint_as_float(q[0][k] & 0xffff0000u);
        } else {
            const float2 z = unpack_half(q[0][k]);
            u[2 * k] = z.x, u[2 * k + 1] = z.y;
        }
    }
}

// Element (i, j) of U where the image holds f32: 8 along the image's rows are 4 in plane 0 and 4 in plane 1.
__device__ __forceinline__ float tiny_u(const Image &x, int i, int j)
{
    const int along = x.turned ? i : j, first = along & ~7;
    const uint32_t at = (x.turned ? x.at(first, j) : x.at(i, first)) + ((along & 4) ? x.plane : 0u) + (uint32_t)(along & 3) * 4u;
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}
// ts.p <- the polynomial of the Gram, over (|U|_F + eps): O = ts.p U.  Every CTA of the cluster computes it from the same sums.
__device__ __forceinline__ void tiny_polynomial(TinySquares &ts, const NsSmall &small, const Share &s, const Image &x, int clusters,
                                                double scale, uint32_t smem_ts)
{
    const int pair = (int)threadIdx.x & (kTiny * kTiny - 1), half = (int)threadIdx.x / (kTiny * kTiny);
    const int r = pair / kTiny, c = pair % kTiny;
    static_assert(kThreads == 2 * kTiny * kTiny, "a thread per element and half of the columns");
    double sum = 0.0;
    const int columns = s.columns / 2;
    for (int j = half * columns; j < (half + 1) * columns; ++j)
        sum = fma((double)tiny_u(x, r, j), (double)tiny_u(x, c, j), sum);
    ts.part[half][pair] = sum;
    cluster_sync_all();
    if (half == 0) {
        double g = 0.0;
        for (int k = 0; k < clusters; ++k)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                g += ld_cluster_f64(map_to_cta(smem_ts + (uint32_t)((const char *)&ts.part[h][pair] - (const char *)&ts), (uint32_t)k));
        ts.g[r][c] = g / scale / scale;
        ts.p[r][c] = r == c ? 1.0 / scale : 0.0;
    }
    cluster_sync_all();
    auto product = [&](const double (&a)[kTiny][kTiny + 1], const double (&b)[kTiny][kTiny + 1]) {
        double v = 0.0;
#pragma unroll
        for (int k = 0; k < kTiny; ++k) v = fma(a[r][k], b[k][c], v);
        return v;
    };
    for (int k = 0; k < small.n_steps; ++k) {
        const double sa = small.coefficients[3 * k], sb = small.coefficients[3 * k + 1], sc = small.coefficients[3 * k + 2];
        if (half == 0) ts.q[r][c] = (r == c ? sa : 0.0) + sb * ts.g[r][c] + sc * product(ts.g, ts.g);
        __syncthreads();
        const double next_p = half == 0 ? product(ts.q, ts.p) : 0.0;
        if (half == 1) ts.t[r][c] = product(ts.q, ts.g);
        __syncthreads();
        if (half == 0) ts.p[r][c] = next_p;
        if (half == 1) ts.g[r][c] = product(ts.t, ts.q);
        __syncthreads();
    }
}
// 8 elements of P U along i or along j
__device__ __forceinline__ void tiny_output(const TinySquares &ts, const Image &x, int n, bool along_i, int i, int j, float (&f)[8])
{
    double v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.0;
    for (int k = 0; k < n; ++k) {
        if (along_i) {
            const double u = (double)tiny_u(x, k, j);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = fma(ts.p[min(i + e, kTiny - 1)][k], u, v[e]);
        } else {
            const double p = ts.p[i][k];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = fma(p, (double)tiny_u(x, k, j + e), v[e]);
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = (float)v[e];
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
    const uint32_t squares = smem_u32(smem);

    const int clusters = small.cluster, rank = (int)blockIdx.x % clusters;
    const int index = (int)blockIdx.x / clusters;
    const NsMatrixArg &a = b.m[index];
    const NsSmallMatrix d = small.matrices[b.first + index];
    if (a.live == 0u) return;  // the whole cluster
    const int warp = uniform((int)(threadIdx.x >> 5)), lane = threadIdx.x & 31;
    const bool worker = (warp & 3) < 2;  // TMEM lanes 0 .. 63
    const int row = (warp & 3) * 32 + lane, col = (warp >> 2) * kCols;

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

    // X lies in shared memory as the first array lies in memory: whole 16-byte pieces move, no transposition
    const Image x{smem_u32(x_bytes), (uint32_t)(blocks * kBlockBytes), walks_i(a.a[kStep ? 1 : 0])};

    // ---- the norm: every CTA of the cluster its columns, then all sums in rank order ----
    const Share s{d.n, d.m, rank * small.columns, small.columns, walks_i(a.a[kStep ? 1 : 0])};
    // An input whose elements have as many bytes as the planes (16-bit types and one plane, f32 and two) is copied into
    // the image as it is, all of it on its way at once, and summed and converted there; others are read twice.
    const int type0 = w.types[0];
    const bool copied = !kStep && (type0 == VB_DTYPE_F32) == (kPlanes == 2);
    double sum = 0.0;
    if (copied) {
        const NsArray &in = a.a[0];
        for (int o = threadIdx.x; o < s.octets(); o += kThreads) {
            int i, j, count;
            s.locate(o, i, j, count);
            const uint32_t to = x.at(i, j);
            if (count == 8 && s.vec(in, a.direct & 1u)) {
                const char *from = static_cast<const char *>(in.ptr) + s.offset(in, i, j) * (2 * kPlanes);
#pragma unroll
                for (int pl = 0; pl < kPlanes; ++pl)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + pl * x.plane), "l"(from + pl * 16) : "memory");
            } else {
                float v[8];
                load8(type0, in.ptr, s.offset(in, i, j), s.step(in), count, false, v);
                if (kPlanes == 2) {
#pragma unroll
                    for (int pl = 0; pl < kPlanes; ++pl)
                        st_shared_128(to + pl * x.plane, __float_as_uint(v[4 * pl]), __float_as_uint(v[4 * pl + 1]),
                                      __float_as_uint(v[4 * pl + 2]), __float_as_uint(v[4 * pl + 3]));
                } else {
                    uint32_t h[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {  // the input's own bits again
                        if (type0 == VB_DTYPE_BF16) h[k] = __float_as_uint(v[2 * k]) >> 16 | (__float_as_uint(v[2 * k + 1]) & 0xffff0000u);
                        else h[k] = pack_half(v[2 * k], v[2 * k + 1]);
                    }
                    st_shared_128(to, h[0], h[1], h[2], h[3]);
                }
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        for (int o = threadIdx.x; o < s.octets(); o += kThreads) {  // the octets this thread copied
            int i, j, count;
            s.locate(o, i, j, count);
            float u[8];
            read_copied<kPlanes>(type0, x, i, j, u);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum = fma((double)u[e], (double)u[e], sum);
        }
    } else {
        for_u<kStep>(w, a, s, [&](int, int, int, const float (&)[8], const float (&u)[8]) {
#pragma unroll
            for (int e = 0; e < 8; ++e) sum = fma((double)u[e], (double)u[e], sum);
        });
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
    const bool tiny = kPlanes == 2 && d.n <= kTiny;
    auto put = [&](int i, int j, int count, const float (&u)[8]) {
        if (tiny) {  // as it is
            const uint32_t to = x.at(i, j);
#pragma unroll
            for (int pl = 0; pl < kPlanes; ++pl)
                st_shared_128(to + pl * x.plane, __float_as_uint(u[4 * pl]), __float_as_uint(u[4 * pl + 1]),
                              __float_as_uint(u[4 * pl + 2]), __float_as_uint(u[4 * pl + 3]));
            return;
        }
        __half h[8], l[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float z = e < count ? u[e] * up0 * up1 : 0.0f;
            h[e] = __float2half_rn(z);
            l[e] = __float2half_rn(z - __half2float(h[e]));
        }
        const uint32_t at = x.at(i, j);  // along the image's rows: s.along_i == x.turned
        const uint4 qh = *reinterpret_cast<const uint4 *>(h), ql = *reinterpret_cast<const uint4 *>(l);
        st_shared_128(at, qh.x, qh.y, qh.z, qh.w);
        if (kPlanes == 2) st_shared_128(at + x.plane, ql.x, ql.y, ql.z, ql.w);
    };
    if (copied && !tiny) {
        for (int o = threadIdx.x; o < s.octets(); o += kThreads) {
            int i, j, count;
            s.locate(o, i, j, count);
            float u[8];
            read_copied<kPlanes>(type0, x, i, j, u);
            put(i, j, count, u);
        }
    } else if (!copied) {
        for_u<kStep>(w, a, s, [&](int i, int j, int count, const float (&v)[8], const float (&u)[8]) {
            if (kStep && !dead) s.write(w.types[1], a.a[1], a.direct & 2u, i, j, count, v);
            put(i, j, count, u);
        });
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();

    const uint32_t tmem = uniform(sh.tmem_base), my_tmem = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)col;
    uint32_t phase = 0;
    const Descriptors desc;
    const bool issuer = warp == 3;            // a warp that does not drain; one lane of it issues
    const bool elected = issuer && elect_one();
    const int k_slices = uniform((d.n + 15) / 16);     // of products over the short side
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
    auto square_operand = [&](int k) { return desc.operand(square(k), kBlockBytes, false); };

    TinySquares &ts = *reinterpret_cast<TinySquares *>(smem);
    if (tiny) tiny_polynomial(ts, small, s, x, clusters, norm + (double)w.eps, squares);
    for (int op0 = tiny ? d.n_ops : 0; op0 < d.n_ops;) {
        const NsSmallOp first = sh.ops[op0];
        if (first.kind == 1) {
            // ---- Gram: this CTA's columns, then the cluster's sum ----
            float g[kCols];
#pragma unroll
            for (int k = 0; k < kCols; ++k) g[k] = 0.0f;
            // two planes: an accumulator takes 128 columns (its additions truncate, see ns_products.cu)
            const int chunk = kPlanes == 2 ? 2 : blocks;
            for (int b0 = 0; b0 < blocks; b0 += chunk) {
                if (issuer && !dead && !withhold) {
                    for (int k = b0; k < min(b0 + chunk, blocks); ++k) {
                        const Operand o = desc.operand(x.block(k), x.plane, x.turned);  // turned: columns of X are rows
                        issue_product<kPlanes, kPlanes>(tmem, o, o, k > b0, kSide / 16, elected);
                    }
                    if (elected) tcgen05_commit<1>(&sh.done);
                }
                wait_done();
                if (worker) {
                    float v[kCols];
                    tmem_ld_16_sync(my_tmem, v);
#pragma unroll
                    for (int k = 0; k < kCols; ++k) g[k] += v[k];
                }
                release();
            }
            if (clusters > 1) {
                // f32 [64][64] as 1024 words of 16 bytes; every CTA sums its part of the words over the cluster, in
                // rank order, and writes the sums to all (a word is read and rewritten by one thread only)
                const uint32_t sums = square(kSumSquare);
                const uint32_t mine = sums + (uint32_t)(row * 256);
                if (worker) {
#pragma unroll
                    for (int q = 0; q < kCols / 4; ++q)
                        st_shared_128(mine + (uint32_t)((((col >> 2) + q) ^ (row & 7)) << 4), __float_as_uint(g[4 * q]),
                                      __float_as_uint(g[4 * q + 1]), __float_as_uint(g[4 * q + 2]), __float_as_uint(g[4 * q + 3]));
                }
                cluster_sync_all();
                const int words = kSide * kSide / 4 / clusters;
                for (int k = threadIdx.x; k < words; k += kThreads) {
                    const uint32_t word = sums + (uint32_t)((rank * words + k) * 16);
                    float4 part[kNsSmallCluster];
#pragma unroll
                    for (int r = 0; r < kNsSmallCluster; ++r)
                        if (r < clusters) part[r] = ld_cluster_f32x4(map_to_cta(word, (uint32_t)r));
                    float4 t = part[0];
#pragma unroll
                    for (int r = 1; r < kNsSmallCluster; ++r)
                        if (r < clusters) t.x += part[r].x, t.y += part[r].y, t.z += part[r].z, t.w += part[r].w;
#pragma unroll
                    for (int r = 0; r < kNsSmallCluster; ++r)
                        if (r < clusters) st_cluster_f32x4(map_to_cta(word, (uint32_t)r), t);
                }
                cluster_sync_all();
                if (worker) {
#pragma unroll
                    for (int q = 0; q < kCols / 4; ++q) {
                        uint32_t v[4];
                        ld_shared_128(mine + (uint32_t)((((col >> 2) + q) ^ (row & 7)) << 4), v[0], v[1], v[2], v[3]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) g[4 * q + e] = __uint_as_float(v[e]);
                    }
                }
            }
            if (worker) {
                const float c = first.g * (first.scale_power == 2 ? scale * scale : 1.0f);
#pragma unroll
                for (int k = 0; k < kCols; ++k) g[k] *= c;
                put_row<2>(g, square(first.D), kBlockBytes, row, col);
            }
            release();
            op0 += 1;
        } else if (first.kind == 0) {
            // ---- one stage: one or two independent products ----
            const int count = first.stage_ops;
            if (issuer && !dead) {
                for (int k = 0; k < count; ++k)
                    issue_product<2, 2>(tmem + (uint32_t)(k * 64), square_operand(uniform((int)sh.ops[op0 + k].A)),
                                        square_operand(uniform((int)sh.ops[op0 + k].B)), false, k_slices, elected);
                if (elected) tcgen05_commit<1>(&sh.done);
            }
            // the terms that are there already, while the products run
            float f[2][kCols];
            if (worker) {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
#pragma unroll
                    for (int j = 0; j < kCols; ++j) f[k][j] = 0.0f;
                    if (k >= count) continue;
                    const NsSmallOp op = sh.ops[op0 + k];
                    if (op.E >= 0) add_row<2>(f[k], op.e, square(op.E), kBlockBytes, row, col);
                    if (op.F >= 0) add_row<2>(f[k], op.f, square(op.F), kBlockBytes, row, col);
                }
            }
            wait_done();
            if (worker) {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    if (k >= count) continue;
                    float v[kCols];
                    tmem_ld_16_sync(my_tmem + (uint32_t)(k * 64), v);
                    const float c = sh.ops[op0 + k].g;
#pragma unroll
                    for (int j = 0; j < kCols; ++j) f[k][j] = fmaf(c, v[j], f[k][j]);
                    put_row<2>(f[k], square(sh.ops[op0 + k].D), kBlockBytes, row, col);
                }
            }
            release();
            op0 += count;
        } else {
            // ---- update of X in place, 256 accumulator columns at a time ----
            // P X for four blocks (X's rows in 64 lanes), or, turned, X^T P (P is symmetric) for eight: two blocks
            // follow each other in memory as the 128 rows of one operand
            const float mult = first.scale_power == 1 ? scale : 1.0f;
            const float ce = first.e * mult, cg = first.g * mult;
            const int per_product = x.turned ? 2 : 1;
            const Operand P = square_operand(uniform((int)first.A));
            for (int b0 = 0; b0 < blocks; b0 += 4 * per_product) {
                const int products = min(4, (blocks - b0 + per_product - 1) / per_product);
                if (issuer && !dead) {
                    for (int k = 0; k < products; ++k) {
                        const Operand X = desc.operand(x.block(b0 + k * per_product), x.plane, !x.turned);
                        if (x.turned) issue_product<kPlanes, 2>(tmem + (uint32_t)(k * 64), X, P, false, k_slices, elected);
                        else issue_product<2, kPlanes>(tmem + (uint32_t)(k * 64), P, X, false, k_slices, elected);
                    }
                    if (elected) tcgen05_commit<1>(&sh.done);
                }
                wait_done();
                if (worker || x.turned) {
                    for (int k = 0; k < products; ++k) {
                        const int at = b0 + k * per_product + (row >> 6);
                        float f[kCols];
                        tmem_ld_16_sync(my_tmem + (uint32_t)(k * 64), f);  // the whole warp
                        if (at >= blocks) continue;
#pragma unroll
                        for (int j = 0; j < kCols; ++j) f[j] *= cg;
                        add_row<kPlanes>(f, ce, x.block(at), x.plane, row & 63, col);
                        put_row<kPlanes>(f, x.block(at), x.plane, row & 63, col);
                    }
                }
                release();
            }
            op0 += 1;
        }
    }

    // ---- from the last iterate to the caller ----
    if (!dead) {
        constexpr int kOut = kStep ? 2 : 1;
        const NsArray &dst = a.a[kOut];
        Share out = s;
        out.along_i = walks_i(dst);
        const float rate = w.rate * a.scale, final_scale = tiny ? 1.0f : d.final_scale;
        for (int o0 = threadIdx.x; o0 < out.octets(); o0 += kThreads * kInFlight) {
            Raw p[kStep ? kInFlight : 1];
#pragma unroll
            for (int k = 0; k < (kStep ? kInFlight : 0); ++k) {
                int i, j, count;
                if (o0 + k * kThreads >= out.octets()) break;
                out.locate(o0 + k * kThreads, i, j, count);
                p[k].load(w.types[kOut], dst.ptr, out.offset(dst, i, j), count, out.vec(dst, (a.direct >> kOut) & 1u));
            }
#pragma unroll
            for (int k = 0; k < kInFlight; ++k) {
                int i, j, count;
                if (o0 + k * kThreads >= out.octets()) break;
                out.locate(o0 + k * kThreads, i, j, count);
                if (count == 0) continue;
                float f[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = 0.0f;
                if (tiny) tiny_output(ts, x, d.n, out.along_i, i, j, f);
#pragma unroll
                for (int pl = 0; pl < kPlanes; ++pl) {
                    if (tiny) break;
                    if (out.along_i == x.turned) {
                        uint32_t v[4];
                        ld_shared_128(x.at(i, j) + pl * x.plane, v[0], v[1], v[2], v[3]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float2 z = unpack_half(v[e]);
                            f[2 * e] += z.x, f[2 * e + 1] += z.y;
                        }
                    } else {  // the caller's array lies the other way
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            unsigned short h;
                            const uint32_t from = out.along_i ? x.at(i + e, j) : x.at(i, j + e);
                            asm volatile("ld.shared.b16 %0, [%1];" : "=h"(h) : "r"(from + pl * x.plane) : "memory");
                            f[e] += __half2float(__ushort_as_half(h));
                        }
                    }
                }
                if (kStep) {
                    float pp[8];
                    p[kStep ? k : 0].get(w.types[kOut], dst.ptr, out.offset(dst, i, j), out.step(dst), count, pp);
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[e] = fmaf(-rate, f[e] * final_scale, pp[e] * w.decay);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[e] *= final_scale;
                }
                out.write(w.types[kOut], dst, (a.direct >> kOut) & 1u, i, j, count, f);
            }
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
