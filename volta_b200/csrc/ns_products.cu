// The products of Newton-Schulz on caller-owned matrices (ns_plan.cu) on the 5th-generation tensor
// cores:   D = e E + f F + g sum_k A[m,k] B[n,k]
// f16 operands staged by TMA (128-byte swizzle), tcgen05.mma with f32 accumulators in TMEM, the
// polynomial's other terms added in the epilogue, D rounded once to f16 (or to two f16 planes).
//
// Every product of the iteration is of this form (see ns_plan.cu): the Gram X X^T, the squares and
// products of short-side matrices, which are polynomials in one Gram, hence symmetric and commuting
// (so B[n,k] may be read for B[k,n], and only tiles on and above the diagonal are computed, the others
// stored as their mirror image), and the update P X, whose B is read "MN-major" from X as it lies.
// The constant term of a polynomial is never folded into an operand: q(G) = a I + R is held as R and
// enters as  a E + R E,  so what is rounded to f16 and what the tensor core accumulates (in f32, with
// truncation) is the correction and not the sum.
//
// All sides are padded to 128 with zeros that reproduce themselves, so nothing is masked here except
// the second half of a 256-row or 256-column tile at the edge.
//
// Warp roles as in ns_gemm_tc.cu: warp 0 TMA producer, warp 1 MMA issuer, warps 2-9 epilogue with two
// accumulators; a persistent grid walks the tile list.  Two shapes:
//   256 x 256 by a CTA pair (cta_group::2): half the operand traffic per FLOP; used when a launch
//             has enough such tiles for the device
//   128 x 128 by one CTA: four times as many tiles, for launches that would leave SMs idle
// Two planes (f32 accuracy): the tensor core adds to its f32 accumulator with truncation, which over a long
// contraction of positive terms (the Gram's diagonal) drifts by 2^-25 per addition: 1.7e-5 on the result
// at n = 2048, one accumulator for the whole sum.  So an accumulator takes 128 of the contraction (24
// additions), and the epilogue warps sum the pieces in registers, correctly rounded, while the next piece runs.
// One plane needs none of that: 65536 / 16 additions drift by less than the operands' rounding.
//
// Every wait is bounded; a wait that runs out sets *error, later kernels of the call then store nothing.
#include <cuda_fp16.h>
#include <algorithm>

#include "ns_plan.h"
#include "tc_ptx.h"

namespace vb {

namespace {

constexpr int BM = 128;
constexpr int BK = 64;  // f16 elements: one 128-byte swizzle row
constexpr int UMMA_K = 16;
constexpr int kBoxBytes = 64 * BK * 2;
constexpr int kRows128Bytes = 128 * BK * 2;
constexpr int kEpiWarps = 8;
constexpr int kFirstEpiWarp = 2;  // warp 0 produces, warp 1 issues
constexpr int kThreads = (kFirstEpiWarp + kEpiWarps) * 32;
constexpr int kStageRowBytes = 128;
constexpr int kStageWarpBytes = 32 * kStageRowBytes;
constexpr uint32_t kDefaultWaitLimit = 1u << 22;
constexpr int kMaxStages = 6;

template <int kCtas, int kPlanes>
struct Cfg {
    static constexpr int BN = 128 * kCtas;
    static constexpr int kStages = kPlanes == 1 ? 6 : 3;
    static constexpr int kPlaneBytes = 2 * kRows128Bytes;  // 128 rows of A, 128 rows of B
    static constexpr int kStageBytes = kPlanes * kPlaneBytes;
    static constexpr int kTmemCols = 2 * BN;
    static constexpr int kChunkBlocks = kPlanes == 1 ? 1 << 20 : 128 / BK;  // k blocks one accumulator takes
};

struct alignas(8) Barriers {
    uint64_t full[kMaxStages];
    uint64_t empty[kMaxStages];
    uint64_t tmem_full[2];
    uint64_t tmem_empty[2];
    uint32_t tmem_base;
    uint32_t abort;
    uint32_t skip;
};
template <int kCtas, int kPlanes>
constexpr size_t smem_bytes()
{
    using C = Cfg<kCtas, kPlanes>;
    return 1024 + (size_t)C::kStages * C::kStageBytes + kEpiWarps * kStageWarpBytes + sizeof(Barriers);
}
static_assert(smem_bytes<2, 1>() <= 232448 && smem_bytes<1, 2>() <= 232448, "a CTA has 227 KiB of shared memory");

// 128 rows x 64 k of one plane: one box of a [rows][k] matrix, or one 64 x 64 x 2 box of [k][rows].
template <int kCtas>
__device__ __forceinline__ void load_rows(uint8_t *dst, const CUtensorMap *map, bool mn_major, int row0, int k0,
                                          int plane_rows, uint32_t bar)
{
    if (mn_major) tma_load_3d<kCtas>(dst, map, 0, k0 + plane_rows, row0 >> 6, bar);
    else tma_load_2d<kCtas>(dst, map, k0, row0 + plane_rows, bar);
}
__device__ __forceinline__ uint64_t operand_desc(uint32_t base, bool mn_major, int kk)
{
    return mn_major ? make_smem_desc(base + kk * 2048, kBoxBytes, 1024) : make_smem_desc(base + kk * 32, 16, 1024);
}
__device__ __forceinline__ uint32_t make_idesc(bool b_mn_major, int m, int n)
{
    // f32 accumulator (bit 4), f16 operands (A and B formats 0), A K-major
    return (1u << 4) | ((uint32_t)b_mn_major << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

struct Tile {
    const NsProduct *p;
    int m0, n0, k_blocks;
    bool mirror, b_mn, skipped;
};
__device__ __forceinline__ Tile fetch_tile(const NsLaunch &l, const uint32_t *active, int t)
{
    Tile ti;
    ti.p = l.problems;
    ti.m0 = ti.n0 = ti.k_blocks = 0;
    ti.mirror = ti.b_mn = false;
    ti.skipped = true;
    if (t < l.n_tiles) {
        const NsTile tile = l.tiles[t];
        const NsProduct *p = l.problems + tile.problem;
        ti.p = p;
        ti.m0 = tile.m0;
        ti.n0 = tile.n0;
        ti.mirror = tile.mirror != 0;
        ti.k_blocks = p->K / BK;
        ti.b_mn = (p->flags & NS_B_MN_MAJOR) != 0;
        ti.skipped = __ldcg(active + p->matrix) == 0u;
    }
    return ti;
}

__device__ __forceinline__ uint32_t pack_half(float a, float b)
{
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 unpack_half(uint32_t w)
{
    return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}

// f[kAt ..] += c * (32 values at src, both planes)
template <int kPlanes, int kSize>
__device__ __forceinline__ void add_term(float (&f)[kSize], int kAt, float c, const __half *src, int64_t plane)
{
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const uint4 q0 = reinterpret_cast<const uint4 *>(src)[g];
        const uint32_t w0[4] = {q0.x, q0.y, q0.z, q0.w};
        uint32_t w1[4] = {0u, 0u, 0u, 0u};
        if (kPlanes == 2) {
            const uint4 q1 = reinterpret_cast<const uint4 *>(src + plane)[g];
            w1[0] = q1.x; w1[1] = q1.y; w1[2] = q1.z; w1[3] = q1.w;
        }
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            float2 x = unpack_half(w0[h]);
            if (kPlanes == 2) {
                const float2 y = unpack_half(w1[h]);
                x.x += y.x;
                x.y += y.y;
            }
            f[kAt + g * 8 + 2 * h] = fmaf(c, x.x, f[kAt + g * 8 + 2 * h]);
            f[kAt + g * 8 + 2 * h + 1] = fmaf(c, x.y, f[kAt + g * 8 + 2 * h + 1]);
        }
    }
}

// Drains kCols columns of 32 accumulator rows (kPlanes == 2: finished values, see the epilogue).  A lane owns one row (TMEM lane = row); row-major stores
// go through the warp's staging buffer so that the warp writes 8 whole 128-byte lines per
// instruction (16-byte pieces of row r sit at position piece ^ (r & 7): no bank conflicts either way).
// Mirrored stores are contiguous along the rows the lanes hold: 64 bytes per instruction.
template <int kPlanes, int kCols>
__device__ __forceinline__ void drain(uint32_t taddr, const NsProduct *p, int row0, int col0, bool mirror, float mult,
                                      int lane, uint32_t stage)
{
    const int64_t ld = p->ld, plane = p->plane_d;
    __half *D = p->D;
    const int r_sub = lane >> 2, seg = lane & 3;
    const uint32_t my_row = stage + (uint32_t)(lane * kStageRowBytes), my_sw = (uint32_t)(lane & 7);
    const uint32_t rd_row = stage + (uint32_t)(r_sub * kStageRowBytes);
    const uint32_t rd_c0 = (uint32_t)(((2 * seg) ^ r_sub) << 4), rd_c1 = (uint32_t)(((2 * seg + 1) ^ r_sub) << 4);
#pragma unroll(kPlanes == 2 ? 1 : kCols / 32)
    for (int cc = 0; cc < kCols / 32; ++cc) {
        uint32_t v[32];
        float f[32];
        tmem_ld_32x32_sync(taddr + (uint32_t)(cc * 32), v);
        const float cg = kPlanes == 2 ? 1.0f : p->g * mult;
#pragma unroll
        for (int j = 0; j < 32; ++j) f[j] = cg * __uint_as_float(v[j]);
        if (kPlanes == 1) {
            const int64_t at = (int64_t)(row0 + lane) * ld + col0 + cc * 32;
            if (p->E != nullptr) add_term<1>(f, 0, p->e * mult, p->E + at, 0);
            if (p->F != nullptr) add_term<1>(f, 0, p->f * mult, p->F + at, 0);
        }
        uint32_t high[16], low[kPlanes == 2 ? 16 : 1];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            high[j] = pack_half(f[2 * j], f[2 * j + 1]);
            if (kPlanes == 2) {  // what the first rounding left over (the difference is exact)
                const float2 h = unpack_half(high[j]);
                low[kPlanes == 2 ? j : 0] = pack_half(f[2 * j] - h.x, f[2 * j + 1] - h.y);
            }
        }
        if (mirror) {
            unsigned short *t = reinterpret_cast<unsigned short *>(D) + (int64_t)(col0 + cc * 32) * ld + row0 + lane;
#pragma unroll
            for (int j = 0; j < 32; ++j) {
                *t = (unsigned short)(j & 1 ? high[j >> 1] >> 16 : high[j >> 1] & 0xffffu);
                if (kPlanes == 2) {
                    const uint32_t w = low[kPlanes == 2 ? j >> 1 : 0];
                    t[plane] = (unsigned short)(j & 1 ? w >> 16 : w & 0xffffu);
                }
                t += ld;
                asm volatile("" : "+l"(t));  // one running address: 32 of them kept across the pieces cost 64 registers
            }
        }
        // one plane: two pieces make a 128-byte line of a row; two planes: a piece's 64 bytes of each
#pragma unroll
        for (int q = 0; q < 4; ++q)
            st_shared_128(my_row + ((((uint32_t)((kPlanes == 1 ? (cc & 1) * 4 : 0) + q)) ^ my_sw) << 4), high[4 * q],
                          high[4 * q + 1], high[4 * q + 2], high[4 * q + 3]);
        if (kPlanes == 2) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
                st_shared_128(my_row + ((((uint32_t)(4 + q)) ^ my_sw) << 4), low[(kPlanes == 2 ? 4 * q : 0)],
                              low[kPlanes == 2 ? 4 * q + 1 : 0], low[kPlanes == 2 ? 4 * q + 2 : 0], low[kPlanes == 2 ? 4 * q + 3 : 0]);
        }
        if (kPlanes == 2 || (cc & 1)) {
            __syncwarp();
#pragma unroll
            for (int pass = 0; pass < 4; ++pass) {
                uint32_t q[8];
                const uint32_t src = rd_row + (uint32_t)(pass * 8 * kStageRowBytes);
                ld_shared_128(src + rd_c0, q[0], q[1], q[2], q[3]);
                ld_shared_128(src + rd_c1, q[4], q[5], q[6], q[7]);
                const int64_t row_at = (int64_t)(row0 + r_sub + 8 * pass) * ld + col0;
                if (kPlanes == 1) st_global_256(D + row_at + (cc - 1) * 32 + seg * 16, q);
                else st_global_256(D + (seg >> 1) * plane + row_at + cc * 32 + (seg & 1) * 16, q);
            }
            __syncwarp();
        }
    }
}

// which role gave up: 1 producer, 2 MMA issuer, 3 epilogue
__device__ __forceinline__ void report(const NsError &error, uint32_t role)
{
    atomicExch(error.device, role);
    *reinterpret_cast<volatile uint32_t *>(error.host) = role;
    __threadfence_system();
}

template <int kCtas, int kPlanes>
__global__ void __launch_bounds__(kThreads, 1)
ns_product_kernel(const NsLaunch launch, const uint32_t *active, const NsError error,
                  uint32_t wait_limit, int withhold)
{
    using C = Cfg<kCtas, kPlanes>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *epi_stage = smem + (size_t)C::kStages * C::kStageBytes;
    Barriers *bars = reinterpret_cast<Barriers *>(epi_stage + kEpiWarps * kStageWarpBytes);
    volatile uint32_t *abort_flag = &bars->abort;

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t cta_rank = kCtas == 2 ? cluster_ctarank() : 0u;
    const int group_id = blockIdx.x / kCtas;
    const int n_groups = gridDim.x / kCtas;
    int n_tiles = launch.n_tiles;

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(&bars->full[s], 1);
            mbar_init(&bars->empty[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(&bars->tmem_full[a], 1);
            mbar_init(&bars->tmem_empty[a], kCtas * kEpiWarps);
        }
        bars->abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        if (kCtas == 2) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                             smem_u32(&bars->tmem_base)),
                         "r"((uint32_t)C::kTmemCols)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                             smem_u32(&bars->tmem_base)),
                         "r"((uint32_t)C::kTmemCols)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    // The launch before this one (programmatic dependency): everything above may overlap its end, everything
    // below reads what it wrote.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (threadIdx.x == 0) bars->skip = *reinterpret_cast<volatile uint32_t *>(error.device);
    tcgen05_fence_before();
    __syncthreads();
    if (kCtas == 2) cluster_sync_all();
    tcgen05_fence_after();
    const uint32_t tmem_base = bars->tmem_base;
    // an earlier kernel gave up a wait: its output is half written, so nothing is computed from it.  Both
    // CTAs of a pair read the same word after that kernel's end, so they agree.
    if (bars->skip != 0u) n_tiles = 0;

    if (warp == 0) {
        // ---- TMA producer: lane 0 fetches A and announces the bytes, lane 1 fetches B ----
        if (lane < 2) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            Tile next = fetch_tile(launch, active, n_tiles > 0 ? group_id : launch.n_tiles);
            for (int t = group_id; t < n_tiles && ok; t += n_groups) {
                const Tile ti = next;
                next = fetch_tile(launch, active, t + n_groups);
                if (ti.skipped) continue;
                const int a_row0 = ti.m0 + (int)cta_rank * BM, b_row0 = ti.n0 + (int)cta_rank * 128;
                const int plane_rows = lane == 0 ? ti.p->plane_rows_a : ti.p->plane_rows_b;
                for (int kb = 0; kb < ti.k_blocks; ++kb) {
                    if (!__all_sync(0x3u, mbar_wait(&bars->empty[stage], phase ^ 1u, abort_flag, wait_limit))) {
                        ok = false;
                        break;
                    }
                    uint8_t *slot = smem + (size_t)stage * C::kStageBytes;
                    const uint32_t full_bar =
                        kCtas == 2 ? map_to_cta(smem_u32(&bars->full[stage]), 0) : smem_u32(&bars->full[stage]);
                    if (withhold) {
                        // nothing is announced or staged: the bounded waits run out
                    } else if (lane == 0) {
                        if (cta_rank == 0) mbar_expect_tx(&bars->full[stage], kCtas * C::kStageBytes);
#pragma unroll
                        for (int pl = 0; pl < kPlanes; ++pl)
                            load_rows<kCtas>(slot + pl * C::kPlaneBytes, &ti.p->map_a, false, a_row0, kb * BK,
                                             pl * plane_rows, full_bar);
                    } else {
#pragma unroll
                        for (int pl = 0; pl < kPlanes; ++pl)
                            load_rows<kCtas>(slot + pl * C::kPlaneBytes + kRows128Bytes, &ti.p->map_b, ti.b_mn, b_row0,
                                             kb * BK, pl * plane_rows, full_bar);
                    }
                    if (++stage == C::kStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            if (!ok) {
                bars->abort = 1;
                report(error, 1u);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ---- MMA issuer (leader CTA) ----
        if (lane == 0 && cta_rank == 0) {
            int stage = 0, acc = 0;
            uint32_t phase = 0, acc_phase = 0;
            bool ok = true;
            Tile next = fetch_tile(launch, active, n_tiles > 0 ? group_id : launch.n_tiles);
            for (int t = group_id; t < n_tiles && ok; t += n_groups) {
                const Tile ti = next;
                next = fetch_tile(launch, active, t + n_groups);
                if (ti.skipped) continue;
                const uint32_t idesc = make_idesc(ti.b_mn, BM * kCtas, C::BN);
                for (int k0 = 0; k0 < ti.k_blocks && ok; k0 += C::kChunkBlocks) {
                    const int k1 = min(k0 + C::kChunkBlocks, ti.k_blocks);
                    if (!mbar_wait(&bars->tmem_empty[acc], acc_phase ^ 1u, abort_flag, wait_limit)) {
                        ok = false;
                        break;
                    }
                    tcgen05_fence_after();
                    const uint32_t tmem_d = tmem_base + (uint32_t)(acc * C::BN);
                    for (int kb = k0; kb < k1; ++kb) {
                        if (!mbar_wait(&bars->full[stage], phase, abort_flag, wait_limit)) {
                            ok = false;
                            break;
                        }
                        tcgen05_fence_after();
                        const uint32_t base = smem_u32(smem + (size_t)stage * C::kStageBytes);
                        // two planes: three products, smallest first; the dropped low x low is below 2^-22
#pragma unroll
                        for (int term = 0; term < (kPlanes == 2 ? 3 : 1); ++term) {
                            const uint32_t sa = base + (kPlanes == 2 && term == 1 ? C::kPlaneBytes : 0);
                            const uint32_t sb = base + kRows128Bytes + (kPlanes == 2 && term == 0 ? C::kPlaneBytes : 0);
#pragma unroll
                            for (int kk = 0; kk < BK / UMMA_K; ++kk)
                                tcgen05_mma_bf16<kCtas>(tmem_d, operand_desc(sa, false, kk), operand_desc(sb, ti.b_mn, kk),
                                                        idesc, (kb > k0 || term > 0 || kk > 0) ? 1u : 0u);
                        }
                        tcgen05_commit<kCtas>(&bars->empty[stage]);
                        if (++stage == C::kStages) {
                            stage = 0;
                            phase ^= 1u;
                        }
                    }
                    if (!ok) break;
                    tcgen05_commit<kCtas>(&bars->tmem_full[acc]);
                    if (++acc == 2) {
                        acc = 0;
                        acc_phase ^= 1u;
                    }
                }
            }
            if (!ok) {
                bars->abort = 1;
                report(error, 2u);
            }
        }
        __syncwarp();
    } else if (warp >= kFirstEpiWarp) {
        // ---- epilogue: warp w reads TMEM lane quarter w % 4 and half of the columns ----
        constexpr int kCols = C::BN / 2;
        const int quarter = warp & 3, col_half = (warp - kFirstEpiWarp) >> 2;
        const uint32_t my_stage = smem_u32(epi_stage) + (uint32_t)((warp - kFirstEpiWarp) * kStageWarpBytes);
        int acc = 0;
        uint32_t acc_phase = 0;
        bool ok = true;
        Tile next = fetch_tile(launch, active, n_tiles > 0 ? group_id : launch.n_tiles);
        for (int t = group_id; t < n_tiles && ok; t += n_groups) {
            const Tile ti = next;
            next = fetch_tile(launch, active, t + n_groups);
            if (ti.skipped) continue;
            const NsProduct *p = ti.p;
            float mult = 1.0f;
            if (p->scale_power != 0) {
                mult = *p->scale;
                if (p->scale_power == 2) mult *= mult;
            }
            const int row0 = ti.m0 + (int)cta_rank * BM + quarter * 32;
            const int col0 = ti.n0 + col_half * kCols;
            // extents are multiples of 128: a warp's piece is all in or all out
            const bool inside = row0 < p->M && col0 < p->N;
            float sum[kPlanes == 2 ? kCols : 1];
            if (kPlanes == 2) {  // the polynomial's other terms first: their loads overlap the first products
                const int64_t at = (int64_t)(row0 + lane) * p->ld + col0;
#pragma unroll
                for (int j = 0; j < kCols; ++j) sum[kPlanes == 2 ? j : 0] = 0.0f;
                if (inside && p->E != nullptr) {
#pragma unroll
                    for (int cc = 0; cc < kCols / 32; ++cc) {
                        add_term<2>(sum, kPlanes == 2 ? cc * 32 : 0, p->e * mult, p->E + at + cc * 32, p->plane_d);
                        asm volatile("" ::: "memory");  // no more than a piece's loads in registers at once
                    }
                }
                if (inside && p->F != nullptr) {
#pragma unroll
                    for (int cc = 0; cc < kCols / 32; ++cc) {
                        add_term<2>(sum, kPlanes == 2 ? cc * 32 : 0, p->f * mult, p->F + at + cc * 32, p->plane_d);
                        asm volatile("" ::: "memory");
                    }
                }
            }
            const float cg = p->g * mult;
            for (int k0 = 0; k0 < ti.k_blocks && ok; k0 += C::kChunkBlocks) {
                if (!__all_sync(0xffffffffu, mbar_wait(&bars->tmem_full[acc], acc_phase, abort_flag, wait_limit))) {
                    ok = false;
                    break;
                }
                tcgen05_fence_after();
                const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(acc * C::BN + col_half * kCols);
                if (kPlanes == 1) {
                    if (inside) drain<kPlanes, kCols>(taddr, p, row0, col0, ti.mirror, mult, lane, my_stage);
                } else {
#pragma unroll
                    for (int cc = 0; cc < kCols / 32; ++cc) {
                        uint32_t v[32];
                        tmem_ld_32x32_sync(taddr + (uint32_t)(cc * 32), v);
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            sum[kPlanes == 2 ? cc * 32 + j : 0] =
                                fmaf(cg, __uint_as_float(v[j]), sum[kPlanes == 2 ? cc * 32 + j : 0]);
                    }
                    if (k0 + C::kChunkBlocks >= ti.k_blocks && inside) {
                        // finished: back into this warp's part of the accumulator, drained from there piece by piece
#pragma unroll
                        for (int cc = 0; cc < kCols / 32; ++cc) {
                            uint32_t v[32];
#pragma unroll
                            for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(sum[kPlanes == 2 ? cc * 32 + j : 0]);
                            tmem_st_32x32(taddr + (uint32_t)(cc * 32), v);
                        }
                        tmem_st_wait();
                        drain<kPlanes, kCols>(taddr, p, row0, col0, ti.mirror, mult, lane, my_stage);
                    }
                }
                tcgen05_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (kCtas == 2) mbar_remote_arrive(map_to_cta(smem_u32(&bars->tmem_empty[acc]), 0));
                    else mbar_arrive(&bars->tmem_empty[acc]);
                }
                if (++acc == 2) {
                    acc = 0;
                    acc_phase ^= 1u;
                }
            }
        }
        if (!ok && lane == 0) {
            bars->abort = 1;
            report(error, 3u);
        }
        __syncwarp();
    }

    tcgen05_fence_before();
    __syncthreads();
    if (bars->abort != 0 && threadIdx.x == 0) {
        // copies that may still be in flight get a bounded time to land before shared memory is released
        for (int s = 0; s < C::kStages; ++s)
            for (uint32_t i = 0; i < 4096u; ++i)
                if (mbar_try_wait(&bars->full[s], 0) || mbar_try_wait(&bars->full[s], 1)) break;
    }
    __syncthreads();
    if (kCtas == 2) cluster_sync_all();
    if (warp == 1) {
        tcgen05_fence_after();
        if (kCtas == 2)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base),
                         "r"((uint32_t)C::kTmemCols)
                         : "memory");
        else
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base),
                         "r"((uint32_t)C::kTmemCols)
                         : "memory");
    }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                  const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

template <int kCtas, int kPlanes>
int launch_variant(const NsLaunch &l, const uint32_t *d_active, NsError error, int sm_count, cudaStream_t stream,
                   uint32_t wait_limit, bool withhold)
{
    const size_t smem = smem_bytes<kCtas, kPlanes>();
    VB_CUDA(cudaFuncSetAttribute(ns_product_kernel<kCtas, kPlanes>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = kCtas;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = kCtas == 2 ? 2 : 1;
    // groups never wait for one another, so a grid larger than the device holds would still be right
    const int groups = std::min(sm_count / kCtas, l.n_tiles);
    cfg.gridDim = dim3((unsigned)(groups * kCtas));
    VB_CUDA(cudaLaunchKernelEx(&cfg, ns_product_kernel<kCtas, kPlanes>, l, d_active, error, wait_limit, withhold ? 1 : 0));
    return VB_OK;
}

}  // namespace

void ns_tile_extent(int shape, int *bm, int *bn) { *bm = *bn = shape == NS_TILE_PAIR_256 ? 256 : 128; }

// Tensor map over a row-major f16 matrix [outer][inner], 128-byte swizzle: 64 x 128 boxes, or (mn_major)
// 64 x 64 x 2 boxes of the 3-D view [inner / 64][outer][64].
int make_ns_map(CUtensorMap *map, const void *base, int64_t inner, int64_t outer, bool mn_major)
{
    static EncodeTiledFn fn = nullptr;
    if (!fn) {
        void *sym = nullptr;
        cudaDriverEntryPointQueryResult qres;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &qres) == cudaSuccess &&
            qres == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(sym);
    }
    if (!fn) return fail(VB_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
    CUresult r;
    cuuint32_t estr[3] = {1, 1, 1};
    if (mn_major) {
        cuuint64_t dims[3] = {64, (cuuint64_t)outer, (cuuint64_t)(inner / 64)};
        cuuint64_t strides[2] = {(cuuint64_t)inner * 2, 128};
        cuuint32_t box[3] = {64, 64, 2};
        r = fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void *>(base), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    } else {
        cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)outer};
        cuuint64_t strides[1] = {(cuuint64_t)inner * 2};
        cuuint32_t box[2] = {64, 128};
        r = fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void *>(base), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    }
    if (r != CUDA_SUCCESS) return fail(VB_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
    return VB_OK;
}

int launch_ns_products(const NsLaunch &l, int shape, int planes, const uint32_t *d_active, NsError error,
                       int sm_count, cudaStream_t stream, uint32_t wait_limit, bool withhold)
{
    if (l.n_tiles <= 0) return VB_OK;
    if (wait_limit == 0) wait_limit = kDefaultWaitLimit;
    if (shape == NS_TILE_PAIR_256)
        return planes == 2 ? launch_variant<2, 2>(l, d_active, error, sm_count, stream, wait_limit, withhold)
                           : launch_variant<2, 1>(l, d_active, error, sm_count, stream, wait_limit, withhold);
    return planes == 2 ? launch_variant<1, 2>(l, d_active, error, sm_count, stream, wait_limit, withhold)
                       : launch_variant<1, 1>(l, d_active, error, sm_count, stream, wait_limit, withhold);
}

}  // namespace vb
