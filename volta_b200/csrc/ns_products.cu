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
// One persistent, cooperative launch runs all stages of all matrices: every CTA (pair) walks a list of tiles
// that the planner made for it, and a tile starts once all tiles of the same matrix's earlier stages are
// stored (a counter per matrix; release by the storing warps, acquire by the loading ones).  The lists follow
// one order of all tiles in which a tile comes after those it waits for, and all CTAs are resident, so the
// first unfinished tile can always run.  Against one launch per stage this saves the launches' fill and drain
// (10 us a stage for a 256 x 784 matrix by itself) and lets other matrices' tiles fill the gaps between the
// stages of one.
//
// Warp roles as in ns_gemm_tc.cu: warp 0 TMA producer, warp 1 MMA issuer, warps 2-9 epilogue with two
// accumulators.  Two shapes:
//   256 x 256 (two planes: 256 x 128) by a CTA pair (cta_group::2): half the operand traffic per FLOP; the mainloop runs
//             at the tensor core's rate (512 cycles per 64 of the contraction), large products at 1.0 to 1.15 PFLOP/s under
//             the power cap (1.45 to 1.55 GHz).  Two planes do three products on what they load; there 256 columns
//             only cost registers (the sums spilled) and parallelism (2048 x 2048 f32: 870 us against 785)
//   128 x 128 by one CTA: four times as many tiles, for lists that would leave SMs idle
// (the planner picks, see pick_shape).
//
// Epilogue.  A warp owns 32 accumulator rows and takes them 64 columns at a time: TMEM -> registers, the
// terms E and F from its own shared-memory buffer (fetched by TMA while the products run), rounding, D into
// another buffer and from there by TMA to memory; the transposed piece of a symmetric product is built in a
// third (neighbouring lanes exchange halves, so each lane writes words) and stored the same way.  With plain
// loads and stores from registers (a lane per row) a 256 x 256 tile's epilogue took 10 to 13 thousand cycles
// and a fence 3 thousand, against 8 thousand for the products at k = 1024: it, not the tensor core, set the pace.
//
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
constexpr int BK = kNsKBlock;  // f16 elements: one 128-byte swizzle row
constexpr int UMMA_K = 16;
constexpr int kBoxBytes = 64 * BK * 2;
constexpr int kRows128Bytes = 128 * BK * 2;
constexpr int kEpiWarps = 8;
constexpr int kFirstEpiWarp = 2;  // warp 0 produces, warp 1 issues
constexpr int kThreads = (kFirstEpiWarp + kEpiWarps) * 32;
constexpr int kPieceCols = 64;
constexpr int kPieceBytes = 32 * kPieceCols * 2;  // 32 rows of 128 bytes, 16-byte parts of row r at part ^ (r & 7)
constexpr int kMaxStages = 5;
constexpr int kSmemBytes = 232448 - 2048;  // 227 KiB less alignment and barriers

template <int kCtas, int kPlanes>
struct Cfg {
    static constexpr int BN = kCtas == 2 && kPlanes == 1 ? 256 : 128;  // columns of a tile
    static constexpr int kBRows = BN / kCtas;                           // rows of B a CTA stages
    static constexpr int kPlaneBytes = kRows128Bytes + kBRows * BK * 2;  // 128 rows of A, kBRows of B
    static constexpr int kStageBytes = kPlanes * kPlaneBytes;
    // An epilogue warp's buffers: a term, a second term or the mirrored result, and, where it has more pieces than one
    // per tile (so that the next term arrives while a result leaves), a separate one for the result.
    static constexpr int kEpiBuffers = BN / 2 > kPieceCols ? 3 : 2;
    static constexpr int kEpiWarpBytes = kEpiBuffers * kPieceBytes;
    static constexpr int kStages = (kSmemBytes - kEpiWarps * kEpiWarpBytes) / kStageBytes < kMaxStages
                                       ? (kSmemBytes - kEpiWarps * kEpiWarpBytes) / kStageBytes
                                       : kMaxStages;
    static constexpr int kTmemCols = 2 * BN;
    static constexpr int kChunkBlocks = kPlanes == 1 ? 1 << 20 : 128 / BK;  // k blocks one accumulator takes
};

struct alignas(8) Barriers {
    uint64_t full[kMaxStages];
    uint64_t empty[kMaxStages];
    uint64_t tmem_full[2];
    uint64_t tmem_empty[2];
    uint64_t term_full[2 * kEpiWarps];
    uint32_t tmem_base;
    uint32_t abort;
    uint32_t skip;
};
template <int kCtas, int kPlanes>
constexpr size_t smem_bytes()
{
    using C = Cfg<kCtas, kPlanes>;
    return 1024 + (size_t)C::kStages * C::kStageBytes + kEpiWarps * C::kEpiWarpBytes + sizeof(Barriers);
}
static_assert(smem_bytes<2, 1>() <= 232448 && smem_bytes<1, 2>() <= 232448, "a CTA has 227 KiB of shared memory");

// 128 rows x 64 k of one plane: one box of a [rows][k] matrix, or one 64 x 64 x 2 box of [k][rows].
template <int kCtas>
__device__ __forceinline__ void load_rows(uint32_t dst, const CUtensorMap *map, bool mn_major, int row0, int k0,
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
    int m0, n0, kb0, kb1, matrix, part, parts;
    uint32_t after;
    bool mirror, shared, b_mn, skipped;
};
__device__ __forceinline__ Tile fetch_tile(const NsLaunch &l, const uint32_t *active, int t, int end)
{
    Tile ti;
    ti.p = l.problems;
    ti.m0 = ti.n0 = ti.kb0 = ti.kb1 = ti.matrix = ti.parts = 0;
    ti.part = -1;
    ti.after = 0;
    ti.mirror = ti.shared = ti.b_mn = false;
    ti.skipped = true;
    if (t < end) {
        const NsTile tile = l.tiles[t];
        const NsProduct *p = l.problems + tile.problem;
        ti.p = p;
        ti.m0 = tile.m0;
        ti.n0 = tile.n0;
        ti.mirror = (tile.flags & NS_TILE_MIRROR) != 0;
        ti.shared = (tile.flags & NS_TILE_SHARED) != 0;
        ti.after = tile.after;
        ti.matrix = p->matrix;
        ti.kb0 = tile.kb0;
        ti.kb1 = tile.kb1;
        ti.part = tile.part;
        ti.parts = tile.parts;
        ti.b_mn = (p->flags & NS_B_MN_MAJOR) != 0;
        ti.skipped = __ldcg(active + p->matrix) == 0u;
    }
    return ti;
}

__device__ __forceinline__ Tile uniform_tile(const Tile &t)
{
    Tile u;
    u.p = uniform(const_cast<NsProduct *>(t.p));
    u.m0 = uniform(t.m0);
    u.n0 = uniform(t.n0);
    u.kb0 = uniform(t.kb0);
    u.kb1 = uniform(t.kb1);
    u.part = uniform(t.part);
    u.parts = uniform(t.parts);
    u.matrix = uniform(t.matrix);
    u.after = uniform(t.after);
    const int flags = uniform((t.mirror ? 1 : 0) | (t.b_mn ? 2 : 0) | (t.skipped ? 4 : 0) | (t.shared ? 8 : 0));
    u.mirror = flags & 1, u.b_mn = flags & 2, u.skipped = flags & 4, u.shared = flags & 8;
    return u;
}

__device__ __forceinline__ uint32_t load_acquire(const uint32_t *p)
{
    uint32_t v;
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}
// Waits until the matrix's earlier stages are stored.  Bounded, and given up as soon as any CTA reported an error.
__device__ __forceinline__ bool wait_stored(const uint32_t *counter, uint32_t target, const uint32_t *error,
                                            volatile uint32_t *abort_flag, uint32_t wait_limit)
{
    if (target == 0u) return true;
    for (uint32_t i = 0; i < wait_limit; ++i) {
        if (load_acquire(counter) >= target) return true;
        if ((i & 31u) == 31u) {
            if (*abort_flag != 0u || *reinterpret_cast<const volatile uint32_t *>(error) != 0u) return false;
            __nanosleep(64);
        }
    }
    return false;
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

__device__ __forceinline__ void tma_store_2d(const CUtensorMap *map, uint32_t smem_src, int c0, int c1)
{
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                     reinterpret_cast<uint64_t>(map)),
                 "r"(c0), "r"(c1), "r"(smem_src)
                 : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap *map)
{
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// The warp's share of one tile: kCols columns of 32 rows.
template <int kPlanes, int kCols>
struct Drain {
    static constexpr int kResult = kCols > kPieceCols ? kPieceBytes : 0;  // offsets of the buffers
    static constexpr int kMirror = kResult + kPieceBytes;
    const NsProduct *p;
    uint8_t *buffers;     // this warp's
    uint64_t *term_full;  // this warp's two barriers
    uint32_t &term_phase; // bit b: phase of barrier b
    int row0, col0, lane;
    int per_piece;        // loads of a piece: terms x planes
    bool mirror;

    // Load r of a piece: E before F, plane 0 before plane 1.  Even ones go to the term buffer, odd ones to the mirror
    // buffer, which must have been stored from by then.
    __device__ __forceinline__ void fetch(int piece, int r) const
    {
        if (lane != 0 || r >= per_piece || piece >= kCols / kPieceCols) return;
        uint64_t *full = term_full + (r & 1);
        mbar_expect_tx(full, kPieceBytes);
        tma_load_2d<1>(buffers + (r & 1) * kMirror, &p->map_term[r / kPlanes], col0 + piece * kPieceCols,
                       row0 + (r % kPlanes) * p->plane_rows, smem_u32(full));
    }
    // one plane of a finished piece: h[k] holds columns 2k and 2k + 1 of this lane's row
    __device__ __forceinline__ void store(const uint32_t (&h)[32], int piece, int plane) const
    {
        if (lane == 0) bulk_wait_read();  // the stores before this one have left the buffers
        __syncwarp();
        const uint32_t out = smem_u32(buffers) + kResult, row = out + (uint32_t)(lane * 128);
#pragma unroll
        for (int q = 0; q < 8; ++q)
            st_shared_128(row + (uint32_t)((q ^ (lane & 7)) << 4), h[4 * q], h[4 * q + 1], h[4 * q + 2], h[4 * q + 3]);
        const uint32_t turned = smem_u32(buffers) + kMirror;
        if (mirror) {
            // column 2k (even lanes) or 2k + 1 (odd lanes), rows of a pair of lanes: 32 words of two 64-byte rows
            const uint32_t word = turned + (uint32_t)((lane & 1) * 64 + (lane >> 1) * 4);
            const uint32_t pick = (lane & 1) ? 0x3276u : 0x5410u;  // {other.hi, own.hi} or {own.lo, other.lo}
#pragma unroll
            for (int k = 0; k < 32; ++k) {
                const uint32_t other = __shfl_xor_sync(0xffffffffu, h[k], 1);
                const uint32_t w = __byte_perm(h[k], other, pick);
                asm volatile("st.shared.b32 [%0], %1;" ::"r"(word + (uint32_t)(k * 128)), "r"(w) : "memory");
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
            const int c = col0 + piece * kPieceCols, off = plane * p->plane_rows;
            tma_store_2d(&p->map_d, out, c, row0 + off);
            if (mirror) tma_store_2d(&p->map_mirror, turned, row0, c + off);
            bulk_commit();
        }
    }
    // Returns false if a term did not arrive.  `drained` is called once the accumulator has been read.
    template <typename Fn>
    __device__ __forceinline__ bool run(uint32_t taddr, float mult, volatile uint32_t *abort_flag, uint32_t wait_limit,
                                        Fn &&drained)
    {
        const float cg = p->g * mult;
#pragma unroll 1
        for (int piece = 0; piece < kCols / kPieceCols; ++piece) {
            if (piece > 0 && per_piece > 1) {
                if (lane == 0) bulk_wait_read();
                fetch(piece, 1);
            }
            float f[kPieceCols];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t v[32];
                tmem_ld_32x32_sync(taddr + (uint32_t)(piece * kPieceCols + half * 32), v);
#pragma unroll
                for (int j = 0; j < 32; ++j) f[half * 32 + j] = cg * __uint_as_float(v[j]);
            }
            if (piece + 1 == kCols / kPieceCols) drained();
#pragma unroll 1
            for (int r = 0; r < per_piece; ++r) {
                const int buf = r & 1;
                if (!__all_sync(0xffffffffu, mbar_wait(term_full + buf, (term_phase >> buf) & 1u, abort_flag, wait_limit))) return false;
                term_phase ^= 1u << buf;
                const float c = p->term[r / kPlanes] * mult;
                const uint32_t row = smem_u32(buffers) + (uint32_t)(buf * kMirror + lane * 128);
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    uint32_t w[4];
                    ld_shared_128(row + (uint32_t)((q ^ (lane & 7)) << 4), w[0], w[1], w[2], w[3]);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float2 x = unpack_half(w[k]);
                        f[q * 8 + 2 * k] = fmaf(c, x.x, f[q * 8 + 2 * k]);
                        f[q * 8 + 2 * k + 1] = fmaf(c, x.y, f[q * 8 + 2 * k + 1]);
                    }
                }
                __syncwarp();
                if (r + 2 < per_piece) fetch(piece, r + 2);
                else if (buf == 0) fetch(piece + 1, 0);
            }
            uint32_t h[32];
#pragma unroll
            for (int k = 0; k < 32; ++k) {
                h[k] = pack_half(f[2 * k], f[2 * k + 1]);
                if (kPlanes == 2) {  // what the rounding left over (the difference is exact)
                    const float2 x = unpack_half(h[k]);
                    f[2 * k] -= x.x;
                    f[2 * k + 1] -= x.y;
                }
            }
            store(h, piece, 0);
            if (kPlanes == 2) {
#pragma unroll
                for (int k = 0; k < 32; ++k) h[k] = pack_half(f[2 * k], f[2 * k + 1]);
                store(h, piece, 1);
            }
        }
        return true;
    }
};

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
    Barriers *bars = reinterpret_cast<Barriers *>(epi_stage + kEpiWarps * C::kEpiWarpBytes);
    volatile uint32_t *abort_flag = &bars->abort;

    const int warp = uniform((int)(threadIdx.x >> 5));
    const int lane = threadIdx.x & 31;
    const uint32_t cta_rank = kCtas == 2 ? cluster_ctarank() : 0u;
    const int first_tile = launch.begin[blockIdx.x / kCtas];
    int end = launch.begin[blockIdx.x / kCtas + 1];
    constexpr uint32_t kArrivals = kCtas * kEpiWarps;  // on a matrix's counter, per tile

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(&bars->full[s], 1);
            mbar_init(&bars->empty[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(&bars->tmem_full[a], 1);
            mbar_init(&bars->tmem_empty[a], kCtas * kEpiWarps);
        }
        for (int w = 0; w < 2 * kEpiWarps; ++w) mbar_init(&bars->term_full[w], 1);
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
    if (threadIdx.x == 0) bars->skip = *reinterpret_cast<volatile uint32_t *>(error.device);
    tcgen05_fence_before();
    __syncthreads();
    if (kCtas == 2) cluster_sync_all();
    tcgen05_fence_after();
    const uint32_t tmem_base = bars->tmem_base;
    if (bars->skip != 0u) end = first_tile;  // an earlier call gave up a wait

    if (warp == 0) {
        // ---- TMA producer ----
        const bool elected = elect_one();
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        const uint32_t slots = uniform(smem_u32(smem)), empty0 = uniform(smem_u32(&bars->empty[0]));
        // the leader announces the bytes of both CTAs; the peer's may land before that, the phase cannot end before it
        const uint32_t my_full0 = uniform(smem_u32(&bars->full[0]));
        const uint32_t full0 = uniform(kCtas == 2 ? map_to_cta(my_full0, 0) : my_full0);
        Tile next = fetch_tile(launch, active, first_tile, end);
        for (int t = first_tile; t < end && ok; ++t) {
            const Tile ti = uniform_tile(next);
            next = fetch_tile(launch, active, t + 1, end);
            if (ti.skipped) continue;
            const int a_row0 = ti.m0 + (int)cta_rank * BM, b_row0 = ti.n0 + (int)cta_rank * C::kBRows;
            const int plane_rows = uniform(ti.p->plane_rows);
            const CUtensorMap *map_a = &ti.p->map_a, *map_b = &ti.p->map_b;
            if (elected) {
                prefetch_map(map_a);
                prefetch_map(map_b);
            }
            if (!__all_sync(0xffffffffu, wait_stored(launch.stored + ti.matrix, ti.after * kArrivals, error.device, abort_flag,
                                                     wait_limit))) {
                ok = false;
                break;
            }
            asm volatile("fence.proxy.async.global;" ::: "memory");  // TMA reads what other SMs stored
#pragma unroll 1
            for (int kb = ti.kb0; kb < ti.kb1; ++kb) {
                if (!__all_sync(0xffffffffu, mbar_wait(empty0 + 8 * stage, phase ^ 1u, abort_flag, wait_limit))) {
                    ok = false;
                    break;
                }
                if (elected && !withhold) {  // withheld: nothing is announced or staged, the bounded waits run out
                    const uint32_t slot = slots + (uint32_t)stage * C::kStageBytes, full = full0 + 8 * stage;
                    if (cta_rank == 0)
                        mbar_expect_tx(my_full0 + 8 * stage, kCtas * (ti.shared ? kPlanes * kRows128Bytes : C::kStageBytes));
#pragma unroll
                    for (int pl = 0; pl < kPlanes; ++pl) {
                        load_rows<kCtas>(slot + pl * C::kPlaneBytes, map_a, false, a_row0, kb * BK, pl * plane_rows, full);
                        if (!ti.shared)
                            load_rows<kCtas>(slot + pl * C::kPlaneBytes + kRows128Bytes, map_b, ti.b_mn, b_row0, kb * BK,
                                             pl * plane_rows, full);
                    }
                }
                if (++stage == C::kStages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
        }
        if (!ok && lane == 0) {
            bars->abort = 1;
            report(error, 1u);
        }
        __syncwarp();
    } else if (warp == 1) {
        // ---- MMA issuer (leader CTA) ----
        if (cta_rank == 0) {
            const bool elected = elect_one();
            int stage = 0, acc = 0;
            uint32_t phase = 0, acc_phase = 0;
            bool ok = true;
            // descriptors are made once (for slot 0) and moved by adding 16-byte units to their address field
            const uint32_t base = uniform(smem_u32(smem));
            const uint64_t desc_k = operand_desc(base, false, 0), desc_mn = operand_desc(base, true, 0);
            const uint32_t full0 = uniform(smem_u32(&bars->full[0])), empty0 = uniform(smem_u32(&bars->empty[0]));
            const uint32_t tmem = uniform(tmem_base);
            Tile next = fetch_tile(launch, active, first_tile, end);
            for (int t = first_tile; t < end && ok; ++t) {
                const Tile ti = uniform_tile(next);
                next = fetch_tile(launch, active, t + 1, end);
                if (ti.skipped) continue;
                const uint32_t idesc = make_idesc(ti.b_mn, BM * kCtas, C::BN);
                // B's descriptor differs by its major-ness in the fields above the address and in the step of a k slice
                const uint64_t desc_b0 = (ti.b_mn ? desc_mn : desc_k) + (ti.shared ? 0 : kRows128Bytes >> 4);
                const uint32_t step_b = ti.b_mn ? 2048 >> 4 : 32 >> 4;
                // (a tile that sums pieces has nothing to multiply: one round that hands the accumulator over)
                for (int k0 = ti.kb0; (k0 < ti.kb1 || k0 == ti.kb0) && ok; k0 += C::kChunkBlocks) {
                    const int k1 = min(k0 + C::kChunkBlocks, ti.kb1);
                    if (!__all_sync(0xffffffffu, mbar_wait(&bars->tmem_empty[acc], acc_phase ^ 1u, abort_flag, wait_limit))) {
                        ok = false;
                        break;
                    }
                    tcgen05_fence_after();
                    const uint32_t tmem_d = tmem + (uint32_t)(acc * C::BN);
                    if (k0 >= k1 && elected) tcgen05_commit<kCtas>(&bars->tmem_full[acc]);
                    bool ready = false;
#pragma unroll 1
                    for (int kb = k0; kb < k1; ++kb) {
                        if (!ready && !__all_sync(0xffffffffu, mbar_wait(full0 + 8 * stage, phase, abort_flag, wait_limit))) {
                            ok = false;
                            break;
                        }
                        tcgen05_fence_after();
                        const uint32_t slot = (uint32_t)stage * (C::kStageBytes >> 4), used = empty0 + 8 * stage;
                        if (++stage == C::kStages) {
                            stage = 0;
                            phase ^= 1u;
                        }
                        // a look at the next slot's barrier, answered while this one's products are issued
                        const bool peek = kb + 1 < k1 && mbar_try_wait(full0 + 8 * stage, phase);
                        if (elected) {
                            // two planes: three products, smallest first; the dropped low x low is below 2^-22
#pragma unroll
                            for (int term = 0; term < (kPlanes == 2 ? 3 : 1); ++term) {
                                const uint64_t da = desc_k + slot + (kPlanes == 2 && term == 1 ? C::kPlaneBytes >> 4 : 0);
                                const uint64_t db = desc_b0 + slot + (kPlanes == 2 && term == 0 ? C::kPlaneBytes >> 4 : 0);
#pragma unroll
                                for (int kk = 0; kk < BK / UMMA_K; ++kk)
                                    tcgen05_mma_bf16<kCtas>(tmem_d, da + kk * (32 >> 4), db + kk * step_b, idesc,
                                                            (kb > k0 || term > 0 || kk > 0) ? 1u : 0u);
                            }
                            tcgen05_commit<kCtas>(used);
                            if (kb + 1 == k1) tcgen05_commit<kCtas>(&bars->tmem_full[acc]);
                        }
                        ready = __all_sync(0xffffffffu, peek);
                    }
                    if (!ok) break;
                    acc ^= 1;
                    acc_phase ^= acc == 0 ? 1u : 0u;
                }
            }
            if (!ok && lane == 0) {
                bars->abort = 1;
                report(error, 2u);
            }
        }
        __syncwarp();
    } else if (warp >= kFirstEpiWarp) {
        // ---- epilogue: warp w reads TMEM lane quarter w % 4 and half of the columns ----
        constexpr int kCols = C::BN / 2;
        const int quarter = warp & 3, col_half = (warp - kFirstEpiWarp) >> 2;
        uint8_t *const my_buffers = epi_stage + (size_t)(warp - kFirstEpiWarp) * C::kEpiWarpBytes;
        uint64_t *const term_full = &bars->term_full[2 * (warp - kFirstEpiWarp)];
        uint32_t term_phase = 0;
        int acc = 0;
        uint32_t acc_phase = 0;
        bool ok = true;
        Tile next = fetch_tile(launch, active, first_tile, end);
        for (int t = first_tile; t < end && ok; ++t) {
            const Tile ti = next;
            next = fetch_tile(launch, active, t + 1, end);
            if (ti.skipped) continue;
            const NsProduct *p = ti.p;
            float mult = 1.0f;
            if (p->scale_power != 0) {
                mult = *p->scale;
                if (p->scale_power == 2) mult *= mult;
            }
            const int row0 = ti.m0 + (int)cta_rank * BM + quarter * 32;
            const int col0 = ti.n0 + col_half * kCols;
            // extents are multiples of 128: a warp's share is all in or all out
            const bool inside = row0 < p->M && col0 < p->N;
            Drain<kPlanes, kCols> drain{p, my_buffers, term_full, term_phase, row0, col0, lane, p->n_terms * kPlanes, ti.mirror};
            if (lane == 0) {
                if (p->n_terms > 0) prefetch_map(&p->map_term[0]);
                prefetch_map(&p->map_d);
            }
            if (inside && !(ti.part >= 0 && ti.parts == 0) && drain.per_piece > 0) {  // the first term: its matrix must be stored
                if (!__all_sync(0xffffffffu, wait_stored(launch.stored + ti.matrix, ti.after * kArrivals, error.device,
                                                         abort_flag, wait_limit))) {
                    ok = false;
                    break;
                }
                asm volatile("fence.proxy.async.global;" ::: "memory");
                drain.fetch(0, 0);
                drain.fetch(0, 1);
            }
            auto drained = [&](int buffer) {
                tcgen05_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (kCtas == 2) mbar_remote_arrive(map_to_cta(smem_u32(&bars->tmem_empty[buffer]), 0));
                    else mbar_arrive(&bars->tmem_empty[buffer]);
                }
            };
            const uint32_t my_tmem = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(col_half * kCols);
            auto wait_acc = [&] {
                const bool full = __all_sync(0xffffffffu, mbar_wait(&bars->tmem_full[acc], acc_phase, abort_flag, wait_limit));
                tcgen05_fence_after();
                return full;
            };
            const bool piece = ti.part >= 0 && ti.parts == 0;
            float *const slot = launch.partials + (ti.part >= 0 ? (int64_t)ti.part * BM * BM : 0) +
                                (int64_t)(quarter * 32 + lane) * BM + col_half * kCols;
            float sum[kPlanes == 2 ? kCols : 1];
#pragma unroll
            for (int j = 0; j < (kPlanes == 2 ? kCols : 1); ++j) sum[j] = 0.0f;
            if (kPlanes == 2) {
                const int chunks = (ti.kb1 - ti.kb0 + C::kChunkBlocks - 1) / C::kChunkBlocks;
                for (int c = 0; c + 1 < chunks && ok; ++c) {
                    ok = wait_acc();
                    if (!ok) break;
#pragma unroll
                    for (int cc = 0; cc < kCols / 32; ++cc) {
                        uint32_t v[32];
                        tmem_ld_32x32_sync(my_tmem + (uint32_t)(acc * C::BN + cc * 32), v);
#pragma unroll
                        for (int j = 0; j < 32; ++j) sum[kPlanes == 2 ? cc * 32 + j : 0] += __uint_as_float(v[j]);
                    }
                    drained(acc);
                    acc ^= 1;
                    acc_phase ^= acc == 0 ? 1u : 0u;
                }
            }
            if (ok) ok = wait_acc();
            if (!ok) break;
            const uint32_t acc_tmem = my_tmem + (uint32_t)(acc * C::BN);
            if (kCtas == 1 && ti.parts > 0) {
                // the pieces in order, into this warp's part of the (unused) accumulator
                if (!__all_sync(0xffffffffu, wait_stored(launch.stored + ti.matrix, ti.after * kArrivals, error.device,
                                                         abort_flag, wait_limit))) {
                    ok = false;
                    break;
                }
#pragma unroll 1
                for (int cc = 0; cc < kCols / 32; ++cc) {
                    float t[32];
#pragma unroll
                    for (int j = 0; j < 32; ++j) t[j] = 0.0f;
#pragma unroll 2
                    for (int k = 0; k < ti.parts; ++k) {
                        const float4 *from = reinterpret_cast<const float4 *>(slot + (int64_t)k * BM * BM + cc * 32);
#pragma unroll
                        for (int q = 0; q < 8; ++q) {
                            const float4 x = __ldcg(from + q);  // written by other SMs in this launch
                            t[4 * q] += x.x, t[4 * q + 1] += x.y, t[4 * q + 2] += x.z, t[4 * q + 3] += x.w;
                        }
                    }
                    uint32_t v[32];
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(t[j]);
                    tmem_st_32x32(acc_tmem + (uint32_t)(cc * 32), v);
                }
                tmem_st_wait();
            } else if (kPlanes == 2 || (kCtas == 1 && piece)) {
                // two planes: the last part joins, and the sum goes back into this warp's part of the accumulator, to be
                // drained from there: the sum and the drain do not fit the registers together.  A piece of a cut
                // contraction goes to its slot instead.
#pragma unroll
                for (int cc = 0; cc < kCols / 32; ++cc) {
                    uint32_t v[32];
                    tmem_ld_32x32_sync(acc_tmem + (uint32_t)(cc * 32), v);
                    if (kPlanes == 2) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(sum[kPlanes == 2 ? cc * 32 + j : 0] + __uint_as_float(v[j]));
                    }
                    if (kCtas == 1 && piece) {
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const uint32_t o[8] = {v[8 * q], v[8 * q + 1], v[8 * q + 2], v[8 * q + 3],
                                                   v[8 * q + 4], v[8 * q + 5], v[8 * q + 6], v[8 * q + 7]};
                            st_global_256(slot + cc * 32 + q * 8, o);
                        }
                    } else {
                        tmem_st_32x32(acc_tmem + (uint32_t)(cc * 32), v);
                    }
                }
                tmem_st_wait();
            }
            if (inside && !piece) ok = drain.run(acc_tmem, mult, abort_flag, wait_limit, [&] { drained(acc); });
            else drained(acc);
            acc ^= 1;
            acc_phase ^= acc == 0 ? 1u : 0u;
            if (ok) {  // this warp's part of D (or of a slot) is in memory, for other SMs
                __syncwarp();
                if (lane == 0) {
                    bulk_wait_all();
                    asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(launch.stored + ti.matrix) : "memory");
                }
                __syncwarp();
            }
        }
        if (!ok && lane == 0) {
            bars->abort = 1;
            report(error, 3u);
        }
        if (lane == 0) bulk_wait_all();  // no store reads shared memory after this
        __syncwarp();
    }

    tcgen05_fence_before();
    __syncthreads();
    if (bars->abort != 0 && threadIdx.x == 0) {
        // copies that may still be in flight get a bounded time to land before shared memory is released
        for (int s = 0; s < C::kStages; ++s)
            for (uint32_t i = 0; i < 4096u; ++i)
                if (mbar_try_wait(&bars->full[s], 0) || mbar_try_wait(&bars->full[s], 1)) break;
        for (int w = 0; w < 2 * kEpiWarps; ++w)
            for (uint32_t i = 0; i < 4096u; ++i)
                if (mbar_try_wait(&bars->term_full[w], 0) || mbar_try_wait(&bars->term_full[w], 1)) break;
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
int launch_variant(const NsLaunch &l, const uint32_t *d_active, NsError error, cudaStream_t stream,
                   uint32_t wait_limit, bool withhold)
{
    const size_t smem = smem_bytes<kCtas, kPlanes>();
    VB_CUDA(cudaFuncSetAttribute(ns_product_kernel<kCtas, kPlanes>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeCooperative;  // all CTAs resident at once, or the launch is refused
    attr[0].val.cooperative = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = kCtas;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = kCtas == 2 ? 2 : 1;
    cfg.gridDim = dim3((unsigned)(l.groups * kCtas));
    VB_CUDA(cudaLaunchKernelEx(&cfg, ns_product_kernel<kCtas, kPlanes>, l, d_active, error, wait_limit, withhold ? 1 : 0));
    return VB_OK;
}

}  // namespace

int ns_resident_groups(int shape, int planes, int sm_count, int *groups)
{
    *groups = sm_count;
    if (shape != NS_TILE_PAIR) return VB_OK;
    // pairs are the two SMs of a TPC; where an SM of one is missing, fewer fit than half of the SMs
    auto *kernel = planes == 2 ? ns_product_kernel<2, 2> : ns_product_kernel<2, 1>;
    const size_t smem = planes == 2 ? smem_bytes<2, 2>() : smem_bytes<2, 1>();
    VB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(kThreads);
    cfg.gridDim = dim3((unsigned)(sm_count / 2 * 2));
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int count = 0;
    VB_CUDA(cudaOccupancyMaxActiveClusters(&count, kernel, &cfg));
    if (count < 1) return fail(VB_ERR_CUDA, "the device cannot hold a 2-CTA cluster of the product kernel");
    *groups = std::min(count, sm_count / 2);
    return VB_OK;
}

void ns_tile_extent(int shape, int planes, int *bm, int *bn)
{
    *bm = shape == NS_TILE_PAIR ? 256 : 128;
    *bn = shape == NS_TILE_PAIR && planes == 1 ? 256 : 128;
}

int make_ns_map(CUtensorMap *map, const void *base, int64_t inner, int64_t outer, int kind)
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
    const bool view = kind == NS_MAP_MN || kind == NS_MAP_MN_64;
    cuuint32_t estr[3] = {1, 1, 1};
    cuuint64_t dims[3] = {view ? 64 : (cuuint64_t)inner, (cuuint64_t)outer, (cuuint64_t)(inner / 64)};
    cuuint64_t strides[2] = {(cuuint64_t)inner * 2, 128};
    cuuint32_t box[3] = {kind == NS_MAP_MIRROR ? 32u : 64u, kind == NS_MAP_ROWS ? 128u : kind == NS_MAP_PIECE ? 32u : 64u,
                         kind == NS_MAP_MN_64 ? 1u : 2u};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, view ? 3 : 2, const_cast<void *>(base), dims, strides, box, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, kind == NS_MAP_MIRROR ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(VB_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
    return VB_OK;
}

int launch_ns_products(const NsLaunch &l, int shape, int planes, const uint32_t *d_active, NsError error,
                       cudaStream_t stream, uint32_t wait_limit, bool withhold)
{
    if (l.n_tiles <= 0) return VB_OK;
    if (shape == NS_TILE_PAIR)
        return planes == 2 ? launch_variant<2, 2>(l, d_active, error, stream, wait_limit, withhold)
                           : launch_variant<2, 1>(l, d_active, error, stream, wait_limit, withhold);
    return planes == 2 ? launch_variant<1, 2>(l, d_active, error, stream, wait_limit, withhold)
                       : launch_variant<1, 1>(l, d_active, error, stream, wait_limit, withhold);
}

}  // namespace vb
