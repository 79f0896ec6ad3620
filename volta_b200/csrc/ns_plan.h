// Newton-Schulz on caller-owned matrices (include/volta_b200.h, "vb_ns_plan"): descriptors shared by
// the planner (ns_plan.cu), the element-wise kernels (ns_gather.cu) and the tensor-core products
// (ns_products.cu).
//
// Notation.  A matrix of r x c is worked on as X of n x m, n = min(r, c), m = max(r, c), transposed
// where r > c.  Everything the tensor cores read is f16, in one plane (VB_NS_F16) or two whose sum
// has 22 significand bits (VB_NS_F32_TC), zero-padded to multiples of 128 in both directions, and
// stored times a power of two that the planner picks from bounds of the polynomials.
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>

#include "vb_internal.h"

namespace vb {

constexpr int kNsKBlock = 64;  // of the contraction, as staged in shared memory
constexpr int kNsPad = 128;  // sides of the working matrices are multiples of this

// One product of the iteration:  D = e E + f F + g sum_k A[m,k] B[n,k]
// E and F (f16, leading dimension and planes of D; may be null) are read at D's position.
enum NsProductFlags {
    NS_B_MN_MAJOR = 1,  // B is stored [k][n] (the working matrix X); otherwise [n][k]
    NS_GRAM = 2,        // X X^T: the contraction runs over the long side
    NS_SAME = 4         // A and B are one matrix
};
struct alignas(128) NsProduct {
    // tensor maps, see make_ns_map
    CUtensorMap map_a;         // operand, NS_MAP_ROWS
    CUtensorMap map_b;         // operand, NS_MAP_ROWS or NS_MAP_MN (or their 64-wide forms)
    CUtensorMap map_term[2];   // E and F, NS_MAP_PIECE
    CUtensorMap map_d;         // D, NS_MAP_PIECE
    CUtensorMap map_mirror;    // D, NS_MAP_MIRROR
    int32_t M, N, K;           // padded extents
    int32_t plane_rows;        // rows between the planes of a matrix
    int32_t n_terms;           // 0: D = g acc, 1: E, 2: E and F
    float term[2], g;          // e, f, g
    int32_t scale_power;     // e, f, g are multiplied by scale^scale_power (0, 1 or 2)
    const float *scale;      // the matrix's normalisation (null where scale_power is 0)
    int32_t matrix;          // index into the activity words
    int32_t flags;
};
enum NsTileFlags {
    NS_TILE_MIRROR = 1,  // symmetric product: the tile is also stored transposed
    NS_TILE_SHARED = 2   // A times its own transpose, on the diagonal: the rows of B are those of A, staged once
};
struct NsTile {
    int32_t problem, m0, n0;
    int32_t flags;    // NsTileFlags
    uint32_t after;   // tiles of the matrix's earlier stages: all of them must be stored before this one starts
    int32_t kb0, kb1; // blocks of 64 of the contraction
    // A contraction cut into pieces (128 x 128 tiles): a piece (part >= 0, parts == 0) stores its f32 accumulator in
    // slot `part`; the tile after them (parts > 0, no contraction of its own) sums slots part .. part + parts - 1 in order.
    int32_t part, parts;
};

// The tiles of every stage of every matrix, CTA (pair) by CTA (pair): group g takes tiles begin[g] .. begin[g + 1] - 1 in
// order.  The orders are consistent with one order of all tiles in which every tile follows those it waits for.
struct NsLaunch {
    const NsProduct *problems;
    const NsTile *tiles;
    const int32_t *begin;
    uint32_t *stored;  // per matrix: epilogue warps' arrivals, zeroed by the gather pass
    float *partials;   // slots of 128 x 128
    int n_tiles;
    int groups;
};

// Tile shapes of the product kernel.
enum NsTileShape {
    NS_TILE_PAIR = 0,  // two CTAs, 256 x 256 (two planes: 256 x 128)
    NS_TILE_128 = 1    // one CTA, 128 x 128
};
int ns_resident_groups(int shape, int planes, int sm_count, int *groups);  // CTAs (pairs) the device holds at once
void ns_tile_extent(int shape, int planes, int *bm, int *bn);
// Where a kernel reports a wait that ran out: a device word later kernels look at, a mapped one for the host.
struct NsError {
    uint32_t *device, *host;
};
// withhold: test hook, the producers stage nothing so that every wait runs out
int launch_ns_products(const NsLaunch &launch, int shape, int planes, const uint32_t *d_active, NsError error,
                       cudaStream_t stream, uint32_t wait_limit, bool withhold);
// A row-major f16 matrix [outer][inner] as the kernel moves it.
enum NsMap {
    NS_MAP_ROWS = 0,   // 64 x 128 boxes, 128-byte swizzle: 128 rows x 64 k of an operand
    NS_MAP_MN = 1,     // 64 x 64 x 2 boxes of the view [inner / 64][outer][64], same swizzle: 64 k x 128 columns
    NS_MAP_PIECE = 2,  // 64 x 32 boxes, same swizzle: what an epilogue warp reads or writes at once
    NS_MAP_MIRROR = 3, // 32 x 64 boxes: the same piece transposed
    NS_MAP_ROWS_64 = 4, NS_MAP_MN_64 = 5  // as the first two, 64 rows or columns
};
int make_ns_map(CUtensorMap *map, const void *base, int64_t inner, int64_t outer, int kind);

// ---- element-wise kernels over the caller's matrices ---------------------------------------
// A caller's array of one matrix in the working orientation: element (i, j) of X is at
// ptr[i * si + j * sj].
struct NsArray {
    void *ptr;
    int64_t si, sj;
};
constexpr int kNsBatch = 96;  // matrices of one element-wise launch (bounded by its parameter space)
struct NsMatrixDims {
    int32_t n, m;            // extents
    int32_t np, mp;          // padded
    int64_t x_off;           // element offset of the working matrix (plane 0)
    int64_t final_off;       // the same of the last iterate
    float final_scale;       // a stored value of the last iterate times this is the value
    int32_t tile0, n_tiles;  // element-wise tiles of this matrix
};
struct NsMatrixArg {
    NsArray a[3];   // orthogonalize: input, output; step: gradient, velocity, parameter
    NsMatrixDims d;
    float scale;    // step: s_i of the update
    uint32_t live;  // 0: no gradient, the matrix is left alone
    uint32_t direct; // bit k: array k has sj == 1 and rows on 16-byte boundaries
};
struct NsElementwise {
    double *partials;          // one sum of squares per tile
    float *scale;              // per matrix: X = scale * working matrix
    uint32_t *active;          // per matrix: 0 = skipped by the products and by what follows
    uint32_t *stored;          // per matrix: set to zero for the products
    const uint32_t *error;     // set once a product kernel gave up a wait: nothing more is stored
    __half *x;                 // working matrices
    int planes;
    int types[3];              // vb_dtype of the arrays of NsMatrixArg
    float eps;
    float momentum, decay, rate;
    int nesterov;
};
struct NsBatchArgs {
    NsMatrixArg m[kNsBatch];
    int32_t first;  // index of m[0] in the plan
    int32_t count;
    int32_t tile0, n_tiles;
};
constexpr int kNsTileI = 64, kNsTileJ = 128;  // an element-wise tile of the working matrix
// turned: some array of the list is contiguous along the short side
int launch_ns_norm(const NsElementwise &w, const NsBatchArgs &b, const int32_t *d_tile_matrix, bool step, bool turned, cudaStream_t stream);
int launch_ns_gather(const NsElementwise &w, const NsBatchArgs &b, const int32_t *d_tile_matrix, bool step, bool turned, cudaStream_t stream);
int launch_ns_finish(const NsElementwise &w, const NsBatchArgs &b, const int32_t *d_tile_matrix, bool step, bool turned, cudaStream_t stream);

// ---- matrices with a short side of at most 64 (ns_small.cu) ----------------------------------
constexpr int kNsSmallSide = 64;
constexpr int kNsTinySide = 16;      // up to here VB_NS_F32_TC keeps the short side in f64
constexpr int kNsSmallOps = 128;     // longest program
constexpr int kNsSmallSquares = 5;
constexpr int kNsSmallCluster = 8;   // most CTAs of one matrix
struct alignas(16) NsSmallOp {
    int8_t A, B, E, F, D;   // short-side matrices (0 ..), -1: none; of a Gram D, of an update A only
    int8_t kind;            // 0 product of two short-side matrices, 1 Gram, 2 update of X
    int8_t stage_ops;       // products of this op's stage from this one on
    int8_t scale_power;
    float e, f, g;          // as in NsProduct
    int32_t pad[3];
};
struct NsSmallMatrix {
    int32_t n, m;
    int32_t op0, n_ops;     // its program
    float final_scale;
};
struct NsSmall {
    const NsSmallMatrix *matrices;  // of a whole plan
    const NsSmallOp *ops;
    const double *coefficients;     // a, b, c of every step
    int n_steps;
    int cluster;                    // CTAs per matrix
    int columns;                    // columns of X per CTA, a multiple of 64
};
int ns_small_columns(int planes);  // columns of X that fit one CTA
int launch_ns_small(const NsElementwise &w, const NsSmall &s, const NsBatchArgs &b, NsError error, bool step, cudaStream_t stream,
                    uint32_t wait_limit, bool withhold);

}  // namespace vb
