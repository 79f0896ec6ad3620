// Newton-Schulz on caller-owned matrices: the planner, the workspace and the C entry points
// (include/volta_b200.h, vb_ns_plan_*, vb_orthogonalize, vb_muon_multi_tensor_step).
//
// The iteration X' = q(G) X with G = X X^T and q(t) = a + b t + c t^2 is run in groups of steps.
// Inside a group everything is a polynomial of the group's first Gram, so it stays on the short side:
//     G      = X X^T                                    n^2 m   (symmetric: half a product)
//     R      = b G + c G G                              n^3     (q(G) = a I + R)
//     T      = a G + R G;     P' = a P + alpha R + R P   n^3 each (alpha I + P: the group's polynomial so far)
//     G'     = a T + T R                                n^3     (the Gram of the next iterate: q(G)^2 G)
//     X'     = alpha X + P X                            2 n^2 m (once per group)
// The longer a group, the less is paid on the long side: a step by itself costs 3 n^2 m + n^3, every
// further one of a group 4 n^3.  What limits a group is rounding: noise of size d in G (2^-12 |G|_F
// spread over the spectrum) grows by the slope of t q(t)^2 with every step and reaches small eigenvalues'
// q after k steps as d prod a^2.  In f16 the 1024-sided quintic run as one group is wrong by 10 to
// 100 % on gradients with a decaying spectrum.  The first group of a call may amplify 150-fold where
// n >= 256 (its Gram has trace 1, and d falls with sqrt(n): less for smaller n), later ones, whose Gram is
// near the identity, 17-fold: with these limits the error equals that of one step at a time (1e-3 to 4e-3
// relative) on Gaussian, low-rank-plus-noise and power-law spectra.  For the usual quintic this means groups
// of 3 and 2.  Matrices whose long
// side is less than 1.5 times the short one run one step at a time: grouping saves nothing there.
//
// Powers of two.  Every stored matrix carries 2^e with e from the largest value its polynomial takes
// on [0, 1] (sampled), so that f16 neither overflows nor loses small entries.
#include <cmath>

#include <algorithm>
#include <atomic>
#include <map>
#include <functional>
#include <memory>
#include <numeric>
#include <queue>

#include "engine.h"
#include "ns_plan.h"

namespace vb {
namespace {

constexpr int kSquares = 5;  // short-side matrices alive at once: G, T, R, P and the one being written
constexpr int kMaxSteps = 64;
constexpr int64_t kMaxSide = 65536;
constexpr uint32_t kDefaultWaitLimit = 1u << 22;  // polls, about a second
constexpr double kDiverged = 1048576.0;
// Elements of an element-wise launch.  Norm and gather of a batch follow each other; small batches would find the
// second read in the L2 cache, but their launches fill and drain more often: 4, 8, 16, 64 Mi elements measured
// 1073, 970, 886, 748 us for the d = 1024 set.
constexpr int64_t kBatchElements = 64 << 20;

// ---- schedule ----------------------------------------------------------------------------
enum BufferId { BUF_X0 = 0, BUF_X1 = 1, BUF_SQUARE = 2 };  // BUF_SQUARE + k: k-th short-side matrix

struct Product {
    int A, B, E, F, D;  // buffers; E, F may be -1
    double e, f, g;
    int scale_power;
    bool update;     // M x N x K = n x m x n with B = X; otherwise n x n, symmetric
    bool gram;       // K = m
};
struct Schedule {
    std::vector<std::vector<Product>> stages;  // products of a stage are independent
    int final_buffer = BUF_X0;
    double final_scale = 1.0;  // 2^-e of the last iterate
};

struct Step {
    double a, b, c;
    double q(double t) const { return a + t * (b + c * t); }
};

int exponent_for(double bound)
{
    // twice the bound below 2^15: rounding noise may push eigenvalues past the polynomial's range
    const int e = (int)std::floor(14.0 - std::log2(std::max(bound, 1e-12)));
    return std::min(e, 40);
}

// How much a group may amplify the rounding of its Gram: the first one, and the others.  0: one step at a time.
struct GroupLimits {
    double first, later;
};

std::vector<std::vector<int>> make_groups(const std::vector<Step> &steps, const GroupLimits &limits)
{
    std::vector<std::vector<int>> groups;
    std::vector<double> lam(4097);
    for (size_t i = 0; i < lam.size(); ++i) lam[i] = (double)i / (double)(lam.size() - 1);
    double gain = 1.0;
    for (int k = 0; k < (int)steps.size(); ++k) {
        const Step &s = steps[(size_t)k];
        const bool fits = !groups.empty() && gain <= (groups.size() == 1 ? limits.first : limits.later);
        if (!fits) {
            groups.emplace_back();
            gain = 1.0;
        }
        groups.back().push_back(k);
        // steepest slope of t q(t)^2 on the range the eigenvalues are in
        double top = 0.0, slope = s.a * s.a;
        for (double t : lam) top = std::max(top, t);
        for (int i = 0; i <= 1024; ++i) {
            const double t = top * i / 1024.0, q = s.q(t);
            slope = std::max(slope, std::fabs(q * q + 2.0 * t * q * (s.b + 2.0 * s.c * t)));
        }
        gain *= slope;
        for (double &t : lam) t = t * s.q(t) * s.q(t);
    }
    return groups;
}

// Returns false if the iterates leave the range that is sensible to hold.
bool make_schedule(const std::vector<Step> &steps, const GroupLimits &limits, Schedule *out)
{
    const auto groups = make_groups(steps, limits);
    const int kSamples = 8192;
    std::vector<double> lam, sv;  // samples of the spectrum: of G, and the singular values of X
    for (int i = 0; i <= kSamples; ++i) lam.push_back((double)i / kSamples);
    for (int i = 0; i < 256; ++i) lam.push_back(std::exp2(-i / 8.0));
    for (double t : lam) sv.push_back(std::sqrt(t));
    auto bound = [&](auto &&fn) {
        double top = 0.0;
        for (size_t i = 0; i < lam.size(); ++i) top = std::max(top, std::fabs(fn(i)));
        return top;
    };
    int x = BUF_X0, ex = 0;  // the first working matrix has a scale of its own (on the device)
    for (size_t gi = 0; gi < groups.size(); ++gi) {
        const bool first = gi == 0;
        auto square = [&](std::initializer_list<int> live) {
            for (int k = BUF_SQUARE; k < BUF_SQUARE + kSquares; ++k)
                if (std::find(live.begin(), live.end(), k) == live.end()) return k;
            return -1;
        };
        int G = BUF_SQUARE, P = -1, eP = 0;
        int eG = exponent_for(bound([&](size_t i) { return lam[i]; }));
        out->stages.push_back({{x, x, -1, -1, G, 0.0, 0.0, std::exp2(eG - 2 * ex), first ? 2 : 0, false, true}});
        double alpha = 1.0, fP = 1.0;  // the group's polynomial is alpha I + fP P
        std::vector<double> poly(lam.size(), 1.0);
        for (size_t k = 0; k < groups[gi].size(); ++k) {
            const Step s = steps[(size_t)groups[gi][k]];
            const bool last = k + 1 == groups[gi].size();
            // R, held as fR times a stored matrix: a linear step's R is b G itself
            int R = G, eR = eG;
            double fR = s.b;
            if (s.c != 0.0) {
                R = square({G, P});
                eR = exponent_for(bound([&](size_t i) { return lam[i] * (s.b + s.c * lam[i]); }));
                fR = 1.0;
                out->stages.push_back({{G, G, G, -1, R, s.b * std::exp2(eR - eG), 0.0, s.c * std::exp2(eR - 2 * eG), 0, false, false}});
            }
            std::vector<Product> both;
            int T = -1, eT = 0;
            if (!last) {
                T = square({G, R, P});
                eT = exponent_for(bound([&](size_t i) { return lam[i] * s.q(lam[i]); }));
                both.push_back({R, G, G, -1, T, s.a * std::exp2(eT - eG), 0.0, fR * std::exp2(eT - eR - eG), 0, false, false});
            }
            for (size_t i = 0; i < lam.size(); ++i) poly[i] *= s.q(lam[i]);
            if (P < 0) {
                P = R, eP = eR, fP = fR;
            } else {
                const double next = alpha * s.a;
                const int N = square({G, R, P, T});
                const int eN = exponent_for(bound([&](size_t i) { return poly[i] - next; }));
                both.push_back({R, P, P, R, N, s.a * fP * std::exp2(eN - eP), alpha * fR * std::exp2(eN - eR),
                                fR * fP * std::exp2(eN - eR - eP), 0, false, false});
                P = N, eP = eN, fP = 1.0;
            }
            alpha *= s.a;
            if (!both.empty()) out->stages.push_back(both);
            for (double &t : lam) t = t * s.q(t) * s.q(t);
            if (!last) {
                const int N = square({T, R, P});
                const int eN = exponent_for(bound([&](size_t i) { return lam[i]; }));
                out->stages.push_back({{T, R, T, -1, N, s.a * std::exp2(eN - eT), 0.0, fR * std::exp2(eN - eT - eR), 0, false, false}});
                G = N, eG = eN;
            }
        }
        for (size_t i = 0; i < sv.size(); ++i) sv[i] *= poly[i];
        const double top = bound([&](size_t i) { return sv[i]; });
        if (!(top < kDiverged)) return false;
        const int eX = exponent_for(top), y = x == BUF_X0 ? BUF_X1 : BUF_X0;
        out->stages.push_back({{P, x, x, -1, y, alpha * std::exp2(eX - ex), 0.0, fP * std::exp2(eX - eP - ex), first ? 1 : 0, true, false}});
        x = y, ex = eX;
    }
    out->final_buffer = x;
    out->final_scale = std::exp2(-ex);
    return true;
}

const char *const kDivergedText = "these coefficients take singular values in [0, 1] beyond 2^20";

int read_steps(int n_steps, const float *coefficients, std::vector<Step> *steps)
{
    if (n_steps < 1 || n_steps > kMaxSteps || !coefficients)
        return fail(VB_ERR_INVALID_ARG, "1 to %d steps with coefficients are needed", kMaxSteps);
    for (int k = 0; k < n_steps; ++k) {
        const Step s{coefficients[3 * k], coefficients[3 * k + 1], coefficients[3 * k + 2]};
        if (!std::isfinite(s.a) || !std::isfinite(s.b) || !std::isfinite(s.c))
            return fail(VB_ERR_INVALID_ARG, "coefficients of step %d are not finite", k);
        steps->push_back(s);
    }
    return VB_OK;
}
// Matrices of ns_small.cu keep the short side in two planes whatever the mode: 2^-11 of the rounding, so that
// much more amplification is allowed where f16 accuracy is asked for.
GroupLimits group_limits(int64_t rows, int64_t cols, int planes, bool small)
{
    const double n = (double)std::min(rows, cols), m = (double)std::max(rows, cols);
    if (small && planes == 1) return {5e4 * std::sqrt(n / 64.0), 2e4 * std::sqrt(n / 64.0)};
    if (small) return {75.0 * std::sqrt(n / 64.0), 17.0 * std::min(1.0, std::sqrt(n / 32.0))};
    if (2.0 * m < 3.0 * n) return {0.0, 0.0};
    return {150.0 * std::min(1.0, std::sqrt(n / 256.0)), 17.0};
}
bool is_small(int64_t rows, int64_t cols, int planes)
{
    const int64_t n = std::min(rows, cols), m = std::max(rows, cols);
    return n > 0 && n <= kNsSmallSide && m <= (int64_t)kNsSmallCluster * ns_small_columns(planes);
}
std::vector<NsSmallOp> small_program(const Schedule &s)
{
    std::vector<NsSmallOp> ops;
    auto square = [](int buffer) { return (int8_t)(buffer >= BUF_SQUARE ? buffer - BUF_SQUARE : -1); };
    for (const auto &stage : s.stages)
        for (size_t k = 0; k < stage.size(); ++k) {
            const Product &p = stage[k];
            ops.push_back({square(p.A), square(p.B), square(p.E), square(p.F), square(p.D), (int8_t)(p.update ? 2 : p.gram ? 1 : 0),
                           (int8_t)(stage.size() - k), (int8_t)p.scale_power, (float)p.e, (float)p.f, (float)p.g, {}});
        }
    return ops;
}

int check_mode(int ns_mode)
{
    if (ns_mode == VB_NS_F16 || ns_mode == VB_NS_F32_TC) return VB_OK;
    return fail(ns_mode == VB_NS_F32 || ns_mode == VB_NS_BF16 ? VB_ERR_UNSUPPORTED : VB_ERR_INVALID_ARG,
                "a plan's ns_mode is VB_NS_F16 or VB_NS_F32_TC, not %d", ns_mode);
}

struct DeviceGuard {  // runs the call on the engine's device and leaves the caller's current one as it was
    int before = -1;
    int enter(int device)
    {
        VB_CUDA(cudaGetDevice(&before));
        if (before == device) before = -1;
        else VB_CUDA(cudaSetDevice(device));
        return VB_OK;
    }
    ~DeviceGuard()
    {
        if (before >= 0) cudaSetDevice(before);
    }
};

// what ns_small.cu executes for one matrix: M = 128 with 64 rows in use, 64-column blocks, plane products
double small_flops(const Schedule &s, int64_t m, int planes)
{
    double products = 0.0;
    for (const auto &stage : s.stages)
        for (const Product &p : stage)
            products += p.gram ? (double)((m + 63) / 64) * (planes == 2 ? 3 : 1) : p.update ? (double)((m + 63) / 64) * (planes == 2 ? 3 : 2) : 3.0;
    return products * 2.0 * 128 * 64 * 64;
}
int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

}  // namespace
}  // namespace vb

struct vb_ns_matrices {
    uint64_t plan = 0;  // serial number of its plan: an address may come back after the plan is gone
    int dtype = 0;
    std::vector<vb::NsArray> arrays;  // in the working orientation
    std::vector<uint8_t> vec;         // rows (or columns) on 16-byte boundaries
    std::vector<std::pair<const void *, int64_t>> starts;  // first addresses in order, with their matrices
    bool writable = true;             // no two elements at one address
    bool turned = false;              // an array is contiguous along the short side
    bool any_null = false;            // a matrix with elements has no array
    const char *why = "";             // why it is not writable
};

struct vb_ns_plan {
    vb_engine *eng = nullptr;
    uint64_t serial = 0;
    int device = 0;
    int64_t n = 0;
    std::vector<int64_t> rows, cols;
    std::vector<vb::NsMatrixDims> dims;
    int planes = 1;
    float eps = 0.0f;
    double flops = 0.0;
    size_t workspace = 0;
    char *d_base = nullptr;  // one allocation: everything below lies in it
    vb::NsElementwise ew{};  // device pointers of the element-wise passes
    const int32_t *d_tile_matrix = nullptr;
    vb::NsLaunch products{};
    int shape = 0;
    struct Batch {
        int32_t first, count, tile0, n_tiles;
    };
    std::vector<Batch> batches;
    std::vector<int32_t> small_matrices;  // those that ns_small.cu runs, in its order
    vb::NsSmall small{};
    // Small matrices run beside the others, and their launches (one per kNsBatch matrices) two at a time: the next one
    // takes the SMs that the clusters of a last wave leave idle.  Measured, one after the other / two at a time:
    // 120 of 1024 x 64 in f16 121 / 65 us, 400 of 64 x 64 172 / 107 us, 400 of 576 x 48 in f32 496 / 329 us.
    cudaStream_t side[2] = {nullptr, nullptr};
    cudaEvent_t forked = nullptr, joined[2] = {nullptr, nullptr};
    int sides = 0;
    vb::NsError error{};
    uint32_t *h_error = nullptr;
    bool withhold = false;
    uint32_t wait_limit = 0;  // of the next call, 0: the default
    uint32_t default_wait_limit = 0;
    std::unique_ptr<vb::NsBatchArgs> args;  // scratch of a call
};

namespace vb {

int ns_plan_check_error(vb_ns_plan *p)
{
    if (p->h_error && *reinterpret_cast<volatile uint32_t *>(p->h_error) != 0)
        return fail(VB_ERR_TIMEOUT, "a Newton-Schulz product kernel gave up waiting on a pipeline barrier (role %u)", *p->h_error);
    return VB_OK;
}
void ns_plan_orphan(vb_ns_plan *p) { p->eng = nullptr; }

namespace {

void free_plan(vb_ns_plan *p)
{
    if (p->d_base) cudaFree(p->d_base);
    if (p->forked) cudaEventDestroy(p->forked);
    for (int k = 0; k < 2; ++k) {
        if (p->joined[k]) cudaEventDestroy(p->joined[k]);
        if (p->side[k]) cudaStreamDestroy(p->side[k]);
    }
    if (p->h_error) cudaFreeHost(p->h_error);
    delete p;
}

// Device addresses of the parts of the workspace, in the order they are asked for.
struct Carver {
    char *base = nullptr;
    size_t used = 0;
    template <typename T>
    T *take(size_t count)
    {
        used = (used + 1023) / 1024 * 1024;
        T *p = reinterpret_cast<T *>(base + used);
        used += count * sizeof(T);
        return p;
    }
};

// Calls fn(m0, n0, flags) for every tile of a product that is computed; returns their number.
template <typename Fn>
uint32_t for_tiles(const NsProduct &pr, int shape, int planes, Fn &&fn)
{
    int bm, bn;
    ns_tile_extent(shape, planes, &bm, &bn);
    const bool symmetric = (pr.flags & NS_B_MN_MAJOR) == 0;
    uint32_t count = 0;
    for (int m0 = 0; m0 < pr.M; m0 += bm)
        for (int n0 = symmetric ? m0 : 0; n0 < pr.N; n0 += bn, ++count)
            fn(m0, n0, (symmetric && n0 >= m0 + bm ? NS_TILE_MIRROR : 0) | ((pr.flags & NS_SAME) && n0 == m0 && bm == bn ? NS_TILE_SHARED : 0));
    return count;
}

// Into how many pieces the contraction of a product is cut: a Gram over a long side whose stage would leave most
// SMs idle (128 x 9216: one tile of 144 blocks) is spread over them, in pieces of at least 8 blocks.  Summing the
// pieces is a stage more, about 8 us: a block takes 0.4 us (0.6 with two planes), so 32 blocks are where it pays
// (at 16, 513 x 1000, it cost 28 us of 158).
int gram_parts(const NsProduct &pr, int shape, uint32_t stage_tiles, int sm_count)
{
    if (shape != NS_TILE_128 || (pr.flags & NS_GRAM) == 0 || stage_tiles == 0 || pr.K < 32 * kNsKBlock) return 1;
    return std::max(1, std::min(pr.K / kNsKBlock / 8, sm_count / (int)stage_tiles));
}

constexpr double kTileCycles[2][2] = {{8.0, 9.1}, {15.6, 17.0}};  // per element of the contraction: [planes - 1][shape]

// The shape whose stages take less time if every stage is waited for: whole rounds of tiles over the device's
// CTAs (pairs), at the measured cycles of a tile per element of the contraction (one plane: 128 x 128 9.1, issue bound,
// 256 x 256 by a pair 8.0, the tensor core's rate; two planes 17.0 and, 256 x 128, 15.6), plus what a stage costs
// besides: signals, first loads and epilogue, 12000 cycles, 19000 with the pair's 256 columns (1000 x 513 bf16: 125 us with
// 128 x 128 tiles, 180 with the pair's).
int pick_shape(const std::vector<NsProduct> &problems, const std::vector<size_t> &stage_begin, int planes, int sm_count)
{
    const double per_stage[2] = {planes == 1 ? 19000.0 : 12000.0, 12000.0};
    double cost[2] = {0.0, 0.0};
    for (int shape = 0; shape < 2; ++shape) {
        const double groups = shape == NS_TILE_PAIR ? sm_count / 2 : sm_count;
        for (size_t k = 0; k + 1 < stage_begin.size(); ++k) {
            double work = 0.0, longest = 0.0;
            uint32_t tiles = 0;
            bool cut = false;
            for (size_t q = stage_begin[k]; q < stage_begin[k + 1]; ++q) tiles += for_tiles(problems[q], shape, planes, [](int, int, int) {});
            for (size_t q = stage_begin[k]; q < stage_begin[k + 1]; ++q) {
                const int parts = gram_parts(problems[q], shape, tiles, sm_count);
                cut = cut || parts > 1;
                work += (double)for_tiles(problems[q], shape, planes, [](int, int, int) {}) * problems[q].K;
                longest = std::max(longest, (double)problems[q].K / parts);
            }
            if (tiles == 0) continue;
            const double rounds = std::ceil(tiles / groups), mean = work / tiles;
            cost[shape] += per_stage[shape] * (cut ? 2 : 1) + kTileCycles[planes - 1][shape] * std::max(longest, cut ? work / groups : rounds * mean);
        }
    }
    return cost[NS_TILE_PAIR] <= cost[NS_TILE_128] ? NS_TILE_PAIR : NS_TILE_128;
}

// Deals the tiles out to the groups: the device is played through with the measured cost of a tile (see pick_shape), a
// free group takes a tile of the matrix that has the longest way to go among those whose last stage is stored by
// then.  So a long contraction of one matrix does not hold up the stages of the others, as it does where tiles are dealt
// round robin (bf16 products of 2 x (300x2000), 3 x (700x700), 10 x (200x200): 179 against 166 us).  A stage is dealt after the one before it: every group's
// list follows the order of dealing, in which a tile comes after those it waits for.
void deal_tiles(const std::vector<NsTile> &tiles, const std::vector<NsProduct> &problems, int64_t n_matrices, double cycles_per_k,
                int groups, std::vector<NsTile> *dealt, std::vector<int32_t> *begin)
{
    const double epilogue = 6000.0, signal = 3000.0;
    struct Matrix {
        std::vector<std::vector<int32_t>> stages;  // tiles that wait for the same earlier ones
        std::vector<double> way;                   // from the start of a stage to the end
        size_t stage = 0, next = 0;
        double stored = 0.0, ready = 0.0;  // the stage's last tile; the one before's
    };
    std::vector<Matrix> ms((size_t)n_matrices);
    auto cost = [&](int32_t t) { return cycles_per_k * kNsKBlock * (tiles[(size_t)t].kb1 - tiles[(size_t)t].kb0); };
    for (int32_t t = 0; t < (int32_t)tiles.size(); ++t) {
        Matrix &m = ms[(size_t)problems[(size_t)tiles[(size_t)t].problem].matrix];
        if (m.stages.empty() || tiles[(size_t)m.stages.back().front()].after != tiles[(size_t)t].after) m.stages.emplace_back();
        m.stages.back().push_back(t);
    }
    using Event = std::pair<double, int64_t>;
    std::priority_queue<Event, std::vector<Event>, std::greater<Event>> free, waiting;  // (time, group) and (time, matrix)
    std::priority_queue<Event> ready;                                                    // (way to go, matrix)
    for (int64_t i = 0; i < n_matrices; ++i) {
        Matrix &m = ms[(size_t)i];
        m.way.assign(m.stages.size() + 1, 0.0);
        for (size_t k = m.stages.size(); k-- > 0;) {
            double longest = 0.0, sum = 0.0;
            for (int32_t t : m.stages[k]) longest = std::max(longest, cost(t)), sum += cost(t);
            m.way[k] = m.way[k + 1] + std::max(longest, sum / groups) + epilogue + signal;
        }
        if (!m.stages.empty()) waiting.push({0.0, i});
    }
    for (int64_t g = 0; g < groups; ++g) free.push({0.0, g});
    std::vector<std::vector<int32_t>> lists((size_t)groups);
    for (size_t left = tiles.size(); left > 0; --left) {
        auto [now, g] = free.top();
        free.pop();
        if (ready.empty()) now = std::max(now, waiting.top().first);
        while (!waiting.empty() && waiting.top().first <= now) {
            const int64_t i = waiting.top().second;
            waiting.pop();
            ready.push({ms[(size_t)i].way[ms[(size_t)i].stage], i});
        }
        const int64_t i = ready.top().second;
        Matrix &m = ms[(size_t)i];
        const int32_t t = m.stages[m.stage][m.next++];
        lists[(size_t)g].push_back(t);
        now = std::max(now, m.ready);
        free.push({now + std::max(cost(t), epilogue), g});
        m.stored = std::max(m.stored, now + cost(t) + epilogue + signal);
        if (m.next == m.stages[m.stage].size()) {
            ready.pop();
            m.next = 0;
            m.ready = m.stored;
            if (++m.stage < m.stages.size()) waiting.push({m.stored, i});
        }
    }
    dealt->clear();
    begin->assign(1, 0);
    for (const auto &list : lists) {
        for (int32_t t : list) dealt->push_back(tiles[(size_t)t]);
        begin->push_back((int32_t)dealt->size());
    }
}

int build_plan(vb_ns_plan *p, const std::vector<Step> &steps)
{
    const int64_t n = p->n;
    std::vector<Schedule> schedules;       // the different ones among the matrices
    std::vector<std::vector<std::vector<int>>> groupings;
    std::map<std::pair<double, double>, size_t> by_limits;
    std::vector<size_t> kind((size_t)n);
    std::vector<NsSmallMatrix> small;
    std::vector<NsSmallOp> small_ops;
    std::vector<int32_t> program_at;
    int64_t small_m = 0;
    std::vector<int32_t> tile_matrix;
    std::vector<int64_t> square_off((size_t)n);
    int64_t x_total = 0, square_total = 0, tiles = 0, batch_elements = 0;
    p->dims.resize((size_t)n);
    for (int64_t i = 0; i < n; ++i) {
        NsMatrixDims &d = p->dims[(size_t)i];
        d = NsMatrixDims{};
        d.n = (int32_t)std::min(p->rows[i], p->cols[i]);
        d.m = (int32_t)std::max(p->rows[i], p->cols[i]);
        if (d.n == 0) d.m = 0;
        const auto limits = [&](bool as_small) { return group_limits(d.n, d.m, p->planes, as_small); };
        auto find = [&](const GroupLimits &l, size_t *which) -> int {
            const auto known = by_limits.find({l.first, l.later});
            if (known != by_limits.end()) {
                *which = known->second;
                return VB_OK;
            }
            const auto groups = make_groups(steps, l);
            *which = 0;
            while (*which < groupings.size() && groupings[*which] != groups) ++*which;
            by_limits[{l.first, l.later}] = *which;
            if (*which < groupings.size()) return VB_OK;
            groupings.push_back(groups);
            schedules.emplace_back();
            program_at.push_back(-1);
            return make_schedule(steps, l, &schedules.back()) ? VB_OK : fail(VB_ERR_INVALID_ARG, kDivergedText);
        };
        size_t &which = kind[(size_t)i];
        if (is_small(d.n, d.m, p->planes)) {
            VB_TRY(find(limits(true), &which));
            const auto ops = small_program(schedules[which]);
            if (ops.size() <= kNsSmallOps) {
                if (program_at[which] < 0) {
                    program_at[which] = (int32_t)small_ops.size();
                    small_ops.insert(small_ops.end(), ops.begin(), ops.end());
                }
                small.push_back({d.n, d.m, program_at[which], (int32_t)ops.size(), (float)schedules[which].final_scale});
                p->small_matrices.push_back((int32_t)i);
                small_m = std::max<int64_t>(small_m, d.m);
                p->flops += small_flops(schedules[which], d.m, p->planes);
                d.n = d.m = 0;  // nothing left for the other path
            }
        }
        if (d.n > 0 || p->small_matrices.empty() || p->small_matrices.back() != (int32_t)i) VB_TRY(find(limits(false), &which));
        d.np = (int32_t)round_up(d.n, kNsPad);
        d.mp = (int32_t)round_up(d.m, kNsPad);
        const Schedule &s = schedules[kind[(size_t)i]];
        d.x_off = x_total;
        d.final_off = s.final_buffer;  // buffer number for now
        d.final_scale = (float)s.final_scale;
        square_off[(size_t)i] = square_total;
        x_total += (int64_t)p->planes * d.np * d.mp;
        square_total += (int64_t)kSquares * p->planes * d.np * d.np;
        d.tile0 = (int32_t)tiles;
        d.n_tiles = (d.np / kNsTileI) * (d.mp / kNsTileJ);
        tiles += d.n_tiles;
        if (tiles > INT32_MAX) return fail(VB_ERR_UNSUPPORTED, "the plan's matrices have too many elements");
        tile_matrix.insert(tile_matrix.end(), (size_t)d.n_tiles, (int32_t)i);
        const int64_t elements = (int64_t)d.n * d.m;
        if (p->batches.empty() || p->batches.back().count == kNsBatch || batch_elements + elements > kBatchElements) {
            p->batches.push_back({(int32_t)i, 0, d.tile0, 0});
            batch_elements = 0;
        }
        batch_elements += elements;
        p->batches.back().count += 1;
        p->batches.back().n_tiles += d.n_tiles;
    }
    for (auto &d : p->dims) d.final_off = d.x_off + (d.final_off == BUF_X1 ? x_total : 0);

    // stages of all matrices side by side: stage k of every matrix, then stage k + 1
    size_t n_stages = 0;
    for (int64_t i = 0; i < n; ++i)
        if (p->dims[(size_t)i].n > 0) n_stages = std::max(n_stages, schedules[kind[(size_t)i]].stages.size());
    std::vector<NsProduct> problems;
    std::vector<NsTile> tile_list;

    if (!small.empty()) {
        // CTAs per matrix: as many as its columns need, more while the device has SMs and they have columns
        const int64_t fit = ns_small_columns(p->planes), count = (int64_t)small.size();
        int c = 1;
        while (round_up((small_m + c - 1) / c, 64) > fit) c *= 2;
        while (c < kNsSmallCluster && count * c * 2 <= p->eng->sm_count && small_m > 64 * c) c *= 2;
        p->small.cluster = c;
        p->small.columns = (int)round_up((small_m + c - 1) / c, 64);
    }

    // The carving is done twice: for the size, then with the addresses (tensor maps need them).
    __half *x_base = nullptr, *square_base = nullptr;
    for (int pass = 0; pass < 2; ++pass) {
        Carver c;
        c.base = p->d_base;
        x_base = c.take<__half>((size_t)(2 * x_total));
        square_base = c.take<__half>((size_t)square_total);
        p->ew.x = x_base;
        p->ew.partials = c.take<double>((size_t)tiles);
        p->ew.scale = c.take<float>((size_t)n);
        p->ew.active = c.take<uint32_t>((size_t)n);
        p->ew.stored = c.take<uint32_t>((size_t)n);
        p->error.device = c.take<uint32_t>(1);
        p->ew.error = p->error.device;
        int32_t *d_tile_matrix = c.take<int32_t>(tile_matrix.size());
        NsSmallMatrix *d_small = c.take<NsSmallMatrix>(small.size());
        NsSmallOp *d_small_ops = c.take<NsSmallOp>(small_ops.size());
        p->small.matrices = d_small;
        p->small.ops = d_small_ops;
        double *d_coefficients = c.take<double>(3 * steps.size());
        p->small.coefficients = d_coefficients;
        p->small.n_steps = (int)steps.size();
        p->d_tile_matrix = d_tile_matrix;
        problems.clear();
        std::vector<size_t> stage_begin;  // of every stage's products in `problems`
        for (size_t k = 0; k < n_stages; ++k) {
            stage_begin.push_back(problems.size());
            for (int64_t i = 0; i < n; ++i) {
                const NsMatrixDims &d = p->dims[(size_t)i];
                const Schedule &s = schedules[kind[(size_t)i]];
                if (d.n == 0 || k >= s.stages.size()) continue;
                const int64_t sp = (int64_t)d.np * d.np;
                auto address = [&](int buffer) -> __half * {
                    if (buffer < 0) return nullptr;
                    if (buffer == BUF_X0) return x_base + d.x_off;
                    if (buffer == BUF_X1) return x_base + x_total + d.x_off;
                    return square_base + square_off[(size_t)i] + (int64_t)(buffer - BUF_SQUARE) * p->planes * sp;
                };
                for (const Product &pr : s.stages[k]) {
                    NsProduct q{};
                    q.M = d.np;
                    q.N = pr.update ? d.mp : d.np;
                    q.K = pr.gram ? d.mp : d.np;
                    q.plane_rows = d.np;
                    q.n_terms = pr.F >= 0 ? 2 : pr.E >= 0 ? 1 : 0;
                    q.term[0] = (float)pr.e, q.term[1] = (float)pr.f, q.g = (float)pr.g;
                    q.scale_power = pr.scale_power;
                    q.scale = p->ew.scale + i;
                    q.matrix = (int32_t)i;
                    q.flags = (pr.update ? NS_B_MN_MAJOR : 0) | (pr.gram ? NS_GRAM : 0) |
                              (pr.A == pr.B && !pr.update ? NS_SAME : 0);
                    if (pass == 1) {
                        const int64_t outer = (int64_t)p->planes * d.np;
                        VB_TRY(make_ns_map(&q.map_a, address(pr.A), q.K, outer, NS_MAP_ROWS));
                        const bool narrow = p->planes == 2 && p->shape == NS_TILE_PAIR;  // 64 rows of B per CTA
                        VB_TRY(make_ns_map(&q.map_b, address(pr.B), pr.update ? q.N : q.K, outer,
                                           pr.update ? (narrow ? NS_MAP_MN_64 : NS_MAP_MN) : (narrow ? NS_MAP_ROWS_64 : NS_MAP_ROWS)));
                        if (pr.E >= 0) VB_TRY(make_ns_map(&q.map_term[0], address(pr.E), q.N, outer, NS_MAP_PIECE));
                        if (pr.F >= 0) VB_TRY(make_ns_map(&q.map_term[1], address(pr.F), q.N, outer, NS_MAP_PIECE));
                        VB_TRY(make_ns_map(&q.map_d, address(pr.D), q.N, outer, NS_MAP_PIECE));
                        if (!pr.update) VB_TRY(make_ns_map(&q.map_mirror, address(pr.D), q.N, outer, NS_MAP_MIRROR));
                    }
                    problems.push_back(q);
                }
            }
            // long contractions first: what is left at a stage's end is then short
            std::stable_sort(problems.begin() + (ptrdiff_t)stage_begin.back(), problems.end(),
                             [](const NsProduct &a, const NsProduct &b) { return a.K > b.K; });
        }
        stage_begin.push_back(problems.size());
        p->shape = pick_shape(problems, stage_begin, p->planes, p->eng->sm_count);
        tile_list.clear();
        std::vector<uint32_t> done((size_t)n, 0), stage_done((size_t)n, 0);
        size_t widest = 0;
        auto count_tiles = [&](const NsProduct &pr) { return for_tiles(pr, p->shape, p->planes, [](int, int, int) {}); };
        std::vector<uint32_t> stage_tiles(n_stages, 0);
        for (size_t k = 0; k < n_stages; ++k)
            for (size_t q = stage_begin[k]; q < stage_begin[k + 1]; ++q) stage_tiles[k] += count_tiles(problems[q]);
        // every matrix has slots of its own for the pieces of its Grams, which follow one another
        std::vector<int32_t> slot0((size_t)n, 0);
        for (size_t k = 0; k < n_stages; ++k)
            for (size_t q = stage_begin[k]; q < stage_begin[k + 1]; ++q) {
                const int parts = gram_parts(problems[q], p->shape, stage_tiles[k], p->eng->sm_count);
                int32_t &need = slot0[(size_t)problems[q].matrix];
                if (parts > 1) need = std::max(need, (int32_t)count_tiles(problems[q]) * parts);
            }
        int32_t slots = 0;
        for (int32_t &s : slot0) {
            const int32_t need = s;
            s = slots;
            slots += need;
        }
        for (size_t k = 0; k < n_stages; ++k) {
            const size_t stage_at = tile_list.size();
            std::vector<NsTile> sums;  // of cut contractions, behind the stage's other tiles
            for (size_t q = stage_begin[k]; q < stage_begin[k + 1]; ++q) {
                const NsProduct &pr = problems[q];
                const size_t i = (size_t)pr.matrix;
                const int blocks = pr.K / kNsKBlock;
                const int parts = gram_parts(pr, p->shape, stage_tiles[k], p->eng->sm_count);
                int32_t slot = slot0[i];
                uint32_t count = 0;
                for_tiles(pr, p->shape, p->planes, [&](int m0, int n0, int flags) {
                    if (parts == 1) {
                        tile_list.push_back({(int32_t)q, m0, n0, flags, done[i], 0, blocks, -1, 0});
                        ++count;
                        return;
                    }
                    sums.push_back({(int32_t)q, m0, n0, flags, 0, 0, 0, slot, parts});
                    for (int part = 0; part < parts; ++part, ++count)
                        tile_list.push_back({(int32_t)q, m0, n0, flags & NS_TILE_SHARED, done[i], blocks * part / parts, blocks * (part + 1) / parts, slot++, 0});
                });
                stage_done[i] += count;
            }
            widest = std::max(widest, tile_list.size() - stage_at);
            for (NsTile &t : sums) t.after = stage_done[(size_t)problems[(size_t)t.problem].matrix];
            for (const NsTile &t : sums) {
                tile_list.push_back(t);
                stage_done[(size_t)problems[(size_t)t.problem].matrix] += 1;
            }
            for (size_t q = stage_begin[k]; q < stage_begin[k + 1]; ++q) done[(size_t)problems[q].matrix] = stage_done[(size_t)problems[q].matrix];
        }
        float *partials = c.take<float>((size_t)slots * 128 * 128);
        NsProduct *d_problems = c.take<NsProduct>(problems.size());
        NsTile *d_tiles = c.take<NsTile>(tile_list.size());
        if (tile_list.size() > (size_t)INT32_MAX) return fail(VB_ERR_UNSUPPORTED, "the plan's products have too many tiles");
        // more groups than the largest stage has tiles would mostly wait, on SMs that others could use
        int groups = 0;
        VB_TRY(ns_resident_groups(p->shape, p->planes, p->eng->sm_count, &groups));
        groups = std::max(1, std::min(groups, (int)widest));
        int32_t *d_begin = c.take<int32_t>((size_t)groups + 1);
        p->products = {d_problems, d_tiles, d_begin, p->ew.stored, partials, (int)tile_list.size(), groups};
        std::vector<int32_t> begin;
        if (pass == 1) {
            std::vector<NsTile> dealt;
            deal_tiles(tile_list, problems, n, kTileCycles[p->planes - 1][p->shape], groups, &dealt, &begin);
            tile_list.swap(dealt);
            VB_CUDA(cudaMemcpyAsync(d_begin, begin.data(), begin.size() * sizeof(int32_t), cudaMemcpyHostToDevice, p->eng->stream));
            VB_CUDA(cudaStreamSynchronize(p->eng->stream));  // `begin` goes out of scope
        }
        if (pass == 1) {
            VB_CUDA(cudaMemcpyAsync(d_problems, problems.data(), problems.size() * sizeof(NsProduct), cudaMemcpyHostToDevice, p->eng->stream));
            VB_CUDA(cudaMemcpyAsync(d_tiles, tile_list.data(), tile_list.size() * sizeof(NsTile), cudaMemcpyHostToDevice, p->eng->stream));
            int bm, bn;
            ns_tile_extent(p->shape, p->planes, &bm, &bn);
            double stage_flops = 0.0;  // of the largest product
            for (size_t q = 0; q < problems.size(); ++q)
                stage_flops = std::max(stage_flops, 2.0 * (double)problems[q].M * problems[q].N * problems[q].K * 3.0);
            // the default bound (about a second) plus two per 1e14 FLOPs of the largest product: a role may rightly
            // wait for a whole stage
            p->default_wait_limit = (uint32_t)std::min(1e9, kDefaultWaitLimit * (1.0 + 2.0 * std::floor(stage_flops / 1e14)));
            for (const NsTile &t : tile_list)
                p->flops += 2.0 * (p->planes == 2 ? 3.0 : 1.0) * bm * bn * (double)(t.kb1 - t.kb0) * kNsKBlock;
        }
        if (pass == 0) {
            p->workspace = c.used;
            const cudaError_t err = cudaMalloc((void **)&p->d_base, std::max<size_t>(c.used, 1024));
            if (err != cudaSuccess) {
                cudaGetLastError();  // nothing of it is left for the checks after later launches
                p->d_base = nullptr;
                return fail(VB_ERR_CUDA, "the plan's workspace of %zu bytes could not be allocated: %s", c.used, cudaGetErrorString(err));
            }
        } else {
            if (!small.empty()) {
                static_assert(sizeof(Step) == 3 * sizeof(double), "copied as a, b, c");
                VB_CUDA(cudaMemcpyAsync(d_coefficients, steps.data(), steps.size() * sizeof(Step), cudaMemcpyHostToDevice, p->eng->stream));
                VB_CUDA(cudaMemcpyAsync(d_small, small.data(), small.size() * sizeof(NsSmallMatrix), cudaMemcpyHostToDevice, p->eng->stream));
                VB_CUDA(cudaMemcpyAsync(d_small_ops, small_ops.data(), small_ops.size() * sizeof(NsSmallOp), cudaMemcpyHostToDevice, p->eng->stream));
            }
            VB_CUDA(cudaMemsetAsync(p->error.device, 0, sizeof(uint32_t), p->eng->stream));
            VB_CUDA(cudaMemcpyAsync(d_tile_matrix, tile_matrix.data(), tile_matrix.size() * sizeof(int32_t), cudaMemcpyHostToDevice, p->eng->stream));
        }
    }
    // two streams for the launches of small matrices; without other matrices the engine's own is one of them
    const int small_launches = ((int)small.size() + kNsBatch - 1) / kNsBatch;
    p->sides = std::min(2, small_launches);
    if (p->products.n_tiles == 0) p->sides = std::max(0, p->sides - 1);
    if (p->sides > 0) VB_CUDA(cudaEventCreateWithFlags(&p->forked, cudaEventDisableTiming));
    for (int k = 0; k < p->sides; ++k) {
        VB_CUDA(cudaStreamCreateWithFlags(&p->side[k], cudaStreamNonBlocking));
        VB_CUDA(cudaEventCreateWithFlags(&p->joined[k], cudaEventDisableTiming));
    }
    VB_CUDA(cudaHostAlloc((void **)&p->h_error, sizeof(uint32_t), cudaHostAllocMapped));
    *p->h_error = 0;
    VB_CUDA(cudaHostGetDevicePointer((void **)&p->error.host, p->h_error, 0));
    VB_CUDA(cudaStreamSynchronize(p->eng->stream));  // the host copies above go out of scope
    return VB_OK;
}

// What both operators share; `fill` sets the arrays of one matrix.
template <typename Fill>
int run_plan(vb_ns_plan *p, const NsElementwise &w, bool step, bool turned, Fill &&fill)
{
    vb_engine *e = p->eng;
    NsBatchArgs &args = *p->args;
    auto load = [&](const vb_ns_plan::Batch &b) {
        args.first = b.first;
        args.count = b.count;
        args.tile0 = b.tile0;
        args.n_tiles = b.n_tiles;
        for (int32_t k = 0; k < b.count; ++k) {
            fill(b.first + k, args.m[k]);
            args.m[k].d = p->dims[(size_t)(b.first + k)];
        }
    };
    const uint32_t wait_limit = p->wait_limit ? p->wait_limit : p->default_wait_limit;
    const bool others = p->products.n_tiles > 0;
    if (p->sides > 0) {
        VB_CUDA(cudaEventRecord(p->forked, e->stream));
        for (int k = 0; k < p->sides; ++k) VB_CUDA(cudaStreamWaitEvent(p->side[k], p->forked, 0));
    }
    if (!others) prof_begin(e, VB_PHASE_MUON_NS);
    size_t launch = 0;
    for (size_t k0 = 0; k0 < p->small_matrices.size(); k0 += kNsBatch, ++launch) {
        args.first = (int32_t)k0;
        args.count = (int32_t)std::min<size_t>(kNsBatch, p->small_matrices.size() - k0);
        for (int32_t k = 0; k < args.count; ++k) fill(p->small_matrices[k0 + (size_t)k], args.m[k]);
        cudaStream_t on = others ? p->side[launch % (size_t)p->sides] : launch % 2 ? p->side[0] : e->stream;
        VB_TRY(launch_ns_small(w, p->small, args, p->error, step, on, wait_limit, p->withhold));
        e->launches += 1;
        p->withhold = false;
    }
    for (int k = 0; k < p->sides; ++k) {
        VB_CUDA(cudaEventRecord(p->joined[k], p->side[k]));
        if (!others) VB_CUDA(cudaStreamWaitEvent(e->stream, p->joined[k], 0));
    }
    if (!others) {
        prof_end(e, VB_PHASE_MUON_NS);
        p->wait_limit = 0;
        return VB_OK;
    }
    prof_begin(e, VB_PHASE_MUON_PRE);
    for (const auto &b : p->batches) {
        if (b.n_tiles == 0) continue;
        load(b);
        VB_TRY(launch_ns_norm(w, args, p->d_tile_matrix, step, turned, e->stream));
        VB_TRY(launch_ns_gather(w, args, p->d_tile_matrix, step, turned, e->stream));
        e->launches += 2;
    }
    prof_end(e, VB_PHASE_MUON_PRE);
    prof_begin(e, VB_PHASE_MUON_NS);
    VB_TRY(launch_ns_products(p->products, p->shape, p->planes, w.active, p->error, e->stream, wait_limit, p->withhold));
    e->launches += 1;
    p->withhold = false;
    prof_end(e, VB_PHASE_MUON_NS);
    p->wait_limit = 0;
    prof_begin(e, VB_PHASE_MUON_APPLY);
    for (const auto &b : p->batches) {
        if (b.n_tiles == 0) continue;
        load(b);
        VB_TRY(launch_ns_finish(w, args, p->d_tile_matrix, step, turned, e->stream));
        e->launches += 1;
    }
    prof_end(e, VB_PHASE_MUON_APPLY);
    for (int k = 0; k < p->sides; ++k) VB_CUDA(cudaStreamWaitEvent(e->stream, p->joined[k], 0));
    return VB_OK;
}

int check_list(const vb_ns_plan *p, const vb_ns_matrices *l, const char *name, bool written, bool may_be_absent)
{
    if (!l) return fail(VB_ERR_INVALID_ARG, "%s is null", name);
    if (l->plan != p->serial) return fail(VB_ERR_INVALID_ARG, "%s belongs to another plan", name);
    if (l->any_null && !may_be_absent) return fail(VB_ERR_INVALID_ARG, "%s has a null pointer", name);
    if (written && !l->writable) return fail(VB_ERR_INVALID_ARG, "%s cannot be written: %s", name, l->why);
    return VB_OK;
}
// Two lists, of which at least one is written, may share a matrix's memory only as the very same array of the same
// matrix.  Found by the first addresses; strided arrays may interleave otherwise.
int check_alias(const vb_ns_matrices *a, const vb_ns_matrices *b, const char *names, bool same_allowed)
{
    size_t k = 0;
    for (const auto &s : a->starts) {
        while (k < b->starts.size() && std::less<const void *>()(b->starts[k].first, s.first)) ++k;
        for (size_t q = k; q < b->starts.size() && b->starts[q].first == s.first; ++q) {
            const NsArray &x = a->arrays[(size_t)s.second], &y = b->arrays[(size_t)b->starts[q].second];
            if (s.second != b->starts[q].second)
                return fail(VB_ERR_INVALID_ARG, "%s of matrices %lld and %lld start at one address", names, (long long)s.second,
                            (long long)b->starts[q].second);
            if (!same_allowed || a->dtype != b->dtype || x.si != y.si || x.sj != y.sj)
                return fail(VB_ERR_INVALID_ARG, "%s of matrix %lld start at one address", names, (long long)s.second);
        }
    }
    return VB_OK;
}

int begin_call(vb_ns_plan *p, DeviceGuard *guard)
{
    if (!p) return fail(VB_ERR_INVALID_ARG, "plan is null");
    if (!p->eng) return fail(VB_ERR_STATE, "the plan's engine has been destroyed");
    VB_TRY(ns_plan_check_error(p));
    return guard->enter(p->device);
}

}  // namespace
}  // namespace vb

using namespace vb;

#define VB_NS_BEGIN try {
#define VB_NS_END                                                                                    \
    }                                                                                                \
    catch (const std::bad_alloc &) { return fail(VB_ERR_STATE, "out of host memory"); }              \
    catch (const std::exception &ex) { return fail(VB_ERR_STATE, "exception: %s", ex.what()); }      \
    catch (...) { return fail(VB_ERR_STATE, "unknown exception"); }

extern "C" {

int vb_plan_newton_schulz(int64_t rows, int64_t cols, int n_steps, const float *coefficients, int ns_mode,
                          int64_t capacity, int64_t *n_products, int32_t *ints, double *doubles, double *final_scale)
{
    VB_NS_BEGIN
    if (!n_products) return fail(VB_ERR_INVALID_ARG, "n_products is null");
    if (rows < 0 || cols < 0) return fail(VB_ERR_INVALID_ARG, "negative side");
    std::vector<Step> steps;
    VB_TRY(read_steps(n_steps, coefficients, &steps));
    Schedule s;
    VB_TRY(check_mode(ns_mode));
    const int planes = ns_mode == VB_NS_F32_TC ? 2 : 1;
    if (!make_schedule(steps, group_limits(rows, cols, planes, is_small(rows, cols, planes)), &s)) return fail(VB_ERR_INVALID_ARG, kDivergedText);
    int64_t k = 0;
    for (size_t stage = 0; stage < s.stages.size(); ++stage)
        for (const Product &p : s.stages[stage]) {
            if (k < capacity && ints) {
                const int32_t v[9] = {(int32_t)stage, p.A, p.B, p.E, p.F, p.D, p.scale_power, p.update, p.gram};
                std::copy(v, v + 9, ints + 9 * k);
            }
            if (k < capacity && doubles) doubles[3 * k] = p.e, doubles[3 * k + 1] = p.f, doubles[3 * k + 2] = p.g;
            ++k;
        }
    *n_products = k;
    if (final_scale) *final_scale = s.final_scale;
    if ((ints || doubles) && capacity < k) return fail(VB_ERR_INVALID_ARG, "%lld products, room for %lld", (long long)k, (long long)capacity);
    return VB_OK;
    VB_NS_END
}

int vb_ns_plan_create(vb_engine *e, int64_t n, const int64_t *rows, const int64_t *cols, int n_steps,
                      const float *coefficients, float eps, int ns_mode, vb_ns_plan **out)
{
    VB_NS_BEGIN
    if (!out) return fail(VB_ERR_INVALID_ARG, "out is null");
    *out = nullptr;
    if (!e) return fail(VB_ERR_INVALID_ARG, "engine is null");
    if (n < 0 || n > (1 << 20) || (n > 0 && (!rows || !cols))) return fail(VB_ERR_INVALID_ARG, "bad list of %lld matrices", (long long)n);
    std::vector<Step> steps;
    VB_TRY(read_steps(n_steps, coefficients, &steps));
    if (!(eps >= 0.0f) || !std::isfinite(eps)) return fail(VB_ERR_INVALID_ARG, "eps must be finite and >= 0");
    VB_TRY(check_mode(ns_mode));
    for (int64_t i = 0; i < n; ++i)
        if (rows[i] < 0 || cols[i] < 0 || rows[i] > kMaxSide || cols[i] > kMaxSide)
            return fail(VB_ERR_INVALID_ARG, "matrix %lld is %lld x %lld: sides are 0 to %lld", (long long)i, (long long)rows[i], (long long)cols[i], (long long)kMaxSide);
    DeviceGuard guard;
    VB_TRY(guard.enter(e->device));
    vb_ns_plan *p = new vb_ns_plan();
    static std::atomic<uint64_t> serials{0};
    p->serial = ++serials;
    p->eng = e;
    p->device = e->device;
    p->n = n;
    p->rows.assign(rows, rows + n);
    p->cols.assign(cols, cols + n);
    p->planes = ns_mode == VB_NS_F32_TC ? 2 : 1;
    p->eps = eps;
    int status;
    try {
        p->args.reset(new NsBatchArgs());
        status = build_plan(p, steps);
        if (status == VB_OK) e->ns_plans.push_back(p);
    } catch (...) {
        free_plan(p);
        throw;
    }
    if (status != VB_OK) {
        cudaStreamSynchronize(e->stream);
        free_plan(p);
        return status;
    }
    *out = p;
    return VB_OK;
    VB_NS_END
}

int vb_ns_plan_destroy(vb_ns_plan *p)
{
    if (!p) return VB_OK;
    int before = -1;
    cudaGetDevice(&before);
    cudaSetDevice(p->device);
    if (p->eng) {
        cudaStreamSynchronize(p->eng->stream);
        for (int k = 0; k < p->sides; ++k) cudaStreamSynchronize(p->side[k]);  // a call that failed half-way may not have joined them
        auto &all = p->eng->ns_plans;
        all.erase(std::remove(all.begin(), all.end(), p), all.end());
    }
    free_plan(p);
    if (before >= 0) cudaSetDevice(before);
    return VB_OK;
}

int vb_ns_plan_workspace(vb_ns_plan *p, size_t *bytes)
{
    if (!p || !bytes) return fail(VB_ERR_INVALID_ARG, "null argument");
    *bytes = p->workspace;
    return VB_OK;
}

int vb_ns_plan_flops(vb_ns_plan *p, double *flops)
{
    if (!p || !flops) return fail(VB_ERR_INVALID_ARG, "null argument");
    *flops = p->flops;
    return VB_OK;
}

int vb_ns_matrices_create(vb_ns_plan *p, int dtype, void *const *pointers, const int64_t *strides, vb_ns_matrices **out)
{
    VB_NS_BEGIN
    if (!out) return fail(VB_ERR_INVALID_ARG, "out is null");
    *out = nullptr;
    if (!p) return fail(VB_ERR_INVALID_ARG, "plan is null");
    if (dtype != VB_DTYPE_F32 && dtype != VB_DTYPE_BF16 && dtype != VB_DTYPE_F16) return fail(VB_ERR_INVALID_ARG, "unknown dtype %d", dtype);
    if (p->n > 0 && !pointers) return fail(VB_ERR_INVALID_ARG, "pointers is null");
    const int64_t size = dtype == VB_DTYPE_F32 ? 4 : 2, per16 = 16 / size;
    std::unique_ptr<vb_ns_matrices> l(new vb_ns_matrices());
    l->plan = p->serial;
    l->dtype = dtype;
    l->arrays.resize((size_t)p->n);
    l->vec.assign((size_t)p->n, 0);
    auto &starts = l->starts;
    for (int64_t i = 0; i < p->n; ++i) {
        const int64_t rows = p->rows[i], cols = p->cols[i];
        if (rows == 0 || cols == 0) continue;
        const int64_t sr = strides ? strides[2 * i] : cols, sc = strides ? strides[2 * i + 1] : 1;
        if (sr < 0 || sc < 0) return fail(VB_ERR_INVALID_ARG, "matrix %lld has a negative stride", (long long)i);
        if (sr > (INT64_MAX >> 22) || sc > (INT64_MAX >> 22)) return fail(VB_ERR_INVALID_ARG, "matrix %lld has strides out of range", (long long)i);
        NsArray &a = l->arrays[(size_t)i];
        a.ptr = pointers[i];
        a.si = rows > cols ? sc : sr;  // the working matrix has the short side first
        a.sj = rows > cols ? sr : sc;
        if (!a.ptr) {
            l->any_null = true;
            continue;
        }
        const uintptr_t at = reinterpret_cast<uintptr_t>(a.ptr);
        if (at % (uintptr_t)size) return fail(VB_ERR_INVALID_ARG, "pointer %lld is not aligned to its elements", (long long)i);
        cudaPointerAttributes attr;
        const cudaError_t err = cudaPointerGetAttributes(&attr, a.ptr);
        if (err != cudaSuccess) {
            cudaGetLastError();
            return fail(VB_ERR_INVALID_ARG, "pointer %lld is not one CUDA knows: %s", (long long)i, cudaGetErrorString(err));
        }
        if (attr.type != cudaMemoryTypeDevice && attr.type != cudaMemoryTypeManaged)
            return fail(VB_ERR_INVALID_ARG, "pointer %lld is not device memory", (long long)i);
        if (attr.type == cudaMemoryTypeDevice && attr.device != p->device)
            return fail(VB_ERR_INVALID_ARG, "pointer %lld lives on device %d, the engine runs on device %d", (long long)i, attr.device, p->device);
        // where a side is 1 its stride says nothing: the matrix is then contiguous along the other
        const int64_t n = std::min(rows, cols), m = std::max(rows, cols);
        if (n == 1 && a.sj == 1) a.si = round_up(m, per16);
        if (m == 1) a.si = per16, a.sj = 1;
        const int64_t across = a.sj == 1 ? a.si : a.si == 1 ? a.sj : 1;
        l->vec[(size_t)i] = (a.sj == 1 || a.si == 1) && at % 16 == 0 && across % per16 == 0;
        if (a.si == 1 && a.sj != 1) l->turned = true;
        const bool apart = (a.sj >= 1 && a.si >= (m - 1) * a.sj + 1) || (a.si >= 1 && a.sj >= (n - 1) * a.si + 1) ||
                           (n == 1 && (a.sj >= 1 || m == 1));
        if (!apart) l->writable = false, l->why = "elements of a matrix share an address";
        starts.emplace_back(a.ptr, i);
    }
    std::sort(starts.begin(), starts.end());
    const auto same = [](const auto &x, const auto &y) { return x.first == y.first; };
    if (std::adjacent_find(starts.begin(), starts.end(), same) != starts.end()) l->writable = false, l->why = "two matrices start at one address";
    *out = l.release();
    return VB_OK;
    VB_NS_END
}

int vb_ns_matrices_destroy(vb_ns_matrices *l)
{
    delete l;
    return VB_OK;
}

int vb_orthogonalize(vb_ns_plan *p, const vb_ns_matrices *inputs, const vb_ns_matrices *outputs)
{
    VB_NS_BEGIN
    DeviceGuard guard;
    VB_TRY(begin_call(p, &guard));
    VB_TRY(check_list(p, inputs, "inputs", false, false));
    VB_TRY(check_list(p, outputs, "outputs", true, false));
    VB_TRY(check_alias(inputs, outputs, "input and output", true));
    NsElementwise w = p->ew;
    w.planes = p->planes;
    w.eps = p->eps;
    w.types[0] = inputs->dtype;
    w.types[1] = outputs->dtype;
    return run_plan(p, w, false, inputs->turned || outputs->turned, [&](int64_t i, NsMatrixArg &a) {
        const size_t k = (size_t)i;
        a.a[0] = inputs->arrays[k];
        a.a[1] = outputs->arrays[k];
        a.direct = (uint32_t)inputs->vec[k] | (uint32_t)outputs->vec[k] << 1;
        a.live = 1;
        a.scale = 1.0f;
    });
    VB_NS_END
}

int vb_muon_multi_tensor_step(vb_ns_plan *p, const vb_muon_step_params *hp, const vb_ns_matrices *params,
                              const vb_ns_matrices *grads, const vb_ns_matrices *velocities, const float *scales)
{
    VB_NS_BEGIN
    DeviceGuard guard;
    VB_TRY(begin_call(p, &guard));
    if (!hp) return fail(VB_ERR_INVALID_ARG, "hp is null");
    if (!std::isfinite(hp->lr) || !std::isfinite(hp->momentum) || !std::isfinite(hp->weight_decay))
        return fail(VB_ERR_INVALID_ARG, "hyper-parameters must be finite");
    VB_TRY(check_list(p, params, "params", true, false));
    VB_TRY(check_list(p, grads, "grads", false, true));
    VB_TRY(check_list(p, velocities, "velocities", true, false));
    VB_TRY(check_alias(params, velocities, "parameter and velocity", false));
    VB_TRY(check_alias(params, grads, "parameter and gradient", false));
    VB_TRY(check_alias(velocities, grads, "velocity and gradient", false));
    NsElementwise w = p->ew;
    w.planes = p->planes;
    w.eps = p->eps;
    w.types[0] = grads->dtype;
    w.types[1] = velocities->dtype;
    w.types[2] = params->dtype;
    w.momentum = hp->momentum;
    w.nesterov = hp->nesterov != 0;
    w.decay = (float)(1.0 - (double)hp->lr * (double)hp->weight_decay);
    w.rate = hp->lr;
    return run_plan(p, w, true, grads->turned || velocities->turned || params->turned, [&](int64_t i, NsMatrixArg &a) {
        const size_t k = (size_t)i;
        a.a[0] = grads->arrays[k];
        a.a[1] = velocities->arrays[k];
        a.a[2] = params->arrays[k];
        a.direct = (uint32_t)grads->vec[k] | (uint32_t)velocities->vec[k] << 1 | (uint32_t)params->vec[k] << 2;
        a.live = grads->arrays[k].ptr != nullptr;
        a.scale = scales ? scales[i] : 1.0f;
    });
    VB_NS_END
}

int vb_debug_ns_plan_withhold_loads(vb_ns_plan *p, uint32_t wait_limit)
{
    if (!p) return fail(VB_ERR_INVALID_ARG, "plan is null");
    p->withhold = true;
    p->wait_limit = wait_limit;
    return VB_OK;
}

}  // extern "C"
