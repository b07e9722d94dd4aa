// experts.hip -- posterior means of many local experts at once: a query point has k slots, each names an expert and its weight,
//     mean(q) = prior(q) + sum_j w_qj m_{e(q,j)}(x_q),     m_e(x) = sum_{i in expert e} k(x, x_i) alpha_i
// (mod.rs:226-244 with cached K^-1 y, for one expert), and the gradients
//     dw_qj = dmean_q m_{e(q,j)}(x_q),     dalpha_i = sum over the slots (q, j) of i's expert of dmean_q w_qj k(x_q, x_i).
// Both sums are the same product of a covariance block with a vector, once along the points and once along the slots, so one kernel does
// both.  Slots are first sorted by expert (stable: every sum keeps one order) and their query points packed in that order.
#include "kprog_device.hpp"
#include "typed.hpp"

namespace fr {

constexpr int kMaxExperts = 1024;
constexpr int kPlanThreads = 1024;
constexpr int kPlanHeld = 4096;  // slots of an expert whose list stays in LDS
constexpr int kSide = 64;   // lanes of a wave, one slot (or point) each
constexpr int kStep = 8;    // points (or slots) that a lane works on at a time

struct PlanArgs {
    int64_t m, k, slots, d, ldq, lde, ldw;
    int experts;
    const int* chosen;
    const double *Xq, *weights, *dmean;
    int64_t* starts;  // experts + 1: where an expert's slots begin in the list
    int* list;        // list place -> slot (slot j m + q: the j-th of query q); experts of more than kPlanHeld slots only
    int* place;       // slot -> its place in the list, -1 unused
    double* packed;   // d x slots, feature-major: query points in list order (null: blocks instead)
    double* blocks;   // ... or blocks of 8 places of the list: 8 (d + 1) doubles, feature by feature, then dmean_q w_qj (backward)
    // the other side in blocks, alpha behind the features: by the workgroups behind the experts'
    const double *X, *alpha;
    double* points;
    int64_t n, ldx;
};

// element (row, f) of a side that is kept in blocks of 8 rows: features in fours (the last four padded with zeros on both sides, which add
// nothing to a distance or a product), then the weights
__host__ __device__ __forceinline__ int64_t fours(int64_t d) { return (d + 3) & ~(int64_t)3; }
__device__ __forceinline__ int64_t block_index(int64_t row, int64_t f, int64_t d) { return (row >> 3) * (8 * (fours(d) + 1)) + f * 8 + (row & 7); }

// A workgroup per expert: every wave counts, among its share of the queries, the slots that name this expert and those that name an earlier
// one, which is where the expert's list begins; a second walk puts each slot in its place, and the workgroup packs its list's query
// points.  No atomics: a list's order is that of (share, j, q) on every run.  Every workgroup reads all slots twice (16384 slots: 64 KB, from
// L2), which costs less than a launch to sort them first while experts times slots are few: 64 x 16384 are 0.1 GB, 1024 x 2^20 would be 8.6 GB
// and take longer than the products of experts of 64 points.  Bound by
// latency, the two walks and the packing behind them: 6.5 us for 6 slots of 16 experts, 14 us for 16384 slots of 64 experts and 65536 points of 16
// features (8 MB read and written).  The list stays in LDS where it fits: written to memory and read again it took 1 us more.
// (loads under a condition are waited for one by one: out of range they read the last place instead)
__global__ __launch_bounds__(kPlanThreads) void experts_plan_kernel(const PlanArgs a)
{
    constexpr int WAVES = kPlanThreads / 64;
    __shared__ int mine[WAVES], before[WAVES], held[kPlanHeld];
    if ((int)blockIdx.x >= a.experts) {
        const int64_t step = (int64_t)(gridDim.x - a.experts) * kPlanThreads;
        for (int64_t i = (int64_t)(blockIdx.x - a.experts) * kPlanThreads + threadIdx.x; i < a.n; i += step) {
            for (int64_t f0 = 0; f0 < a.d; f0 += 8) {
                double v[8];
#pragma unroll
                for (int f = 0; f < 8; ++f) v[f] = a.X[i + (f0 + f < a.d ? f0 + f : a.d - 1) * a.ldx];
#pragma unroll
                for (int f = 0; f < 8; ++f)
                    if (f0 + f < a.d) a.points[block_index(i, f0 + f, a.d)] = v[f];
            }
            for (int64_t f = a.d; f < fours(a.d); ++f) a.points[block_index(i, f, a.d)] = 0.0;
            a.points[block_index(i, fours(a.d), a.d)] = a.alpha[i];
        }
        return;
    }
    const int e = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int m = (int)a.m, k = (int)a.k;
    const int share = (m + WAVES * 64 - 1) / (WAVES * 64) * 64;
    const int lo = wave * share < m ? wave * share : m, hi = lo + share < m ? lo + share : m;
    // eight looks at a time: the stores of the second walk would put each load behind the one before it
    constexpr int LOOKS = 8;
    auto look = [&](int j, int q, int (&at)[LOOKS]) {
        const int* chosen = a.chosen + j * a.lde;
#pragma unroll
        for (int i = 0; i < LOOKS; ++i) {
            const int p = q + 64 * i + lane;
            const int v = chosen[p < hi ? p : hi - 1];
            at[i] = p < hi ? v : -1;
        }
    };
    int own = 0, early = 0;
    for (int j = 0; j < k; ++j)
        for (int q = lo; q < hi; q += 64 * LOOKS) {
            int at[LOOKS];
            look(j, q, at);
#pragma unroll
            for (int i = 0; i < LOOKS; ++i) {
                own += __popcll(__ballot(at[i] == e));
                early += __popcll(__ballot(at[i] >= 0 && at[i] < e));
            }
        }
    if (lane == 0) {
        mine[wave] = own;
        before[wave] = early;
    }
    __syncthreads();
    int start = 0, place = 0, total = 0;
    for (int w = 0; w < WAVES; ++w) {
        start += before[w];
        if (w < wave) place += mine[w];
        total += mine[w];
    }
    place += start;
    if (threadIdx.x == 0) {
        a.starts[e] = start;
        if (e == a.experts - 1) a.starts[a.experts] = start + total;
    }
    for (int j = 0; j < k; ++j)
        for (int q = lo; q < hi; q += 64 * LOOKS) {
            int at[LOOKS];
            look(j, q, at);
#pragma unroll
            for (int i = 0; i < LOOKS; ++i) {
                const unsigned long long all = __ballot(at[i] == e);
                const int slot = q + 64 * i + lane;
                if (at[i] == e) {
                    const int p = place + __popcll(all & ((1ull << lane) - 1));
                    a.place[j * a.m + slot] = p;
                    if (total <= kPlanHeld)
                        held[p - start] = (int)(j * a.m) + slot;
                    else
                        a.list[p] = (int)(j * a.m) + slot;
                } else if (e == 0 && slot < hi && (at[i] < 0 || at[i] >= a.experts))
                    a.place[j * a.m + slot] = -1;
                place += __popcll(all);
            }
        }
    __syncthreads();  // (the list is this workgroup's own: no other reads or writes its part)
    for (int i = threadIdx.x; i < total; i += kPlanThreads) {
        const int slot = total <= kPlanHeld ? held[i] : a.list[start + i], j = slot / m, q = slot - j * m;
        if (a.dmean) a.blocks[block_index(start + i, fours(a.d), a.d)] = a.dmean[q] * a.weights[q + j * a.ldw];
        if (a.blocks)
            for (int64_t f = a.d; f < fours(a.d); ++f) a.blocks[block_index(start + i, f, a.d)] = 0.0;
        for (int64_t f0 = 0; f0 < a.d; f0 += 8) {
            double v[8];
#pragma unroll
            for (int f = 0; f < 8; ++f) v[f] = a.Xq[q + (f0 + f < a.d ? f0 + f : a.d - 1) * a.ldq];
#pragma unroll
            for (int f = 0; f < 8; ++f)
                if (f0 + f < a.d) (a.packed ? a.packed[(f0 + f) * a.slots + start + i] : a.blocks[block_index(start + i, f0 + f, a.d)]) = v[f];
        }
    }
}

struct BlockArgs {
    fr_kprog prog;
    int64_t d;
    int experts;
    // two sides of points, expert e's rows are [begin[e], begin[e+1]) of each: one by columns, feature f at x + f * ld, one in blocks of 8
    // rows, whose last row of 8 are its weights
    const double *x, *xv, *blocks;
    int64_t ld, rows, block_rows;
    const int64_t *begin, *block_begin;
    double* part;  // sums over a piece of the side summed over: row of the other side + piece * its rows
    int64_t piece;
};

__device__ __forceinline__ int64_t row_of(const int64_t* begin, int e, int64_t rows)
{
    const int64_t v = begin[e];
    return v < 0 ? 0 : (v > rows ? rows : v);
}

// A piece is `piece` rows (a multiple of 8) of blocks of 8, the first and the last of an expert shared with its neighbours.
__device__ __forceinline__ int64_t pieces_of(int64_t r0, int64_t r1, int64_t piece)
{
    return r1 > r0 ? ((((r1 + 7) >> 3) - (r0 >> 3)) * 8 + piece - 1) / piece : 0;
}

// read-only data at addresses that are the same for the whole wave: scalar loads, eight neighbouring doubles in one
typedef double eight __attribute__((ext_vector_type(8)));
typedef const char __attribute__((address_space(4))) * scalar_ptr;
__device__ __forceinline__ scalar_ptr scalar(const double* p) { return (scalar_ptr)(uintptr_t)p; }
__device__ __forceinline__ eight load_eight(scalar_ptr p)
{
    eight v;
    __builtin_memcpy(&v, (const double __attribute__((address_space(4)))*)p, sizeof(v));
    return v;
}
__device__ __forceinline__ int64_t same(int64_t v)
{
    const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)v), hi = __builtin_amdgcn_readfirstlane((unsigned)(v >> 32));
    return (int64_t)((unsigned long long)hi << 32 | lo);
}

// 2^y for y <= 0, to a rounding or two: the rest of y after its nearest integer is exact, and the series of 2^r about 0 has a remainder of
// 4e-18 at |r| = 1/2.  A pair of instructions fewer than e^x, and none for large arguments.
__device__ __forceinline__ double exp2_falling(double y)
{
    const double n = __builtin_rint(y), r = y - n;
    constexpr double C[12] = {2.5678435993488206e-11, 4.4455382718708116e-10, 7.054911620801123e-09, 1.01780860092397e-07,  1.321548679014431e-06, 1.5252733804059841e-05,
                              0.0001540353039338161,  0.0013333558146428443,  0.009618129107628477,  0.05550410866482158, 0.24022650695910072, 0.6931471805599453};
    double p = 1.3691488853904128e-12;  // ln(2)^13 / 13!
#pragma unroll
    for (int i = 0; i < 12; ++i) p = __builtin_fma(p, r, C[i]);
    const double e = __builtin_ldexp(__builtin_fma(p, r, 1.0), (int)n);
    return y < -1080.0 ? 0.0 : e;  // (-inf has no r)
}

// The covariance from s and u, without the amplitude that kernels of one length scale begin with: it multiplies the sum.  They also multiply by
// the length's inverse, worked out once, where the Gram kernel divides: a rounding of the exponent more, which the sum over the points
// hides, for five instructions less a pair.
constexpr double kLog2e = 1.4426950408889634;
template <int LEAF>
__device__ __forceinline__ double pair_value(const fr_kprog& p, double inverse, double s, double u)
{
    if constexpr (LEAF == FR_K_SQUAREDEXP) return exp2_falling(-(s * inverse));
    if constexpr (LEAF == FR_K_EXPONENTIAL) return exp2_falling(-(sqrt(s) * inverse));
    if constexpr (LEAF == FR_K_MATERN1) {
        const double x = sqrt(s) * inverse;
        return (1.0 + x) * exp2_falling(-(x * kLog2e));
    }
    if constexpr (LEAF == FR_K_MATERN2) {
        const double x = sqrt(s) * inverse;
        return __builtin_fma(x, x * (1.0 / 3.0), 1.0 + x) * exp2_falling(-(x * kLog2e));
    }
    return kprog_eval_k<LEAF>(p, s, u);
}
template <int LEAF>
__device__ __forceinline__ double pair_inverse(const fr_kprog& p)
{
    const double ls = p.ops[0].params[0];
    if constexpr (LEAF == FR_K_SQUAREDEXP || LEAF == FR_K_EXPONENTIAL) return kLog2e / (2.0 * ls * ls);
    if constexpr (LEAF == FR_K_MATERN1) return sqrt(3.0) / fabs(ls);
    if constexpr (LEAF == FR_K_MATERN2) return sqrt(5.0) / fabs(ls);  // 5 s / (3 ls^2) = x^2 / 3
    return 0.0;
}
template <int LEAF>
__device__ __forceinline__ double pair_scale(const fr_kprog& p)
{
    return LEAF == FR_K_SQUAREDEXP || LEAF == FR_K_EXPONENTIAL || LEAF == FR_K_MATERN1 || LEAF == FR_K_MATERN2 ? fabs(p.ops[0].params[1]) : 1.0;
}

// kStep covariances of the lane's point with the points of a block.  The distance is summed from the differences, feature by feature, as the
// Gram kernel does: |x|^2 + |y|^2 - 2 x.y on the matrix cores would lose near points' distances to cancellation, which the square root in
// three of the kernels turns into an error of 1e-8.  That makes 2 d + about 22 f64 instructions a pair, at 4 cycles a wave and SIMD.  The
// block comes through scalar loads of one line each, eight points of a feature: it costs no vector register and no LDS traffic (a broadcast
// read of LDS for every 16 instructions would keep the LDS pipe of the CU busier than its SIMDs), and a block is contiguous, so its
// lines need one address.
template <int LEAF>
struct Pairs {
    static constexpr bool S = LEAF < 0 || !(LEAF == FR_K_LINEAR || LEAF == FR_K_POLYNOMIAL || LEAF == FR_K_HYPERTAN);
    static constexpr bool U = LEAF < 0 || !S;
    double s[kStep], u[kStep];
    __device__ __forceinline__ void feature(const eight& y, double x)
    {
#pragma unroll
        for (int t = 0; t < kStep; ++t) {
            if constexpr (S) {
                const double z = x - y[t];
                s[t] = __builtin_fma(z, z, s[t]);
            }
            if constexpr (U) u[t] = __builtin_fma(x, y[t], u[t]);
        }
    }
    // x: the lane's point, features in fours
    __device__ __forceinline__ void four(scalar_ptr block, const double (&x)[4])
    {
        const eight y0 = load_eight(block), y1 = load_eight(block + 64), y2 = load_eight(block + 128), y3 = load_eight(block + 192);
        __builtin_amdgcn_sched_barrier(0);
        feature(y0, x[0]);
        feature(y1, x[1]);
        feature(y2, x[2]);
        feature(y3, x[3]);
    }
    __device__ __forceinline__ void clear()
    {
#pragma unroll
        for (int t = 0; t < kStep; ++t) s[t] = u[t] = 0.0;
    }
};

// four features of a point kept by columns, 0 behind the last
__device__ __forceinline__ void load_four(const double* x, int64_t ld, int f, int d, double (&v)[4])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = x[(f + i < d ? f + i : d - 1) * ld];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = f + i < d ? v[i] : 0.0;
}

// number of items in front of each expert's, and of all
__device__ __forceinline__ void count_items(const BlockArgs& a, int64_t* items, bool blocks_are_tiles)
{
    const int lane = threadIdx.x & 63;
    if (threadIdx.x < 64) {
        int64_t total = 0;
        for (int e0 = 0; e0 < a.experts; e0 += 64) {
            const int e = e0 + lane;
            int64_t v = 0;
            if (e < a.experts) {
                const int64_t r0 = row_of(a.begin, e, a.rows), r1 = row_of(a.begin, e + 1, a.rows);
                const int64_t b0 = row_of(a.block_begin, e, a.block_rows), b1 = row_of(a.block_begin, e + 1, a.block_rows);
                if (r1 > r0 && b1 > b0) v = blocks_are_tiles ? pieces_of(b0, b1, 8) * ((r1 - r0 + a.piece - 1) / a.piece) : (r1 - r0 + kSide - 1) / kSide * pieces_of(b0, b1, a.piece);
            }
            int64_t s = v;
            for (int step = 1; step < 64; step *= 2) {
                const int64_t o = __shfl_up(s, step);
                if (lane >= step) s += o;
            }
            if (e < a.experts) items[e] = total + s - v;
            total += __shfl(s, 63);
        }
        if (lane == 0) items[a.experts] = total;
    }
    __syncthreads();
}
__device__ __forceinline__ int expert_of(const BlockArgs& a, const int64_t* items, int64_t item)
{
    int lo = 0, hi = a.experts - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (items[mid] <= item)
            lo = mid;
        else
            hi = mid - 1;
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

// A lane for each row of the columns' side, the sum over the blocks: an item is a wave of 64 lanes times a piece of blocks.  FOURS > 0: the
// lanes' features stay in registers; 0: there are more than 16, and they are read again for every block.  Bound by issue of f64
// instructions, which take three fifths of the SIMDs' time: 16777216 pairs of 16 features (squared exponential, 64 experts of 500 to 1500
// points) take 51 us, where 54 instructions a pair would take 23; the rest are lanes of partial tiles, waits for scalar loads and uneven
// ends; 7500000 in the backward pass 27 us.  40 items a CU, on no more workgroups than the chip
// holds, even skewed experts out: whole calls with 20 items on 8 workgroups took 74 and 41 us, with 40 on 5 70 and 39, with 80 on 5 75 and 48.
template <int LEAF, int FOURS>
__global__ __launch_bounds__(256) void experts_lanes_kernel(const BlockArgs a)
{
    __shared__ int64_t items[kMaxExperts + 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const double inverse = pair_inverse<LEAF>(a.prog);
    count_items(a, items, false);
    const int64_t all = items[a.experts];
    const int d = (int)a.d;
    const int64_t stride = 64 * (fours(a.d) + 1);  // of a block, in bytes
    // workgroups are dealt to the 8 XCDs in turn: each XCD takes a stretch of the items, so that an expert's points are in one L2; the
    // waves of a workgroup take neighbouring tiles of the same piece, so that a line in the scalar cache serves all four
    const int64_t share = (all + 31) / 32 * 4, xcd = blockIdx.x & 7;
    for (int64_t turn = (blockIdx.x >> 3) * 4 + wave; turn < share; turn += (gridDim.x >> 3) * 4) {
        const int64_t item = xcd * share + turn;
        if (item >= all) break;
        const int e = expert_of(a, items, item);
        const int64_t r0 = row_of(a.begin, e, a.rows), r1 = row_of(a.begin, e + 1, a.rows);
        const int64_t b0 = same(row_of(a.block_begin, e, a.block_rows)), b1 = same(row_of(a.block_begin, e + 1, a.block_rows));
        const int64_t tiles = (r1 - r0 + kSide - 1) / kSide, mine = item - items[e];
        const int64_t piece = same(mine / tiles), tile = mine - piece * tiles;
        const int64_t row = r0 + tile * kSide + lane;
        const double* x = a.x + (row < r1 ? row : r1 - 1);
        double held[FOURS ? FOURS : 1][4];
        if constexpr (FOURS > 0)
#pragma unroll
            for (int f = 0; f < FOURS; ++f) load_four(x, a.ld, 4 * f, d, held[f]);
        const int64_t from = (b0 & ~(int64_t)7) + piece * a.piece, to = from + a.piece < b1 ? from + a.piece : b1;
        scalar_ptr block = scalar(a.blocks) + (from >> 3) * stride;
        double acc = 0.0;
        for (int64_t j = from; j < to; j += 8, block += stride) {
            Pairs<LEAF> p;
            p.clear();
            if constexpr (FOURS > 0) {
#pragma unroll
                for (int f = 0; f < FOURS; ++f) p.four(block + f * 256, held[f]);
            } else
                for (int f = 0; f < d; f += 4) {
                    load_four(x, a.ld, f, d, held[0]);
                    p.four(block + f * 64, held[0]);
                }
            const eight v = load_eight(block + stride - 64);
            if (j >= b0 && j + 8 <= to) {
#pragma unroll
                for (int t = 0; t < kStep; ++t) acc = __builtin_fma(pair_value<LEAF>(a.prog, inverse, p.s[t], p.u[t]), v[t], acc);
            } else {
#pragma unroll
                for (int t = 0; t < kStep; ++t)
                    if (j + t >= b0 && j + t < to) acc = __builtin_fma(pair_value<LEAF>(a.prog, inverse, p.s[t], p.u[t]), v[t], acc);
            }
        }
        if (row < r1) a.part[row + piece * a.rows] = acc * pair_scale<LEAF>(a.prog);
    }
}

// A lane for each row of the columns' side too, but the sum is over the lanes: an item is a block of 8 slots times a piece of the expert's
// points, which the four waves share out; the points' features are read again for every block.  For few slots an expert, where lanes of slots
// would be empty (16 experts of 1024 points of 16
// features, 3 queries of 2 slots: 7 us, most of it latency).  4 items a CU: with 2, 512 queries
// of 40 features took 33 us instead of 29, 8 took as long.
template <int LEAF>
__global__ __launch_bounds__(256) void experts_few_kernel(const BlockArgs a)
{
    __shared__ int64_t items[kMaxExperts + 1];
    __shared__ double sums[4][kStep];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const double inverse = pair_inverse<LEAF>(a.prog);
    count_items(a, items, true);
    const int64_t all = items[a.experts];
    for (int64_t item = blockIdx.x; item < all; item += gridDim.x) {
        const int e = expert_of(a, items, item);
        const int64_t r0 = row_of(a.begin, e, a.rows), r1 = row_of(a.begin, e + 1, a.rows);
        const int64_t b0 = same(row_of(a.block_begin, e, a.block_rows)), b1 = same(row_of(a.block_begin, e + 1, a.block_rows));
        const int64_t pieces = (r1 - r0 + a.piece - 1) / a.piece, mine = item - items[e];
        const int64_t tile = same(mine / pieces), piece = mine - tile * pieces;
        const int64_t j = (b0 & ~(int64_t)7) + tile * 8;
        const int64_t from = r0 + piece * a.piece, to = from + a.piece < r1 ? from + a.piece : r1;
        const int d = (int)a.d;
        scalar_ptr block = scalar(a.blocks) + (j >> 3) * (64 * (fours(a.d) + 1));
        double acc[kStep];
#pragma unroll
        for (int t = 0; t < kStep; ++t) acc[t] = 0.0;
        for (int64_t i = from + wave * kSide; i < to; i += 4 * kSide) {
            const bool in = i + lane < to;
            const double* x = a.x + (in ? i + lane : to - 1);
            const double v = a.xv[in ? i + lane : to - 1];
            Pairs<LEAF> p;
            p.clear();
            for (int f = 0; f < d; f += 4) {
                double w[4];
                load_four(x, a.ld, f, d, w);
                p.four(block + f * 64, w);
            }
#pragma unroll
            for (int t = 0; t < kStep; ++t) acc[t] = __builtin_fma(pair_value<LEAF>(a.prog, inverse, p.s[t], p.u[t]), in ? v : 0.0, acc[t]);
        }
#pragma unroll
        for (int step = 1; step < 64; step *= 2)
#pragma unroll
            for (int t = 0; t < kStep; ++t) acc[t] += __shfl_xor(acc[t], step);
        if (lane == 0)
#pragma unroll
            for (int t = 0; t < kStep; ++t) sums[wave][t] = acc[t];
        __syncthreads();
        if (threadIdx.x < kStep && j + threadIdx.x >= b0 && j + threadIdx.x < b1)
            a.part[j + threadIdx.x + piece * a.block_rows] =
                (((sums[0][threadIdx.x] + sums[1][threadIdx.x]) + sums[2][threadIdx.x]) + sums[3][threadIdx.x]) * pair_scale<LEAF>(a.prog);
        __syncthreads();
    }
}

struct JoinArgs {
    int64_t m, k, slots, n, lde, ldw, lds, lddw, piece;
    int experts;
    bool few;
    const int* chosen;
    const int* place;
    const int64_t *begin, *starts;
    const double *part, *weights, *prior, *dmean;
    const double* slots_in;
    double *mean, *slots_out, *dweights, *dalpha;
};

// the sum of a row's pieces, in their order
__device__ __forceinline__ double add_pieces(const double* part, int64_t ld, int64_t pieces)
{
    double v = 0.0;
    for (int64_t c0 = 0; c0 < pieces; c0 += 8) {
        double next[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) next[c] = part[(c0 + c < pieces ? c0 + c : c0) * ld];
#pragma unroll
        for (int c = 0; c < 8; ++c) v += c0 + c < pieces ? next[c] : 0.0;
    }
    return v;
}

// Forward: a workgroup takes 64 query points, a thread adds up the pieces of a slot, then the first 64 threads the slots of a point (16384
// slots: 8 us; a thread for each query, adding its slots one after the other, took 5 us more).
constexpr int kMeanPoints = 64, kMeanThreads = 256;
__global__ __launch_bounds__(kMeanThreads) void experts_mean_kernel(const JoinArgs a)
{
    __shared__ double terms[64][kMeanPoints];
    const int64_t q0 = (int64_t)blockIdx.x * kMeanPoints;
    const int points = a.m - q0 < kMeanPoints ? (int)(a.m - q0) : kMeanPoints;
    for (int i = threadIdx.x; i < (int)a.k * kMeanPoints; i += kMeanThreads) {
        const int j = i / kMeanPoints, at = i % kMeanPoints;
        if (at >= points) continue;
        const int64_t q = q0 + at;
        const int e = a.chosen[q + j * a.lde];
        const int64_t p = a.place[j * a.m + q];
        const double w = a.weights[q + j * a.ldw];
        double v = 0.0;
        if (p >= 0) {
            const int64_t r0 = row_of(a.begin, e, a.n), r1 = row_of(a.begin, e + 1, a.n);
            v = add_pieces(a.part + p, a.slots, a.few ? (r1 - r0 + a.piece - 1) / a.piece : pieces_of(r0, r1, a.piece));
        }
        if (a.slots_out) a.slots_out[q + j * a.lds] = v;
        terms[j][at] = w * v;
    }
    __syncthreads();
    if ((int)threadIdx.x < points) {
        double mean = a.prior ? a.prior[q0 + threadIdx.x] : 0.0;
        for (int64_t j = 0; j < a.k; ++j) mean += terms[j][threadIdx.x];
        a.mean[q0 + threadIdx.x] = mean;
    }
}

// backward: the gradient of each coefficient from its pieces, of each weight from its slot's mean (32768 points, 8192 slots: 4.2 us, latency)
__global__ __launch_bounds__(256) void experts_gradient_kernel(const JoinArgs a)
{
    const int64_t id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (a.dalpha && id < a.n) {
        int lo = 0, hi = a.experts - 1;  // the expert of point id, if any
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (row_of(a.begin, mid, a.n) <= id)
                lo = mid;
            else
                hi = mid - 1;
        }
        const bool owned = id >= row_of(a.begin, lo, a.n) && id < row_of(a.begin, lo + 1, a.n);
        a.dalpha[id] = owned ? add_pieces(a.part + id, a.n, pieces_of(a.starts[lo], a.starts[lo + 1], a.piece)) : 0.0;
    }
    if (a.dweights && id < a.slots) {
        const int64_t q = id % a.m, j = id / a.m;
        const int e = a.chosen[q + j * a.lde];
        a.dweights[q + j * a.lddw] = e >= 0 && e < a.experts ? a.dmean[q] * a.slots_in[q + j * a.lds] : 0.0;
    }
}

// Rows of a piece, so that there are about `want` items of `tiles` tiles; a multiple of `least`, kept from making more than 256 MB of pieces
// for `lanes` results on skewed experts (a result's pieces lie apart whatever its expert's real size).
static int64_t piece_rows(int64_t want, int64_t tiles, int64_t rows, int64_t experts, int64_t lanes, int64_t least)
{
    const int64_t pieces = (want + tiles - 1) / tiles, each = rows / experts + 1;
    int64_t piece = (each + pieces - 1) / pieces;
    const int64_t bound = lanes * rows >> 25;
    return round_up(piece > bound ? piece : bound, least);
}

template <int LEAF, bool FEW>
static void leaf_launch(fr_ctx* ctx, const BlockArgs& a, dim3 grid)
{
    const dim3 block(256);
    if constexpr (FEW)
        hipLaunchKernelGGL((experts_few_kernel<LEAF>), grid, block, 0, ctx->ls, a);
    else if (a.d <= 4)
        hipLaunchKernelGGL((experts_lanes_kernel<LEAF, 1>), grid, block, 0, ctx->ls, a);
    else if (a.d <= 8)
        hipLaunchKernelGGL((experts_lanes_kernel<LEAF, 2>), grid, block, 0, ctx->ls, a);
    else if (a.d <= 12)
        hipLaunchKernelGGL((experts_lanes_kernel<LEAF, 3>), grid, block, 0, ctx->ls, a);
    else if (a.d <= 16)
        hipLaunchKernelGGL((experts_lanes_kernel<LEAF, 4>), grid, block, 0, ctx->ls, a);
    else
        hipLaunchKernelGGL((experts_lanes_kernel<LEAF, 0>), grid, block, 0, ctx->ls, a);
}

template <bool FEW>
static int block_launch(fr_ctx* ctx, const BlockArgs& a, int64_t items)
{
    // a workgroup for each item if the experts are alike (any number of them finishes the list), no more than the chip holds: 4 or 5 waves a SIMD
    const int64_t cap = (int64_t)ctx->num_cus * 5;
    const dim3 grid((unsigned)round_up(items < 1 ? 1 : (items < cap ? items : cap), 8));
    const int leaf = a.prog.nops == 1 ? a.prog.ops[0].kind : -1;
#define FR_EXPERTS_LEAF(KIND) \
    case KIND: leaf_launch<KIND, FEW>(ctx, a, grid); break;
    switch (leaf) {
        FR_EXPERTS_LEAF(FR_K_LINEAR)
        FR_EXPERTS_LEAF(FR_K_POLYNOMIAL)
        FR_EXPERTS_LEAF(FR_K_SQUAREDEXP)
        FR_EXPERTS_LEAF(FR_K_EXPONENTIAL)
        FR_EXPERTS_LEAF(FR_K_MATERN1)
        FR_EXPERTS_LEAF(FR_K_MATERN2)
        FR_EXPERTS_LEAF(FR_K_HYPERTAN)
        FR_EXPERTS_LEAF(FR_K_MULTIQUADRIC)
        FR_EXPERTS_LEAF(FR_K_RATIONALQUADRATIC)
    default: leaf_launch<-1, FEW>(ctx, a, grid);
    }
#undef FR_EXPERTS_LEAF
    FR_HIP(ctx, hipGetLastError());
    return FR_OK;
}

static int experts_check(fr_ctx* ctx, const fr_kprog* kernel, int64_t n, int64_t d, int64_t n_experts, int64_t m, int64_t k, const void* offsets)
{
    FR_TRY(kprog_check(ctx, kernel));
    if (n < 0 || d < 1 || m < 0) return set_err(ctx, FR_SHAPE, "%lld points of %lld features, %lld queries", (long long)n, (long long)d, (long long)m);
    if (d > (int64_t)1 << 24) return set_err(ctx, FR_SHAPE, "%lld features: at most 2^24", (long long)d);  // (the kernels count a block's bytes in 32 bits)
    if (n_experts < 1 || n_experts > kMaxExperts) return set_err(ctx, FR_SHAPE, "%lld experts: 1 to %d", (long long)n_experts, kMaxExperts);
    if (k < 1 || k > 64) return set_err(ctx, FR_SHAPE, "%lld slots a query: 1 to 64", (long long)k);
    if (m > ((int64_t)1 << 30) / k || n > (int64_t)1 << 31) return set_err(ctx, FR_SHAPE, "more than 2^30 slots or 2^31 points");
    if (!offsets) return set_err(ctx, FR_INVALID_ARGUMENT, "offsets: null pointer");
    return FR_OK;
}

// offsets that the host can see are checked here; those in device memory the kernels keep inside [0, n]
static int experts_offsets(fr_ctx* ctx, Operand& o, const void* offsets, int64_t n_experts, int64_t n)
{
    FR_TRY(o.stage(offsets, n_experts + 1, 1, n_experts + 1, 8, "offsets"));
    if ((const void*)o.dev == offsets) return FR_OK;
    const int64_t* v = (const int64_t*)offsets;
    for (int64_t e = 0; e <= n_experts; ++e)
        if (v[e] < (e ? v[e - 1] : 0) || v[e] > n) return set_err(ctx, FR_SHAPE, "offsets[%lld] = %lld: not in order within [0, %lld]", (long long)e, (long long)v[e], (long long)n);
    return FR_OK;
}

}  // namespace fr

using namespace fr;

extern "C" {

int fr_experts_predict(fr_ctx* ctx, const fr_kprog* kernel, const double* X, int64_t n, int64_t ldx, int64_t d, const double* alpha, const void* offsets,
                       int64_t n_experts, const double* Xq, int64_t m, int64_t ldq, const void* experts, int64_t lde, const double* weights, int64_t ldw,
                       int64_t k, const double* prior_q, double* out_mean, double* out_slots, int64_t lds)
{
    return op_entry(ctx, [&]() -> int {
        FR_TRY(experts_check(ctx, kernel, n, d, n_experts, m, k, offsets));
        Operand ox(ctx), oa(ctx), oo(ctx), oq(ctx), oe(ctx), ow(ctx), op(ctx), om(ctx), os(ctx);
        FR_TRY(ox.stage(X, n, d, ldx, 8, "X"));
        FR_TRY(oa.stage(alpha, n, 1, n, 8, "alpha"));
        FR_TRY(experts_offsets(ctx, oo, offsets, n_experts, n));
        FR_TRY(oq.stage(Xq, m, d, ldq, 8, "Xq"));
        FR_TRY(oe.stage(experts, m, k, lde, 4, "experts"));
        FR_TRY(ow.stage(weights, m, k, ldw, 8, "weights"));
        if (prior_q) FR_TRY(op.stage(prior_q, m, 1, m, 8, "prior_q"));
        FR_TRY(om.stage(out_mean, m, 1, m, 8, "out_mean", true));
        if (out_slots) FR_TRY(os.stage(out_slots, m, k, lds, 8, "out_slots", true));
        if (m == 0) return FR_OK;
        const int64_t slots = m * k;
        // Few slots an expert: sums over lanes of points; else a lane for each slot.  us, the one / the other, at 32, 64, 128, 192 and 256 slots an
        // expert: 64 experts of 128 points of 16 features 20 / 21, 20 / 24, 26 / 26, 29 / 29, 34 / 33; 8 of 8192 of 8 features 20 / 60,
        // 26 / 65, 33 / 58, 40 / 58, 51 / 61; at 64, 128, 192, 256 and 1024: 64 of 1024 of 16 features 39 / 44, 47 / 51, 57 / 59, 65 / 67,
        // 221 / 185; of 40 features at 256 and 1024 110 / 119, 403 / 393
        const bool few = slots < n_experts * 256;
        const int64_t used = slots < n_experts ? slots : n_experts, blocks = (slots + 7) / 8 + used, tiles = few ? blocks : slots / kSide + used;
        const int64_t want = (int64_t)ctx->num_cus * (few ? 4 : 40);
        const int64_t piece = piece_rows(want, tiles, n, n_experts, slots, few ? 256 : 8), pieces = n / piece + 2;
        const int64_t wide = 8 * (fours(d) + 1);
        OpWorkspace ws(ctx);
        // [points in blocks | slots in blocks or by columns | sums of pieces | where lists begin | slot <-> place]
        const int64_t in_points = few ? 0 : (n + 7) / 8 * wide, in_slots = few ? blocks * wide : d * slots;
        FR_TRY(ws.get((size_t)(8 * (in_points + in_slots + pieces * slots + n_experts + 1) + 8 * slots)));
        PlanArgs p = {};
        p.m = m, p.k = k, p.slots = slots, p.d = d, p.ldq = oq.ld, p.lde = oe.ld, p.ldw = ow.ld, p.experts = (int)n_experts;
        p.chosen = oe.as<int>(), p.Xq = oq.as<double>(), p.weights = ow.as<double>();
        p.points = (double*)ws.p;
        (few ? p.blocks : p.packed) = p.points + in_points;
        double* part = p.points + in_points + in_slots;
        p.starts = (int64_t*)(part + pieces * slots);
        p.place = (int*)(p.starts + n_experts + 1), p.list = p.place + slots;
        p.X = ox.as<double>(), p.alpha = oa.as<double>(), p.n = few ? 0 : n, p.ldx = ox.ld;
        const int64_t packers = few ? 0 : (n + kPlanThreads - 1) / kPlanThreads;
        hipLaunchKernelGGL(experts_plan_kernel, dim3((unsigned)(n_experts + (packers < 1024 ? packers : 1024))), dim3(kPlanThreads), 0, ctx->ls, p);
        BlockArgs b = {};
        b.prog = *kernel, b.d = d, b.experts = (int)n_experts, b.part = part, b.piece = piece;
        if (few) {
            b.x = ox.as<double>(), b.xv = oa.as<double>(), b.ld = ox.ld, b.rows = n, b.begin = oo.as<int64_t>();
            b.blocks = p.blocks, b.block_rows = slots, b.block_begin = p.starts;
            FR_TRY(block_launch<true>(ctx, b, blocks * (n / n_experts / piece + 1)));
        } else {
            b.x = p.packed, b.ld = slots, b.rows = slots, b.begin = p.starts;
            b.blocks = p.points, b.block_rows = n, b.block_begin = oo.as<int64_t>();
            FR_TRY(block_launch<false>(ctx, b, tiles * (n / n_experts / piece + 1) / 4));
        }
        JoinArgs j = {};
        j.m = m, j.k = k, j.slots = slots, j.n = n, j.lde = oe.ld, j.ldw = ow.ld, j.lds = os.ld, j.piece = piece, j.experts = (int)n_experts, j.few = few;
        j.chosen = p.chosen, j.place = p.place, j.begin = oo.as<int64_t>(), j.part = part, j.weights = p.weights, j.prior = op.as<double>();
        j.mean = om.as<double>(), j.slots_out = os.as<double>();
        hipLaunchKernelGGL(experts_mean_kernel, dim3((unsigned)((m + kMeanPoints - 1) / kMeanPoints)), dim3(kMeanThreads), 0, ctx->ls, j);
        FR_HIP(ctx, hipGetLastError());
        FR_TRY(om.commit());
        return os.commit();
    });
}

int fr_experts_backward(fr_ctx* ctx, const fr_kprog* kernel, const double* X, int64_t n, int64_t ldx, int64_t d, const void* offsets, int64_t n_experts,
                        const double* Xq, int64_t m, int64_t ldq, const void* experts, int64_t lde, const double* weights, int64_t ldw, int64_t k,
                        const double* slots_mean, int64_t lds, const double* dmean, double* dweights, int64_t lddw, double* dalpha)
{
    return op_entry(ctx, [&]() -> int {
        FR_TRY(experts_check(ctx, kernel, n, d, n_experts, m, k, offsets));
        Operand ox(ctx), oo(ctx), oq(ctx), oe(ctx), ow(ctx), os(ctx), om(ctx), odw(ctx), oda(ctx);
        FR_TRY(ox.stage(X, n, d, ldx, 8, "X"));
        FR_TRY(experts_offsets(ctx, oo, offsets, n_experts, n));
        FR_TRY(oq.stage(Xq, m, d, ldq, 8, "Xq"));
        FR_TRY(oe.stage(experts, m, k, lde, 4, "experts"));
        FR_TRY(ow.stage(weights, m, k, ldw, 8, "weights"));
        if (dweights) FR_TRY(os.stage(slots_mean, m, k, lds, 8, "slots"));
        FR_TRY(om.stage(dmean, m, 1, m, 8, "dmean"));
        if (dweights) FR_TRY(odw.stage(dweights, m, k, lddw, 8, "dweights", true));
        if (dalpha) FR_TRY(oda.stage(dalpha, n, 1, n, 8, "dalpha", true));
        if (!dweights && !dalpha) return FR_OK;
        const int64_t slots = m * k;
        JoinArgs j = {};
        j.m = m, j.k = k, j.slots = slots, j.n = n, j.lde = oe.ld, j.ldw = ow.ld, j.lds = os.ld, j.lddw = odw.ld, j.experts = (int)n_experts;
        j.chosen = oe.as<int>(), j.begin = oo.as<int64_t>(), j.dmean = om.as<double>(), j.slots_in = os.as<double>();
        j.dweights = odw.as<double>(), j.dalpha = oda.as<double>();
        OpWorkspace ws(ctx);
        if (dalpha && n > 0) {
            const int64_t used = n < n_experts ? n : n_experts, blocks = (slots + 7) / 8 + 1, tiles = n / kSide + used;
            const int64_t piece = piece_rows((int64_t)ctx->num_cus * 40, tiles, slots, n_experts, n, 8), pieces = slots / piece + 2;
            FR_TRY(ws.get((size_t)(8 * (blocks * 8 * (fours(d) + 1) + pieces * n + n_experts + 1) + 8 * slots)));
            PlanArgs p = {};
            p.m = m, p.k = k, p.slots = slots, p.d = d, p.ldq = oq.ld, p.lde = oe.ld, p.ldw = ow.ld, p.experts = (int)n_experts;
            p.chosen = oe.as<int>(), p.Xq = oq.as<double>(), p.weights = ow.as<double>(), p.dmean = om.as<double>();
            p.blocks = (double*)ws.p;
            double* part = p.blocks + blocks * 8 * (fours(d) + 1);
            p.starts = (int64_t*)(part + pieces * n);
            p.place = (int*)(p.starts + n_experts + 1), p.list = p.place + slots;
            hipLaunchKernelGGL(experts_plan_kernel, dim3((unsigned)n_experts), dim3(kPlanThreads), 0, ctx->ls, p);
            BlockArgs b = {};
            b.prog = *kernel, b.d = d, b.experts = (int)n_experts, b.part = part, b.piece = piece;
            b.x = ox.as<double>(), b.ld = ox.ld, b.rows = n, b.begin = oo.as<int64_t>();
            b.blocks = p.blocks, b.block_rows = slots, b.block_begin = p.starts;
            FR_TRY(block_launch<false>(ctx, b, tiles * (slots / n_experts / piece + 1) / 4));
            j.piece = piece, j.part = part, j.starts = p.starts;
        }
        const int64_t threads = slots > n ? slots : n;
        if (threads > 0) hipLaunchKernelGGL(experts_gradient_kernel, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, ctx->ls, j);
        FR_HIP(ctx, hipGetLastError());
        FR_TRY(odw.commit());
        return oda.commit();
    });
}

}  // extern "C"
