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
constexpr int kSide = 64;   // lanes of a wave, one slot (or point) each
constexpr int kStep = 8;    // points (or slots) that a lane works on at a time

struct PlanArgs {
    int64_t m, k, slots, d, n, ldq, lde, ldw;
    int experts;
    const int* chosen;
    const double *Xq, *weights, *dmean;
    int64_t* starts;  // experts + 1: where an expert's slots begin in the list
    int* place;       // slot -> its place in the list, -1 unused
    double* packed;   // d x slots, feature-major: query points in list order
    double* pull;     // slots: dmean_q w_qj in list order (backward)
};

// A workgroup per expert: every wave counts the slots of its share that name this expert and those that name an earlier one, which is
// where the expert's list begins; a second walk puts each slot in its place.  No atomics: the list keeps the slots' order.
__global__ __launch_bounds__(kPlanThreads) void experts_plan_kernel(const PlanArgs a)
{
    constexpr int WAVES = kPlanThreads / 64;
    __shared__ int64_t mine[WAVES], before[WAVES];
    const int e = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t share = (a.slots + WAVES * 64 - 1) / (WAVES * 64) * 64;
    const int64_t lo = wave * share, hi = lo + share < a.slots ? lo + share : a.slots;
    int64_t own = 0, early = 0;
    for (int64_t i = lo + lane; i - lane < hi; i += 64) {
        const int at = i < hi ? a.chosen[(i / a.k) + (i % a.k) * a.lde] : -1;
        own += __popcll(__ballot(at == e));
        early += __popcll(__ballot(at >= 0 && at < e));
    }
    if (lane == 0) {
        mine[wave] = own;
        before[wave] = early;
    }
    __syncthreads();
    int64_t start = 0, place = 0, total = 0;
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
    for (int64_t i = lo + lane; i - lane < hi; i += 64) {
        const int64_t q = i / a.k, j = i % a.k;
        const int at = i < hi ? a.chosen[q + j * a.lde] : -1;
        const unsigned long long all = __ballot(at == e);
        if (at == e) {
            const int64_t p = place + __popcll(all & ((1ull << lane) - 1));
            a.place[i] = (int)p;
            for (int64_t f = 0; f < a.d; ++f) a.packed[f * a.slots + p] = a.Xq[q + f * a.ldq];
            if (a.pull) a.pull[p] = a.dmean[q] * a.weights[q + j * a.ldw];
        }
        if (e == 0 && i < hi && (at < 0 || at >= a.experts)) a.place[i] = -1;
        place += __popcll(all);
    }
}

struct BlockArgs {
    fr_kprog prog;
    int64_t d;
    int experts;
    // the side a lane stands for and the side it sums over: columns of feature f at p + f * ld; expert e's rows are [begin[e], begin[e+1])
    const double *lane_x, *sum_x, *sum_v;
    int64_t lane_ld, sum_ld, lane_rows, sum_rows;
    const int64_t *lane_begin, *sum_begin;
    double* part;  // lane_rows x pieces: sum over a piece of the other side
    int64_t piece, pieces;
};

__device__ __forceinline__ int64_t row_of(const int64_t* begin, int e, int64_t rows)
{
    const int64_t v = begin[e];
    return v < 0 ? 0 : (v > rows ? rows : v);
}

template <int LEAF>
__global__ __launch_bounds__(256) void experts_block_kernel(const BlockArgs a)
{
    __shared__ int64_t items[kMaxExperts + 1];  // number of (64 lanes) x (piece) blocks in front of an expert's
    __shared__ double sums[4][kSide];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (threadIdx.x < 64) {
        int64_t total = 0;
        for (int e0 = 0; e0 < a.experts; e0 += 64) {
            const int e = e0 + lane;
            int64_t v = 0;
            if (e < a.experts) {
                const int64_t lanes = row_of(a.lane_begin, e + 1, a.lane_rows) - row_of(a.lane_begin, e, a.lane_rows);
                const int64_t rows = row_of(a.sum_begin, e + 1, a.sum_rows) - row_of(a.sum_begin, e, a.sum_rows);
                if (lanes > 0) v = ((lanes + kSide - 1) / kSide) * (rows > 0 ? (rows + a.piece - 1) / a.piece : 0);
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
    for (int64_t item = blockIdx.x; item < items[a.experts]; item += gridDim.x) {
        int lo = 0, hi = a.experts - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (items[mid] <= item)
                lo = mid;
            else
                hi = mid - 1;
        }
        const int e = lo;
        const int64_t lane0 = row_of(a.lane_begin, e, a.lane_rows), lane1 = row_of(a.lane_begin, e + 1, a.lane_rows);
        const int64_t sum0 = row_of(a.sum_begin, e, a.sum_rows), sum1 = row_of(a.sum_begin, e + 1, a.sum_rows);
        const int64_t tiles = (lane1 - lane0 + kSide - 1) / kSide;
        const int64_t piece = (item - items[e]) / tiles, tile = (item - items[e]) % tiles;
        const int64_t row = lane0 + tile * kSide + lane;
        const int64_t at = row < lane1 ? row : lane1 - 1;
        const int64_t p0 = sum0 + piece * a.piece, p1 = p0 + a.piece < sum1 ? p0 + a.piece : sum1;
        double acc = 0.0;
        for (int64_t i = p0 + wave * kStep; i < p1; i += 4 * kStep) {
            double s[kStep], u[kStep];
#pragma unroll
            for (int t = 0; t < kStep; ++t) s[t] = u[t] = 0.0;
            for (int64_t f = 0; f < a.d; ++f) {
                const double x = a.lane_x[at + f * a.lane_ld];
#pragma unroll
                for (int t = 0; t < kStep; ++t) {
                    const int64_t j = i + t < p1 ? i + t : p1 - 1;
                    const double y = a.sum_x[j + f * a.sum_ld];
                    const double z = x - y;
                    s[t] = s[t] + z * z;
                    u[t] = u[t] + x * y;
                }
            }
#pragma unroll
            for (int t = 0; t < kStep; ++t)
                if (i + t < p1) acc += kprog_eval_k<LEAF>(a.prog, s[t], u[t]) * a.sum_v[i + t];
        }
        sums[wave][lane] = acc;
        __syncthreads();
        if (wave == 0 && row < lane1) a.part[row + piece * a.lane_rows] = ((sums[0][lane] + sums[1][lane]) + sums[2][lane]) + sums[3][lane];
        __syncthreads();
    }
}

struct JoinArgs {
    int64_t m, k, slots, n, lde, ldw, lds, lddw, piece;
    int experts;
    const int* chosen;
    const int* place;
    const int64_t *begin, *starts;
    const double *part, *weights, *prior, *dmean;
    const double* slots_in;
    double *mean, *slots_out, *dweights, *dalpha;
};

// forward: a thread per query point adds up its slots' pieces
__global__ __launch_bounds__(256) void experts_mean_kernel(const JoinArgs a)
{
    const int64_t q = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (q >= a.m) return;
    double mean = a.prior ? a.prior[q] : 0.0;
    for (int64_t j = 0; j < a.k; ++j) {
        const int e = a.chosen[q + j * a.lde];
        const int64_t p = a.place[q * a.k + j];
        double v = 0.0;
        if (p >= 0) {
            const int64_t rows = row_of(a.begin, e + 1, a.n) - row_of(a.begin, e, a.n);
            for (int64_t c = 0; c * a.piece < rows; ++c) v += a.part[p + c * a.slots];
        }
        if (a.slots_out) a.slots_out[q + j * a.lds] = v;
        mean += a.weights[q + j * a.ldw] * v;
    }
    a.mean[q] = mean;
}

// backward: the gradient of each coefficient from its pieces, of each weight from its slot's mean
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
        double v = 0.0;
        if (id >= row_of(a.begin, lo, a.n) && id < row_of(a.begin, lo + 1, a.n)) {
            const int64_t rows = a.starts[lo + 1] - a.starts[lo];
            for (int64_t c = 0; c * a.piece < rows; ++c) v += a.part[id + c * a.n];
        }
        a.dalpha[id] = v;
    }
    if (a.dweights && id < a.slots) {
        const int64_t q = id % a.m, j = id / a.m;
        const int e = a.chosen[q + j * a.lde];
        a.dweights[q + j * a.lddw] = e >= 0 && e < a.experts ? a.dmean[q] * a.slots_in[q + j * a.lds] : 0.0;
    }
}

static int block_launch(fr_ctx* ctx, const BlockArgs& a, int64_t most_items)
{
    const int64_t cap = (int64_t)ctx->num_cus * 8;
    const dim3 grid((unsigned)(most_items < 1 ? 1 : (most_items < cap ? most_items : cap))), block(256);
    const int leaf = a.prog.nops == 1 ? a.prog.ops[0].kind : -1;
#define FR_EXPERTS_LEAF(KIND) \
    case KIND: hipLaunchKernelGGL((experts_block_kernel<KIND>), grid, block, 0, ctx->ls, a); break;
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
    default: hipLaunchKernelGGL((experts_block_kernel<-1>), grid, block, 0, ctx->ls, a);
    }
#undef FR_EXPERTS_LEAF
    FR_HIP(ctx, hipGetLastError());
    return FR_OK;
}

static int experts_check(fr_ctx* ctx, const fr_kprog* kernel, int64_t n, int64_t d, int64_t n_experts, int64_t m, int64_t k, const void* offsets)
{
    FR_TRY(kprog_check(ctx, kernel));
    if (n < 0 || d < 0 || m < 0) return set_err(ctx, FR_SHAPE, "negative extent (%lld points, %lld features, %lld queries)", (long long)n, (long long)d, (long long)m);
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

// Rows summed in one piece (kept from growing without bound on skewed experts): whole (no pieces to join) once the lane side alone fills the chip, otherwise cut so that there are about
// four workgroups for each CU.
static int64_t piece_rows(fr_ctx* ctx, int64_t lanes, int64_t rows, int64_t experts)
{
    const int64_t tiles = lanes / kSide + 1, each = rows / experts + 1, want = (int64_t)ctx->num_cus * 4;
    int64_t pieces = (want + tiles - 1) / tiles;
    int64_t piece = (each + pieces - 1) / pieces;
    // (the joined pieces of a lane lie `pieces` apart whatever an expert's real size: at most 256 MB of them)
    const int64_t least = lanes * (rows >> 10) >> 15;
    return round_up(piece > least ? piece : least, 4 * kStep);
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
        const int64_t piece = piece_rows(ctx, slots, n, n_experts), pieces = n / piece + 1;
        OpWorkspace ws(ctx);
        FR_TRY(ws.get((size_t)(8 * (n_experts + 1) + 8 * d * slots + 8 * pieces * slots + 4 * slots)));
        PlanArgs p = {};
        p.m = m, p.k = k, p.slots = slots, p.d = d, p.n = n, p.ldq = oq.ld, p.lde = oe.ld, p.ldw = ow.ld, p.experts = (int)n_experts;
        p.chosen = oe.as<int>(), p.Xq = oq.as<double>(), p.weights = ow.as<double>();
        p.starts = (int64_t*)ws.p;
        p.packed = (double*)(p.starts + n_experts + 1);
        double* part = p.packed + d * slots;
        p.place = (int*)(part + pieces * slots);
        hipLaunchKernelGGL(experts_plan_kernel, dim3((unsigned)n_experts), dim3(kPlanThreads), 0, ctx->ls, p);
        BlockArgs b = {};
        b.prog = *kernel, b.d = d, b.experts = (int)n_experts;
        b.lane_x = p.packed, b.lane_ld = slots, b.lane_rows = slots, b.lane_begin = p.starts;
        b.sum_x = ox.as<double>(), b.sum_ld = ox.ld, b.sum_rows = n, b.sum_begin = oo.as<int64_t>(), b.sum_v = oa.as<double>();
        b.part = part, b.piece = piece, b.pieces = pieces;
        FR_TRY(block_launch(ctx, b, (slots / kSide + n_experts) * pieces));
        JoinArgs j = {};
        j.m = m, j.k = k, j.slots = slots, j.n = n, j.lde = oe.ld, j.ldw = ow.ld, j.lds = os.ld, j.piece = piece, j.experts = (int)n_experts;
        j.chosen = p.chosen, j.place = p.place, j.begin = b.sum_begin, j.part = part, j.weights = p.weights, j.prior = op.as<double>();
        j.mean = om.as<double>(), j.slots_out = os.as<double>();
        hipLaunchKernelGGL(experts_mean_kernel, dim3((unsigned)((m + 255) / 256)), dim3(256), 0, ctx->ls, j);
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
            const int64_t piece = piece_rows(ctx, n, slots, n_experts), pieces = slots / piece + 1;
            FR_TRY(ws.get((size_t)(8 * (n_experts + 1) + 8 * (d + 1) * slots + 8 * pieces * n + 4 * slots)));
            PlanArgs p = {};
            p.m = m, p.k = k, p.slots = slots, p.d = d, p.n = n, p.ldq = oq.ld, p.lde = oe.ld, p.ldw = ow.ld, p.experts = (int)n_experts;
            p.chosen = oe.as<int>(), p.Xq = oq.as<double>(), p.weights = ow.as<double>(), p.dmean = om.as<double>();
            p.starts = (int64_t*)ws.p;
            p.packed = (double*)(p.starts + n_experts + 1);
            p.pull = p.packed + d * slots;
            double* part = p.pull + slots;
            p.place = (int*)(part + pieces * n);
            hipLaunchKernelGGL(experts_plan_kernel, dim3((unsigned)n_experts), dim3(kPlanThreads), 0, ctx->ls, p);
            BlockArgs b = {};
            b.prog = *kernel, b.d = d, b.experts = (int)n_experts;
            b.lane_x = ox.as<double>(), b.lane_ld = ox.ld, b.lane_rows = n, b.lane_begin = oo.as<int64_t>();
            b.sum_x = p.packed, b.sum_ld = slots, b.sum_rows = slots, b.sum_begin = p.starts, b.sum_v = p.pull;
            b.part = part, b.piece = piece, b.pieces = pieces;
            FR_TRY(block_launch(ctx, b, (n / kSide + n_experts) * pieces));
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
