// route.hip -- the router in front of local experts: a score for each expert, the k best of each row, their weights; and its backward pass.
//
// One wave holds a row: lane l keeps the experts l, l + 64, ... in registers.  Scores and the order of the experts are worked out in 64
// bits whatever the logits' type: which of two experts is taken must not hang on a rounding that another program would make otherwise.
#include "typed.hpp"

namespace fr {

constexpr int kRouteMaxExperts = 1024, kRouteMaxSlots = 64;

struct RouteArgs {
    int64_t n;
    int experts, k, groups, top_groups, renormalise;
    double scale;
    const void* logits;
    const double* bias;
    int* chosen;
    void* weights;
    unsigned long long* counts;
    const void* dweights;
    void* dlogits;
    int64_t l_r, l_c, e_r, e_c, w_r, w_c, dl_r, dl_c;  // element (row, column) at row * _r + column * _c
};

__device__ __forceinline__ double wave_max(double v)
{
    for (int s = 1; s < 64; s *= 2) v = fmax(v, __shfl_xor(v, s));
    return v;
}
__device__ __forceinline__ double wave_sum(double v)
{
    for (int s = 1; s < 64; s *= 2) v += __shfl_xor(v, s);
    return v;
}
// the larger key, of equal keys the lower index
__device__ __forceinline__ void wave_best(double& key, int& at)
{
    for (int s = 1; s < 64; s *= 2) {
        const double ok = __shfl_xor(key, s);
        const int oa = __shfl_xor(at, s);
        if (ok > key || (ok == key && oa < at)) {
            key = ok;
            at = oa;
        }
    }
}

// scores of a lane's experts from their logits (-inf beyond the last expert); false: the row has no answer (a NaN, or +inf under softmax)
template <int J, bool SIGMOID>
__device__ __forceinline__ bool row_scores(const double (&v)[J], double (&score)[J])
{
    double top = -INFINITY;
    bool bad = false;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        bad |= v[j] != v[j];
        top = fmax(top, v[j]);
    }
    if constexpr (SIGMOID) {
#pragma unroll
        for (int j = 0; j < J; ++j) score[j] = 1.0 / (1.0 + exp(-v[j]));
        return !__any(bad);
    } else {
        top = wave_max(top);
        if (__any(bad) || top == INFINITY) return false;
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            score[j] = top == -INFINITY ? 0.0 : exp(v[j] - top);
            sum += score[j];
        }
        sum = wave_sum(sum);
#pragma unroll
        for (int j = 0; j < J; ++j) score[j] = sum > 0.0 ? score[j] / sum : 0.0;
        return true;
    }
}

template <typename T, int J, bool SIGMOID>
__global__ __launch_bounds__(256) void route_kernel(const RouteArgs a)
{
    using W = wide_t<T>;
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= a.n) return;
    const T* logits = (const T*)a.logits + row * a.l_r;
    double v[J], score[J], key[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int e = lane + 64 * j;
        v[j] = e < a.experts ? (double)widen(logits[e * a.l_c]) : -INFINITY;
    }
    const bool good = row_scores<J, SIGMOID>(v, score);
    const double open = -INFINITY;
    if (!good) {
        if (lane < a.k) {
            a.chosen[row * a.e_r + lane * a.e_c] = -1;
            ((W*)a.weights)[row * a.w_r + lane * a.w_c] = (W)__builtin_nan("");
        }
        return;
    }
    // without a bias the logits order the experts themselves: no rounding of a score can tie two of them
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int e = lane + 64 * j;
        key[j] = v[j] == open ? open : (a.bias ? score[j] + a.bias[e] : v[j]);
    }
    if (a.top_groups < a.groups) {
        const int size = a.experts / a.groups;
        double mine = open;  // lane g: the value of group g (its two largest open scores together)
        for (int g = 0; g < a.groups; ++g) {
            double best = open, second = open;
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const int e = lane + 64 * j;
                if (v[j] == open || e / size != g) continue;
                const double m = a.bias ? key[j] : score[j];
                if (m > best) {
                    second = best;
                    best = m;
                } else if (m > second)
                    second = m;
            }
            for (int s = 1; s < 64; s *= 2) {
                const double ob = __shfl_xor(best, s), os = __shfl_xor(second, s);
                second = fmax(fmin(best, ob), fmax(second, os));
                best = fmax(best, ob);
            }
            if (lane == g) mine = second == open ? best : best + second;
        }
        unsigned long long kept = 0;
        for (int i = 0; i < a.top_groups; ++i) {
            double b = lane < a.groups && !(kept >> lane & 1) ? mine : open;
            int at = lane < a.groups && !(kept >> lane & 1) ? lane : 64 + lane;
            wave_best(b, at);
            if (at < 64) kept |= 1ull << at;
        }
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int e = lane + 64 * j;
            if (e < a.experts && !(kept >> (e / size) & 1)) key[j] = open;
        }
    }
    int mine = -1;       // lane i: the expert of slot i
    double got = 0.0;    // ... and its score
    double total = 0.0;  // of the chosen
    for (int i = 0; i < a.k; ++i) {
        double b = open;
        int at = INT32_MAX;
#pragma unroll
        for (int j = 0; j < J; ++j)
            if (key[j] > b) {
                b = key[j];
                at = lane + 64 * j;
            }
        wave_best(b, at);
        if (b == open) break;  // nothing open is left: the slots from here on stay unused
        double sc = 0.0;
#pragma unroll
        for (int j = 0; j < J; ++j)
            if (lane + 64 * j == at) {
                sc = score[j];
                key[j] = open;
            }
        sc = __shfl(sc, at & 63);
        total += sc;
        if (lane == i) {
            mine = at;
            got = sc;
        }
    }
    if (lane < a.k) {
        a.chosen[row * a.e_r + lane * a.e_c] = mine;
        const double w = a.renormalise ? (total > 0.0 ? got / total : 0.0) : got;
        ((W*)a.weights)[row * a.w_r + lane * a.w_c] = (W)(w * a.scale);
        if (a.counts && mine >= 0) atomicAdd(&a.counts[mine], 1ull);
    }
}

template <typename T, int J, bool SIGMOID>
__global__ __launch_bounds__(256) void route_backward_kernel(const RouteArgs a)
{
    using W = wide_t<T>;
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= a.n) return;
    const T* logits = (const T*)a.logits + row * a.l_r;
    double v[J], score[J], ds[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int e = lane + 64 * j;
        v[j] = e < a.experts ? (double)widen(logits[e * a.l_c]) : -INFINITY;
        ds[j] = 0.0;
    }
    const bool good = row_scores<J, SIGMOID>(v, score);
    // slot i lives in lane i: its expert, the weight's gradient, the expert's score
    int at = lane < a.k ? a.chosen[row * a.e_r + lane * a.e_c] : -1;
    if (at >= a.experts) at = -1;
    double dw = at >= 0 ? a.scale * (double)((const W*)a.dweights)[row * a.w_r + lane * a.w_c] : 0.0;
    if (a.renormalise) {
        double sc = 0.0;
        for (int i = 0; i < a.k; ++i) {
            const int e = __shfl(at, i);
            double mine = 0.0;
#pragma unroll
            for (int j = 0; j < J; ++j)
                if (lane + 64 * j == e) mine = score[j];
            mine = __shfl(mine, e & 63);
            if (lane == i && e >= 0) sc = mine;
        }
        const double total = wave_sum(sc);
        const double mean = wave_sum(total > 0.0 ? sc / total * dw : 0.0);
        dw = at >= 0 && total > 0.0 ? (dw - mean) / total : 0.0;
    }
    for (int i = 0; i < a.k; ++i) {
        const int e = __shfl(at, i);
        const double g = __shfl(dw, i);
#pragma unroll
        for (int j = 0; j < J; ++j)
            if (lane + 64 * j == e) ds[j] += g;
    }
    double mean = 0.0;
    if constexpr (!SIGMOID) {
#pragma unroll
        for (int j = 0; j < J; ++j) mean += ds[j] * score[j];
        mean = wave_sum(mean);
    }
    T* out = (T*)a.dlogits + row * a.dl_r;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int e = lane + 64 * j;
        if (e >= a.experts) continue;
        double r = SIGMOID ? ds[j] * score[j] * (1.0 - score[j]) : score[j] * (ds[j] - mean);
        if (!good) r = __builtin_nan("");
        out[e * a.dl_c] = narrow<T>((W)r);
    }
}

__global__ __launch_bounds__(256) void zero_counts_kernel(unsigned long long* p, int n)
{
    for (int i = threadIdx.x; i < n; i += 256) p[i] = 0;
}

template <typename T, int J>
static void route_launch(fr_ctx* ctx, const RouteArgs& a, bool sigmoid, bool backward)
{
    const dim3 grid((unsigned)((a.n + 3) / 4)), block(256);
    if (backward) {
        if (sigmoid)
            hipLaunchKernelGGL((route_backward_kernel<T, J, true>), grid, block, 0, ctx->ls, a);
        else
            hipLaunchKernelGGL((route_backward_kernel<T, J, false>), grid, block, 0, ctx->ls, a);
    } else if (sigmoid)
        hipLaunchKernelGGL((route_kernel<T, J, true>), grid, block, 0, ctx->ls, a);
    else
        hipLaunchKernelGGL((route_kernel<T, J, false>), grid, block, 0, ctx->ls, a);
}

template <typename T>
static int route_launch(fr_ctx* ctx, const RouteArgs& a, int score, bool backward)
{
    const bool sigmoid = score == FR_SCORE_SIGMOID;
    if (a.experts <= 64)
        route_launch<T, 1>(ctx, a, sigmoid, backward);
    else if (a.experts <= 128)
        route_launch<T, 2>(ctx, a, sigmoid, backward);
    else if (a.experts <= 256)
        route_launch<T, 4>(ctx, a, sigmoid, backward);
    else if (a.experts <= 512)
        route_launch<T, 8>(ctx, a, sigmoid, backward);
    else
        route_launch<T, 16>(ctx, a, sigmoid, backward);
    FR_HIP(ctx, hipGetLastError());
    return FR_OK;
}

static int route_dispatch(fr_ctx* ctx, const RouteArgs& a, int dtype, int score, bool backward)
{
    switch (dtype) {
    case FR_F64: return route_launch<double>(ctx, a, score, backward);
    case FR_F32: return route_launch<float>(ctx, a, score, backward);
    case FR_BF16: return route_launch<__hip_bfloat16>(ctx, a, score, backward);
    default: return route_launch<__half>(ctx, a, score, backward);
    }
}

static int route_check(fr_ctx* ctx, int dtype, int layout, int score, int64_t n, int64_t experts, int64_t k, double scale)
{
    if (dtype < FR_F64 || dtype > FR_F16) return set_err(ctx, FR_INVALID_ARGUMENT, "unknown element type %d", dtype);
    if (layout != FR_LAYOUT_COLMAJOR && layout != FR_LAYOUT_ROWMAJOR) return set_err(ctx, FR_INVALID_ARGUMENT, "layout %d: column- or row-major", layout);
    if (score != FR_SCORE_SOFTMAX && score != FR_SCORE_SIGMOID) return set_err(ctx, FR_INVALID_ARGUMENT, "unknown score %d", score);
    if (n < 0 || n > (int64_t)1 << 25) return set_err(ctx, FR_SHAPE, "%lld rows: at most 2^25 in a call", (long long)n);
    if (experts < 1 || experts > kRouteMaxExperts) return set_err(ctx, FR_SHAPE, "%lld experts: 1 to %d", (long long)experts, kRouteMaxExperts);
    if (k < 1 || k > experts || k > kRouteMaxSlots) return set_err(ctx, FR_SHAPE, "%lld slots a row: 1 to %d, and no more than %lld experts", (long long)k, kRouteMaxSlots, (long long)experts);
    if (!std::isfinite(scale)) return set_err(ctx, FR_INVALID_ARGUMENT, "scale is not finite");
    return FR_OK;
}

static void route_strides(int layout, int64_t ld, int64_t& row, int64_t& col)
{
    row = layout == FR_LAYOUT_ROWMAJOR ? ld : 1;
    col = layout == FR_LAYOUT_ROWMAJOR ? 1 : ld;
}

}  // namespace fr

using namespace fr;

extern "C" {

int fr_route(fr_ctx* ctx, int dtype, int layout, int score, int64_t n, int64_t n_experts, const void* logits, int64_t ldl, const double* bias,
             int64_t n_groups, int64_t top_groups, int64_t k, int renormalise, double scale, int* experts, int64_t lde, void* weights, int64_t ldw,
             int64_t* counts)
{
    return op_entry(ctx, [&]() -> int {
        FR_TRY(route_check(ctx, dtype, layout, score, n, n_experts, k, scale));
        if (n_groups < 1 || n_groups > 64 || n_experts % n_groups) return set_err(ctx, FR_SHAPE, "%lld groups: 1 to 64, dividing %lld experts", (long long)n_groups, (long long)n_experts);
        if (top_groups < 1 || top_groups > n_groups) return set_err(ctx, FR_SHAPE, "%lld of %lld groups", (long long)top_groups, (long long)n_groups);
        if (k > top_groups * (n_experts / n_groups)) return set_err(ctx, FR_SHAPE, "%lld slots, and %lld experts in the groups kept", (long long)k, (long long)(top_groups * (n_experts / n_groups)));
        Operand ol(ctx), ob(ctx), oe(ctx), ow(ctx), oc(ctx);
        FR_TRY(stage_matrix(ol, layout, logits, n, n_experts, ldl, dtype_size(dtype), "logits"));
        if (bias) FR_TRY(ob.stage(bias, n_experts, 1, n_experts, 8, "bias"));
        FR_TRY(stage_matrix(oe, layout, experts, n, k, lde, 4, "experts", true));
        FR_TRY(stage_matrix(ow, layout, weights, n, k, ldw, wide_size(dtype), "weights", true));
        if (counts) FR_TRY(oc.stage(counts, n_experts, 1, n_experts, 8, "counts", true));
        RouteArgs a = {};
        a.n = n, a.experts = (int)n_experts, a.k = (int)k, a.groups = (int)n_groups, a.top_groups = (int)top_groups, a.renormalise = renormalise != 0, a.scale = scale;
        a.logits = ol.dev, a.bias = ob.as<double>(), a.chosen = oe.as<int>(), a.weights = ow.dev, a.counts = oc.as<unsigned long long>();
        route_strides(layout, ol.ld, a.l_r, a.l_c);
        route_strides(layout, oe.ld, a.e_r, a.e_c);
        route_strides(layout, ow.ld, a.w_r, a.w_c);
        if (counts) hipLaunchKernelGGL(zero_counts_kernel, dim3(1), dim3(256), 0, ctx->ls, a.counts, a.experts);
        if (n > 0) FR_TRY(route_dispatch(ctx, a, dtype, score, false));
        FR_HIP(ctx, hipGetLastError());
        FR_TRY(oe.commit());
        FR_TRY(ow.commit());
        return oc.commit();
    });
}

int fr_route_backward(fr_ctx* ctx, int dtype, int layout, int score, int64_t n, int64_t n_experts, const void* logits, int64_t ldl, const void* experts,
                      int64_t lde, int64_t k, int renormalise, double scale, const void* dweights, int64_t lddw, void* dlogits, int64_t lddl)
{
    return op_entry(ctx, [&]() -> int {
        FR_TRY(route_check(ctx, dtype, layout, score, n, n_experts, k, scale));
        Operand ol(ctx), oe(ctx), ow(ctx), od(ctx);
        FR_TRY(stage_matrix(ol, layout, logits, n, n_experts, ldl, dtype_size(dtype), "logits"));
        FR_TRY(stage_matrix(oe, layout, experts, n, k, lde, 4, "experts"));
        FR_TRY(stage_matrix(ow, layout, dweights, n, k, lddw, wide_size(dtype), "dweights"));
        FR_TRY(stage_matrix(od, layout, dlogits, n, n_experts, lddl, dtype_size(dtype), "dlogits", true));
        if (n == 0) return FR_OK;
        RouteArgs a = {};
        a.n = n, a.experts = (int)n_experts, a.k = (int)k, a.renormalise = renormalise != 0, a.scale = scale;
        a.logits = ol.dev, a.chosen = oe.as<int>(), a.dweights = ow.dev, a.dlogits = od.dev;
        route_strides(layout, ol.ld, a.l_r, a.l_c);
        route_strides(layout, oe.ld, a.e_r, a.e_c);
        route_strides(layout, ow.ld, a.w_r, a.w_c);
        route_strides(layout, od.ld, a.dl_r, a.dl_c);
        FR_TRY(route_dispatch(ctx, a, dtype, score, true));
        return od.commit();
    });
}

}  // extern "C"
