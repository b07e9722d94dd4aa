// recur.hip -- the gated linear recurrence  h_t = a_t h_{t-1} + c_t x_t  over packed sequences, its backward pass, and the product with
// the covariance matrix of an Exponential kernel on ordered inputs that the two directions of it make up.
//
// The step is the affine map h -> a h + u; maps compose to maps,  (A2, H2) o (A1, H1) = (A1 A2, A2 H1 + H2),  so a stretch of rows is
// one pair (A, H) whatever its length.  A row that begins a sequence is the constant map h -> a h0 + u: A = 0 cuts what came before.
// The gradient runs the other way with the same gates: with Q_t = a_{t+1} G_{t+1} (dh_last behind a sequence's last row),
//   G_t = dh_t + Q_t,   dx_t = c_t G_t,   da_t = G_t h_{t-1},   Q_{t-1} = a_t G_t,   dh0 = Q in front of the first row.
// Three launches: every stretch of rows is reduced to its map, the maps are composed along the rows, every stretch is walked again with
// the state it starts from.  A single stretch needs the last launch only.
#include "typed.hpp"

namespace fr {

struct RecArgs {
    int64_t n, d, cols, width, nseq;  // width = d / cols channels share a gate column
    const int64_t* offsets;           // nseq + 1 row numbers, or null: one sequence of n rows
    const void *gate, *x, *h0, *hin, *dh, *dlast;
    void *h, *last, *dgate, *dx, *dh0;
    // element (t, c) of a matrix lies at t * row + c * col; one of the two is 1
    int64_t gate_r, gate_c, x_r, x_c, h_r, h_c, dh_r, dh_c, dx_r, dx_c, dg_r, dg_c;
    int64_t h0_r, h0_c, last_r, last_c, dlast_r, dlast_c, dh0_r, dh0_c;
    int64_t chunk, nchunks;
    void* maps;   // nchunks x d pairs (A, H)
    void* carry;  // nchunks x d states
    void* part;   // shared gates: n x d products before their sum over the channels of a gate
};

// first row of sequence s, kept inside [0, n] whatever the caller's offsets say
__device__ __forceinline__ int64_t seq_row(const RecArgs& a, int64_t s)
{
    if (!a.offsets) return s == 0 ? 0 : a.n;
    const int64_t v = a.offsets[s];
    return v < 0 ? 0 : (v > a.n ? a.n : v);
}

// the sequence that holds row r (the last one that begins at or before it)
__device__ __forceinline__ int64_t seq_of(const RecArgs& a, int64_t r)
{
    int64_t lo = 0, hi = a.nseq - 1;
    while (lo < hi) {
        const int64_t mid = (lo + hi + 1) >> 1;
        if (seq_row(a, mid) <= r)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ double gate_exp(double g) { return exp(g); }
__device__ __forceinline__ float gate_exp(float g) { return expf(g); }
// sqrt(1 - exp(2 g)) without the cancellation of 1 - a^2 where a is near 1
__device__ __forceinline__ double gate_rest(double g) { return sqrt(-expm1(2.0 * g)); }
__device__ __forceinline__ float gate_rest(float g) { return sqrtf(-expm1f(2.0f * g)); }

template <typename S>
struct Gate {
    S a, c;
};
template <int FORM, typename S>
__device__ __forceinline__ Gate<S> gate_of(S g)
{
    if constexpr (FORM == FR_GATE_VALUE) return {g, S(1)};
    if constexpr (FORM == FR_GATE_LOG) return {gate_exp(g), S(1)};
    return {gate_exp(g), gate_rest(g)};
}
// derivative of the row's map with respect to what the caller stores: G h_{t-1} da/dg + G x dc/dg
template <int FORM, typename S>
__device__ __forceinline__ S gate_grad(const Gate<S>& g, S G, S before, S x)
{
    if constexpr (FORM == FR_GATE_VALUE) return G * before;
    if constexpr (FORM == FR_GATE_LOG) return G * before * g.a;
    // c^2 = 1 - e^{2g}: dc/dg = -a^2 / c; a gate of exactly 1 (c = 0) has no finite slope there: taken as 0
    return g.a * (G * before - (g.c > S(0) ? G * x * g.a / g.c : S(0)));
}


// ---- stretches of rows: one thread per (stretch, channel) -------------------------------------------------------------------------

template <typename T, int FORM, bool REDUCE>
__global__ __launch_bounds__(256) void rec_forward_kernel(const RecArgs a)
{
    using S = wide_t<T>;
    const int64_t id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    const int64_t k = id / a.d, c = id - k * a.d;
    if (k >= a.nchunks) return;
    const T* gate = (const T*)a.gate + (c / a.width) * a.gate_c;
    const T* x = (const T*)a.x + c * a.x_c;
    const S* h0 = (const S*)a.h0 + c * a.h0_c;
    T* out = (T*)a.h + c * a.h_c;
    S* last = (S*)a.last + c * a.last_c;
    const int64_t lo = seq_row(a, 0), hi = seq_row(a, a.nseq);
    const int64_t begin = k * a.chunk > lo ? k * a.chunk : lo;
    const int64_t end = (k + 1) * a.chunk < hi ? (k + 1) * a.chunk : hi;
    S A = S(1), h = S(0);
    if (!REDUCE && a.nchunks > 1) h = ((const S*)a.carry)[id];
    if (begin < end) {
        int64_t s = seq_of(a, begin);
        int64_t first = seq_row(a, s), next = seq_row(a, s + 1);
        for (int64_t r = begin; r < end; ++r) {
            if (r == first) {
                h = a.h0 ? h0[s * a.h0_r] : S(0);
                A = S(0);
            }
            const Gate<S> g = gate_of<FORM, S>(widen(gate[r * a.gate_r]));
            S u = widen(x[r * a.x_r]);
            if constexpr (FORM == FR_GATE_STATIONARY) u *= g.c;
            h = g.a * h + u;
            A *= g.a;
            if constexpr (!REDUCE) out[r * a.h_r] = narrow<T>(h);
            if (r + 1 == next) {
                if constexpr (!REDUCE)
                    if (a.last) last[s * a.last_r] = h;
                s = seq_of(a, next);
                first = next;
                next = seq_row(a, s + 1);
            }
        }
    }
    if constexpr (REDUCE) {
        ((S*)a.maps)[2 * id] = A;
        ((S*)a.maps)[2 * id + 1] = h;
    } else if (a.last) {
        for (int64_t s = k; s < a.nseq; s += a.nchunks)  // sequences without rows end in the state they began with
            if (seq_row(a, s + 1) <= seq_row(a, s)) last[s * a.last_r] = a.h0 ? h0[s * a.h0_r] : S(0);
    }
}

// Stretches are counted from the last row, so that the composition of the maps runs in the same direction as forward.
template <typename T, int FORM, bool REDUCE>
__global__ __launch_bounds__(256) void rec_backward_kernel(const RecArgs a)
{
    using S = wide_t<T>;
    const int64_t id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    const int64_t kk = id / a.d, c = id - kk * a.d;
    if (kk >= a.nchunks) return;
    const int64_t k = a.nchunks - 1 - kk;
    const T* gate = (const T*)a.gate + (c / a.width) * a.gate_c;
    const T* x = (const T*)a.x + c * a.x_c;
    const T* hin = (const T*)a.hin + c * a.h_c;
    const T* dh = (const T*)a.dh + c * a.dh_c;
    const S* h0 = (const S*)a.h0 + c * a.h0_c;
    const S* dlast = (const S*)a.dlast + c * a.dlast_c;
    S* dh0 = (S*)a.dh0 + c * a.dh0_c;
    const int64_t lo = seq_row(a, 0), hi = seq_row(a, a.nseq);
    const int64_t begin = k * a.chunk > lo ? k * a.chunk : lo;
    const int64_t end = (k + 1) * a.chunk < hi ? (k + 1) * a.chunk : hi;
    S A = S(1), Q = S(0);
    if (!REDUCE && a.nchunks > 1) Q = ((const S*)a.carry)[id];
    if (begin < end) {
        int64_t s = seq_of(a, end - 1);
        int64_t first = seq_row(a, s), next = seq_row(a, s + 1);
        for (int64_t r = end - 1; r >= begin; --r) {
            if (r + 1 == next) {
                Q = a.dlast ? dlast[s * a.dlast_r] : S(0);
                A = S(0);
            }
            const Gate<S> g = gate_of<FORM, S>(widen(gate[r * a.gate_r]));
            const S G = widen(dh[r * a.dh_r]) + Q;
            if constexpr (!REDUCE) {
                if (a.dx) ((T*)a.dx)[r * a.dx_r + c * a.dx_c] = narrow<T>(FORM == FR_GATE_STATIONARY ? g.c * G : G);
                if (a.dgate) {
                    const S before = r > first ? widen(hin[(r - 1) * a.h_r]) : (a.h0 ? h0[s * a.h0_r] : S(0));
                    const S v = gate_grad<FORM, S>(g, G, before, FORM == FR_GATE_STATIONARY ? widen(x[r * a.x_r]) : S(0));
                    if (a.width == 1)
                        ((T*)a.dgate)[r * a.dg_r + c * a.dg_c] = narrow<T>(v);
                    else
                        ((S*)a.part)[r * a.d + c] = v;
                }
            }
            Q = g.a * G;
            A *= g.a;
            if (r == first) {
                if constexpr (!REDUCE)
                    if (a.dh0) dh0[s * a.dh0_r] = Q;
                if (r > lo) {
                    s = seq_of(a, r - 1);
                    next = r;
                    first = seq_row(a, s);
                }
            }
        }
    }
    if constexpr (REDUCE) {
        ((S*)a.maps)[2 * id] = A;
        ((S*)a.maps)[2 * id + 1] = Q;
    } else if (a.dh0) {
        for (int64_t s = k; s < a.nseq; s += a.nchunks)
            if (seq_row(a, s + 1) <= seq_row(a, s)) dh0[s * a.dh0_r] = a.dlast ? dlast[s * a.dlast_r] : S(0);
    }
}

// state in front of each stretch: the maps of the stretches before it, composed in order (a wave per channel, 64 stretches at a time)
template <typename S>
__global__ __launch_bounds__(64) void rec_carry_kernel(const S* __restrict__ maps, S* __restrict__ carry, int64_t d, int64_t nchunks)
{
    const int64_t c = blockIdx.x;
    const int lane = threadIdx.x;
    S state = S(0);
    for (int64_t k0 = 0; k0 < nchunks; k0 += 64) {
        const int64_t k = k0 + lane;
        S A = S(1), H = S(0);
        if (k < nchunks) {
            A = maps[2 * (k * d + c)];
            H = maps[2 * (k * d + c) + 1];
        }
        for (int step = 1; step < 64; step *= 2) {
            const S pa = __shfl_up(A, step), ph = __shfl_up(H, step);
            if (lane >= step) {
                H = A * ph + H;
                A = pa * A;
            }
        }
        const S after = A * state + H;
        const S before = __shfl_up(after, 1);
        if (k < nchunks) carry[k * d + c] = lane ? before : state;
        state = __shfl(after, 63);
    }
}

// dgate of a shared gate: the sum over the channels that share it, in the order of the channels
template <typename T>
__global__ __launch_bounds__(256) void rec_heads_kernel(const RecArgs a)
{
    using S = wide_t<T>;
    const int64_t lo = seq_row(a, 0), hi = seq_row(a, a.nseq), step = (int64_t)gridDim.x * blockDim.x;
    for (int64_t id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; id < a.n * a.cols; id += step) {
        const int64_t r = id / a.cols, q = id - r * a.cols;
        if (r < lo || r >= hi) continue;
        const S* p = (const S*)a.part + r * a.d + q * a.width;
        S sum = S(0);
        for (int64_t i = 0; i < a.width; ++i) sum += p[i];
        ((T*)a.dgate)[r * a.dg_r + q * a.dg_c] = narrow<T>(sum);
    }
}

// ---- the product with an Exponential kernel's covariance matrix on ordered inputs -----------------------------------------------

// log a_i = -(t_i - t_{i-1}) / (2 ls^2)  (kernel.rs:661-665 between neighbours); inputs out of order have no such product: NaN
__global__ __launch_bounds__(256) void markov_gate_kernel(const double* __restrict__ t, int64_t n, double ls2, double* __restrict__ g)
{
    const int64_t step = (int64_t)gridDim.x * blockDim.x;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += step) {
        const double dt = i ? t[i] - t[i - 1] : 0.0;
        g[i] = dt >= 0.0 ? -dt / ls2 : __builtin_nan("");
    }
}

// out = ampl (f + b - v) + noise^2 v: row i is counted in the sum from the left and in the one from the right
__global__ __launch_bounds__(256) void markov_join_kernel(const double* __restrict__ f, const double* __restrict__ v, int64_t ldv, double* __restrict__ out,
                                                          int64_t ldo, int64_t n, int64_t m, double ampl, double noise2)
{
    const int64_t step = (int64_t)gridDim.x * blockDim.x;
    for (int64_t id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; id < n * m; id += step) {
        const int64_t c = id / n, r = id - c * n;
        const double w = v[r + c * ldv], b = out[r + c * ldo];
        out[r + c * ldo] = ampl * (f[id] + (b - w)) + noise2 * w;
    }
}

// ---- host side ----------------------------------------------------------------------------------------------------------------------

static unsigned blocks_of(int64_t threads) { return (unsigned)((threads + 255) / 256); }
// ... of a kernel that strides over its grid
static unsigned blocks_upto(int64_t threads)
{
    const int64_t b = (threads + 255) / 256;
    return (unsigned)(b < 16384 ? b : 16384);
}

template <typename T, int FORM>
static int rec_launch(fr_ctx* ctx, RecArgs& a, bool backward, OpWorkspace& ws)
{
    using S = wide_t<T>;
    // enough stretches to give every SIMD a few waves, none shorter than 16 rows
    const int64_t want = (262144 + a.d - 1) / a.d;
    int64_t nchunks = a.n / 16;
    if (nchunks > want) nchunks = want;
    if (nchunks > 8192) nchunks = 8192;
    if (nchunks < 1) nchunks = 1;
    a.chunk = (a.n + nchunks - 1) / nchunks;
    a.nchunks = a.n > 0 ? (a.n + a.chunk - 1) / a.chunk : 1;
    if (a.n == 0) a.chunk = 1;
    const bool parts = backward && a.dgate && a.width > 1;
    const int64_t maps = a.nchunks > 1 ? 3 * a.nchunks * a.d : 0;
    const int64_t need = (maps + (parts ? a.n * a.d : 0)) * (int64_t)sizeof(S);
    if (need) FR_TRY(ws.get((size_t)need));
    a.maps = ws.p;
    a.carry = (S*)ws.p + 2 * a.nchunks * a.d;
    a.part = (S*)ws.p + maps;
    const dim3 grid(blocks_of(a.nchunks * a.d)), block(256);
    if (a.nchunks > 1) {
        if (backward)
            hipLaunchKernelGGL((rec_backward_kernel<T, FORM, true>), grid, block, 0, ctx->ls, a);
        else
            hipLaunchKernelGGL((rec_forward_kernel<T, FORM, true>), grid, block, 0, ctx->ls, a);
        hipLaunchKernelGGL((rec_carry_kernel<S>), dim3((unsigned)a.d), dim3(64), 0, ctx->ls, (const S*)a.maps, (S*)a.carry, a.d, a.nchunks);
    }
    if (backward)
        hipLaunchKernelGGL((rec_backward_kernel<T, FORM, false>), grid, block, 0, ctx->ls, a);
    else
        hipLaunchKernelGGL((rec_forward_kernel<T, FORM, false>), grid, block, 0, ctx->ls, a);
    if (parts && a.n > 0) hipLaunchKernelGGL((rec_heads_kernel<T>), dim3(blocks_upto(a.n * a.cols)), block, 0, ctx->ls, a);
    FR_HIP(ctx, hipGetLastError());
    return FR_OK;
}

template <typename T>
static int rec_launch(fr_ctx* ctx, RecArgs& a, int form, bool backward, OpWorkspace& ws)
{
    switch (form) {
    case FR_GATE_VALUE: return rec_launch<T, FR_GATE_VALUE>(ctx, a, backward, ws);
    case FR_GATE_LOG: return rec_launch<T, FR_GATE_LOG>(ctx, a, backward, ws);
    default: return rec_launch<T, FR_GATE_STATIONARY>(ctx, a, backward, ws);
    }
}

static int rec_dispatch(fr_ctx* ctx, RecArgs& a, int dtype, int form, bool backward)
{
    OpWorkspace ws(ctx);
    switch (dtype) {
    case FR_F64: return rec_launch<double>(ctx, a, form, backward, ws);
    case FR_F32: return rec_launch<float>(ctx, a, form, backward, ws);
    case FR_BF16: return rec_launch<__hip_bfloat16>(ctx, a, form, backward, ws);
    default: return rec_launch<__half>(ctx, a, form, backward, ws);
    }
}

static int rec_check(fr_ctx* ctx, int dtype, int layout, int form, int64_t n, int64_t d, int64_t gate_cols, const void* offsets, int64_t nseq)
{
    if (dtype < FR_F64 || dtype > FR_F16) return set_err(ctx, FR_INVALID_ARGUMENT, "unknown element type %d", dtype);
    if (layout != FR_LAYOUT_COLMAJOR && layout != FR_LAYOUT_ROWMAJOR) return set_err(ctx, FR_INVALID_ARGUMENT, "layout %d: column- or row-major", layout);
    if (form < FR_GATE_VALUE || form > FR_GATE_STATIONARY) return set_err(ctx, FR_INVALID_ARGUMENT, "unknown gate form %d", form);
    if (n < 0 || d < 0 || nseq < 0) return set_err(ctx, FR_SHAPE, "negative extent (%lld rows, %lld channels, %lld sequences)", (long long)n, (long long)d, (long long)nseq);
    if (d > 0 && (gate_cols < 1 || d % gate_cols)) return set_err(ctx, FR_SHAPE, "%lld gate columns do not divide %lld channels", (long long)gate_cols, (long long)d);
    if (!offsets && nseq != 1) return set_err(ctx, FR_INVALID_ARGUMENT, "%lld sequences without their offsets", (long long)nseq);
    // (the grids below count in 32 bits)
    if (d > (int64_t)1 << 24 || nseq > (int64_t)1 << 30 || n > (int64_t)1 << 40) return set_err(ctx, FR_SHAPE, "more than 2^24 channels, 2^30 sequences or 2^40 rows");
    return FR_OK;
}

// offsets that the host can see are checked here; those in device memory the kernels keep inside [0, n]
static int rec_offsets(fr_ctx* ctx, Operand& o, const void* offsets, int64_t nseq, int64_t n)
{
    if (!offsets) return FR_OK;
    FR_TRY(o.stage(offsets, nseq + 1, 1, nseq + 1, 8, "offsets"));
    if ((const void*)o.dev == offsets) return FR_OK;
    const int64_t* v = (const int64_t*)offsets;
    for (int64_t s = 0; s <= nseq; ++s)
        if (v[s] < (s ? v[s - 1] : 0) || v[s] > n) return set_err(ctx, FR_SHAPE, "offsets[%lld] = %lld: not in order within [0, %lld]", (long long)s, (long long)v[s], (long long)n);
    return FR_OK;
}

static void rec_strides(int layout, int64_t ld, int64_t& row, int64_t& col)
{
    row = layout == FR_LAYOUT_ROWMAJOR ? ld : 1;
    col = layout == FR_LAYOUT_ROWMAJOR ? 1 : ld;
}

}  // namespace fr

using namespace fr;

extern "C" {

int fr_recurrence(fr_ctx* ctx, int dtype, int layout, int form, int64_t n, int64_t d, const void* gate, int64_t gate_cols, int64_t ldg, const void* x,
                  int64_t ldx, const void* offsets, int64_t nseq, const void* h0, int64_t ldh0, void* h, int64_t ldh, void* h_last, int64_t ldl)
{
    return op_entry(ctx, [&]() -> int {
        FR_TRY(rec_check(ctx, dtype, layout, form, n, d, gate_cols, offsets, nseq));
        if (d == 0 || nseq == 0) return FR_OK;
        const int64_t e = dtype_size(dtype), w = wide_size(dtype);
        Operand o(ctx), og(ctx), ox(ctx), oh0(ctx), oh(ctx), ol(ctx);
        FR_TRY(rec_offsets(ctx, o, offsets, nseq, n));
        FR_TRY(stage_matrix(og, layout, gate, n, gate_cols, ldg, e, "gate"));
        FR_TRY(stage_matrix(ox, layout, x, n, d, ldx, e, "x"));
        if (h0) FR_TRY(stage_matrix(oh0, layout, h0, nseq, d, ldh0, w, "h0"));
        FR_TRY(stage_matrix(oh, layout, h, n, d, ldh, e, "h", true));
        if (h_last) FR_TRY(stage_matrix(ol, layout, h_last, nseq, d, ldl, w, "h_last", true));
        RecArgs a = {};
        a.n = n, a.d = d, a.cols = gate_cols, a.width = d / gate_cols, a.nseq = nseq;
        a.offsets = o.as<int64_t>(), a.gate = og.dev, a.x = ox.dev, a.h0 = oh0.dev, a.h = oh.dev, a.last = ol.dev;
        rec_strides(layout, og.ld, a.gate_r, a.gate_c);
        rec_strides(layout, ox.ld, a.x_r, a.x_c);
        rec_strides(layout, oh0.ld, a.h0_r, a.h0_c);
        rec_strides(layout, oh.ld, a.h_r, a.h_c);
        rec_strides(layout, ol.ld, a.last_r, a.last_c);
        FR_TRY(rec_dispatch(ctx, a, dtype, form, false));
        FR_TRY(oh.commit());
        return ol.commit();
    });
}

int fr_recurrence_backward(fr_ctx* ctx, int dtype, int layout, int form, int64_t n, int64_t d, const void* gate, int64_t gate_cols, int64_t ldg,
                           const void* x, int64_t ldx, const void* offsets, int64_t nseq, const void* h0, int64_t ldh0, const void* h, int64_t ldh,
                           const void* dh, int64_t lddh, const void* dh_last, int64_t lddl, void* dgate, int64_t lddg, void* dx, int64_t lddx, void* dh0,
                           int64_t lddh0)
{
    return op_entry(ctx, [&]() -> int {
        FR_TRY(rec_check(ctx, dtype, layout, form, n, d, gate_cols, offsets, nseq));
        if (d == 0 || nseq == 0 || !(dgate || dx || dh0)) return FR_OK;
        const int64_t e = dtype_size(dtype), w = wide_size(dtype);
        Operand o(ctx), og(ctx), ox(ctx), oh0(ctx), oh(ctx), odh(ctx), odl(ctx), odg(ctx), odx(ctx), odh0(ctx);
        FR_TRY(rec_offsets(ctx, o, offsets, nseq, n));
        FR_TRY(stage_matrix(og, layout, gate, n, gate_cols, ldg, e, "gate"));
        if (dgate && form == FR_GATE_STATIONARY) FR_TRY(stage_matrix(ox, layout, x, n, d, ldx, e, "x"));
        if (h0) FR_TRY(stage_matrix(oh0, layout, h0, nseq, d, ldh0, w, "h0"));
        if (dgate) FR_TRY(stage_matrix(oh, layout, h, n, d, ldh, e, "h"));
        FR_TRY(stage_matrix(odh, layout, dh, n, d, lddh, e, "dh"));
        if (dh_last) FR_TRY(stage_matrix(odl, layout, dh_last, nseq, d, lddl, w, "dh_last"));
        if (dgate) FR_TRY(stage_matrix(odg, layout, dgate, n, gate_cols, lddg, e, "dgate", true));
        if (dx) FR_TRY(stage_matrix(odx, layout, dx, n, d, lddx, e, "dx", true));
        if (dh0) FR_TRY(stage_matrix(odh0, layout, dh0, nseq, d, lddh0, w, "dh0", true));
        RecArgs a = {};
        a.n = n, a.d = d, a.cols = gate_cols, a.width = d / gate_cols, a.nseq = nseq;
        a.offsets = o.as<int64_t>(), a.gate = og.dev, a.x = ox.dev, a.h0 = oh0.dev, a.hin = oh.dev, a.dh = odh.dev, a.dlast = odl.dev;
        a.dgate = odg.dev, a.dx = odx.dev, a.dh0 = odh0.dev;
        rec_strides(layout, og.ld, a.gate_r, a.gate_c);
        rec_strides(layout, ox.ld, a.x_r, a.x_c);
        rec_strides(layout, oh0.ld, a.h0_r, a.h0_c);
        rec_strides(layout, oh.ld, a.h_r, a.h_c);
        rec_strides(layout, odh.ld, a.dh_r, a.dh_c);
        rec_strides(layout, odl.ld, a.dlast_r, a.dlast_c);
        rec_strides(layout, odg.ld, a.dg_r, a.dg_c);
        rec_strides(layout, odx.ld, a.dx_r, a.dx_c);
        rec_strides(layout, odh0.ld, a.dh0_r, a.dh0_c);
        FR_TRY(rec_dispatch(ctx, a, dtype, form, true));
        FR_TRY(odg.commit());
        FR_TRY(odx.commit());
        return odh0.commit();
    });
}

int fr_markov_product(fr_ctx* ctx, const fr_kprog* kernel, const double* t, int64_t n, const double* V, int64_t m, int64_t ldv, double noise, double* out,
                      int64_t ldo)
{
    return op_entry(ctx, [&]() -> int {
        FR_TRY(kprog_check(ctx, kernel));
        if (kernel->nops != 1 || kernel->ops[0].kind != FR_K_EXPONENTIAL)
            return set_err(ctx, FR_UNSUPPORTED_KERNEL, "only a single Exponential kernel is Markov on ordered inputs");
        FR_TRY(rec_check(ctx, FR_F64, FR_LAYOUT_COLMAJOR, FR_GATE_LOG, n, m, 1, nullptr, 1));
        Operand ot(ctx), ov(ctx), oo(ctx);
        FR_TRY(ot.stage(t, n, 1, n, 8, "t"));
        FR_TRY(ov.stage(V, n, m, ldv, 8, "V"));
        FR_TRY(oo.stage(out, n, m, ldo, 8, "out", true));
        if ((const void*)ot.dev != t)
            for (int64_t i = 1; i < n; ++i)
                if (!(t[i] >= t[i - 1])) return set_err(ctx, FR_INVALID_ARGUMENT, "t[%lld] lies before the input in front of it", (long long)i);
        if (n == 0 || m == 0) return FR_OK;
        const double ls = kernel->ops[0].params[0], ampl = std::fabs(kernel->ops[0].params[1]);
        OpWorkspace ws(ctx);
        FR_TRY(ws.get(sizeof(double) * (size_t)(n + n * m)));
        double *g = (double*)ws.p, *f = g + n;
        hipLaunchKernelGGL(markov_gate_kernel, dim3(blocks_upto(n)), dim3(256), 0, ctx->ls, ot.as<double>(), n, 2.0 * ls * ls, g);
        RecArgs a = {};
        a.n = n, a.d = m, a.cols = 1, a.width = m, a.nseq = 1;
        a.gate = g, a.x = ov.dev, a.h = f;
        rec_strides(FR_LAYOUT_COLMAJOR, n, a.gate_r, a.gate_c);
        rec_strides(FR_LAYOUT_COLMAJOR, ov.ld, a.x_r, a.x_c);
        rec_strides(FR_LAYOUT_COLMAJOR, n, a.h_r, a.h_c);
        FR_TRY(rec_dispatch(ctx, a, FR_F64, FR_GATE_LOG, false));
        RecArgs b = {};
        b.n = n, b.d = m, b.cols = 1, b.width = m, b.nseq = 1;
        b.gate = g, b.dh = ov.dev, b.dx = oo.dev;
        b.gate_r = a.gate_r, b.gate_c = a.gate_c, b.dh_r = a.x_r, b.dh_c = a.x_c;
        rec_strides(FR_LAYOUT_COLMAJOR, oo.ld, b.dx_r, b.dx_c);
        FR_TRY(rec_dispatch(ctx, b, FR_F64, FR_GATE_LOG, true));
        hipLaunchKernelGGL(markov_join_kernel, dim3(blocks_upto(n * m)), dim3(256), 0, ctx->ls, (const double*)f, (const double*)ov.dev, ov.ld, oo.as<double>(), oo.ld, n,
                           m, ampl, noise * noise);
        FR_HIP(ctx, hipGetLastError());
        return oo.commit();
    });
}

}  // extern "C"
