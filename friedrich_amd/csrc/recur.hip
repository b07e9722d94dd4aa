// recur.hip -- entry points of the gated linear recurrence (kernels: recur.hpp), and the product with the covariance matrix of an
// Exponential kernel on ordered inputs that its two directions make up.
#include "recur.hpp"

namespace fr {

extern template int rec_run<double>(fr_ctx*, RecArgs&, int, int, bool, OpWorkspace&);
extern template int rec_run<float>(fr_ctx*, RecArgs&, int, int, bool, OpWorkspace&);
extern template int rec_run<__hip_bfloat16>(fr_ctx*, RecArgs&, int, int, bool, OpWorkspace&);
extern template int rec_run<__half>(fr_ctx*, RecArgs&, int, int, bool, OpWorkspace&);

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

static int rec_dispatch(fr_ctx* ctx, RecArgs& a, int dtype, int layout, int form, bool backward)
{
    OpWorkspace ws(ctx);
    switch (dtype) {
    case FR_F64: return rec_run<double>(ctx, a, layout, form, backward, ws);
    case FR_F32: return rec_run<float>(ctx, a, layout, form, backward, ws);
    case FR_BF16: return rec_run<__hip_bfloat16>(ctx, a, layout, form, backward, ws);
    default: return rec_run<__half>(ctx, a, layout, form, backward, ws);
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
        // (a tile reads the states that its sequences enter with twice; another may have written those that they leave with in between)
        if (h_last && h_last == h0) return set_err(ctx, FR_INVALID_ARGUMENT, "h_last: the same memory as h0");
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
        FR_TRY(rec_dispatch(ctx, a, dtype, layout, form, false));
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
        if (dh0 && dh0 == dh_last) return set_err(ctx, FR_INVALID_ARGUMENT, "dh0: the same memory as dh_last");  // (as h_last and h0)
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
        FR_TRY(rec_dispatch(ctx, a, dtype, layout, form, true));
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
        if (out == V) return set_err(ctx, FR_INVALID_ARGUMENT, "out: the same memory as V");  // (V is read again when out is joined)
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
        FR_TRY(rec_dispatch(ctx, a, FR_F64, FR_LAYOUT_COLMAJOR, FR_GATE_LOG, false));
        RecArgs b = {};
        b.n = n, b.d = m, b.cols = 1, b.width = m, b.nseq = 1;
        b.gate = g, b.dh = ov.dev, b.dx = oo.dev;
        b.gate_r = a.gate_r, b.gate_c = a.gate_c, b.dh_r = a.x_r, b.dh_c = a.x_c;
        rec_strides(FR_LAYOUT_COLMAJOR, oo.ld, b.dx_r, b.dx_c);
        FR_TRY(rec_dispatch(ctx, b, FR_F64, FR_LAYOUT_COLMAJOR, FR_GATE_LOG, true));
        hipLaunchKernelGGL(markov_join_kernel, dim3(blocks_upto(n * m)), dim3(256), 0, ctx->ls, (const double*)f, (const double*)ov.dev, ov.ld, oo.as<double>(), oo.ld, n,
                           m, ampl, noise * noise);
        FR_HIP(ctx, hipGetLastError());
        return oo.commit();
    });
}

}  // extern "C"
