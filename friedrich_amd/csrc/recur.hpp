// recur.hpp -- kernels of the gated linear recurrence  h_t = a_t h_{t-1} + c_t x_t  over packed sequences and of its backward pass (one
// translation unit for each element type includes them; the entry points are in recur.hip).
//
// The step is the affine map h -> a h + u; maps compose to maps,  (A2, H2) o (A1, H1) = (A1 A2, A2 H1 + H2),  so a stretch of rows is
// one pair (A, H) whatever its length.  A row that begins a sequence is the constant map h -> a h0 + u: A = 0 cuts what came before.
// The gradient runs the other way with the same gates: with Q_t = a_{t+1} G_{t+1} (dh_last behind a sequence's last row),
//   G_t = dh_t + Q_t,   dx_t = c_t G_t,   da_t = G_t h_{t-1},   Q_{t-1} = a_t G_t,   dh0 = Q in front of the first row.
// One launch walks everything: a workgroup holds a tile of rows in registers, publishes the tile's map, takes the state in front of the
// tile from the maps published before it, and writes.
#pragma once

#include <type_traits>

#include "typed.hpp"

namespace fr {

// workgroups of 256 threads of a kernel that strides over its grid
inline unsigned blocks_upto(int64_t threads)
{
    const int64_t b = (threads + 255) / 256;
    return (unsigned)(b < 16384 ? b : 16384);
}

struct RecArgs {
    int64_t n, d, cols, width, nseq;  // width = d / cols channels share a gate column
    const int64_t* offsets;           // nseq + 1 row numbers, or null: one sequence of n rows
    const void *gate, *x, *h0, *hin, *dh, *dlast;
    void *h, *last, *dgate, *dx, *dh0;
    // element (t, c) of a matrix lies at t * row + c * col; one of the two is 1
    int64_t gate_r, gate_c, x_r, x_c, h_r, h_c, dh_r, dh_c, dx_r, dx_c, dg_r, dg_c;
    int64_t h0_r, h0_c, last_r, last_c, dlast_r, dlast_c, dh0_r, dh0_c;
    int64_t stretches, tiles;  // runs of rows that one lane walks; workgroups along the rows
    int64_t blocks, pieces;    // workgroups across the channels; parts that a shared gate's gradient is summed from
    int lanes;                 // rows layout: log2 of the lanes side by side across the channels
    int sum_lanes;             // ... lanes whose channels share a gate (0: every channel stores its part)
    int64_t part_r, part_c;
    void *ticket, *maps, *carry, *part;
    unsigned* lost;  // host-visible: not 0 after a wait that ran out
    int polls;       // looks that a wait takes before it does
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

// exp(g) and 1 - exp(g) from one polynomial: g = n ln 2 + r with |r| <= 0.3466 (ln 2 in two parts, after Cody and Waite, two fused steps), q = exp(r) - 1 by its Taylor series
// (remainder 0.3466^14 / 14! = 4e-18 in f64, 0.3466^8 / 8! = 5e-9 in f32), exp(g) = 2^n (1 + q).  For n = 0, where 1 - exp(g) would cancel, it
// is -q itself; elsewhere exp(g) is at most 0.71 or at least 1.41 and the difference is exact to a rounding or two.  Against exp, expm1 and
// sqrt of the library (about 100 instructions in f64) this is about 45.
template <typename S>
struct Exponential {
    S a, rest;
};
__device__ __forceinline__ Exponential<double> exponential(double g)
{
    const double n = __builtin_rint(g * 1.44269504088896338700e+00);
    double r = __builtin_fma(n, -6.93147180369123816490e-01, g);
    r = __builtin_fma(n, -1.90821492927058770002e-10, r);
    double p = 1.60590438368216145994e-10;                // 1 / 13!
    p = __builtin_fma(p, r, 2.08767569878680989792e-09);  // 1 / 12!
    p = __builtin_fma(p, r, 2.50521083854417187751e-08);
    p = __builtin_fma(p, r, 2.75573192239858906526e-07);
    p = __builtin_fma(p, r, 2.75573192239858906526e-06);
    p = __builtin_fma(p, r, 2.48015873015873015873e-05);
    p = __builtin_fma(p, r, 1.98412698412698412698e-04);
    p = __builtin_fma(p, r, 1.38888888888888888889e-03);
    p = __builtin_fma(p, r, 8.33333333333333333333e-03);
    p = __builtin_fma(p, r, 4.16666666666666666667e-02);
    p = __builtin_fma(p, r, 1.66666666666666666667e-01);
    p = __builtin_fma(p, r, 0.5);
    const double q = __builtin_fma(p * r, r, r);
    double a = __builtin_ldexp(1.0 + q, (int)n);
    a = g < -746.0 ? 0.0 : (g > 710.0 ? __builtin_inf() : a);  // (NaN falls through: r is NaN)
    return {a, n == 0.0 ? -q : 1.0 - a};
}
__device__ __forceinline__ Exponential<float> exponential(float g)
{
    const float n = __builtin_rintf(g * 1.44269502f);
    float r = __builtin_fmaf(n, -6.93145752e-01f, g);
    r = __builtin_fmaf(n, -1.42860677e-06f, r);
    float p = 1.98412701e-04f;  // 1 / 7!
    p = __builtin_fmaf(p, r, 1.38888892e-03f);
    p = __builtin_fmaf(p, r, 8.33333377e-03f);
    p = __builtin_fmaf(p, r, 4.16666679e-02f);
    p = __builtin_fmaf(p, r, 1.66666672e-01f);
    p = __builtin_fmaf(p, r, 0.5f);
    const float q = __builtin_fmaf(p * r, r, r);
    float a = __builtin_ldexpf(1.0f + q, (int)n);
    a = g < -104.0f ? 0.0f : (g > 89.0f ? __builtin_inff() : a);
    return {a, n == 0.0f ? -q : 1.0f - a};
}
__device__ __forceinline__ double root(double v) { return sqrt(v); }
__device__ __forceinline__ float root(float v) { return sqrtf(v); }

template <typename S>
struct Gate {
    S a, c;
};
template <int FORM, typename S>
__device__ __forceinline__ Gate<S> gate_of(S g)
{
    if constexpr (FORM == FR_GATE_VALUE) return {g, S(1)};
    const Exponential<S> e = exponential(g);
    if constexpr (FORM == FR_GATE_LOG) return {e.a, S(1)};
    return {e.a, root(e.rest * (S(1) + e.a))};  // sqrt(1 - a^2) without the cancellation where a is near 1
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

// ---- what stands in front of a tile ---------------------------------------------------------------------------------------------------
//
// Every tile publishes its map as soon as it has read its rows; the state in front of a tile is the state behind the last whole block of
// tiles (the last tile of a block publishes it) followed by the maps of the block's tiles before it, always in that order: the same
// bits on every run, whichever tile comes first.  A word is 64 bits and says by itself whether it has been written: all ones, which the
// workspace is filled with, is a NaN that no result is published as.  So a word needs no flag and no fence beside it.  A tile waits for tiles
// of lower tickets only, and tickets are drawn by running workgroups: the wait ends, whatever else holds the chip.

// in the place of A: the map ignores what stands in front (NaN patterns that no computed A is published as)
constexpr unsigned long long kCut = 0x7ff8c07c07c07c07ull;
constexpr unsigned kCut32 = 0x7fc0c07cu;

constexpr int kRowsWindow = 16;    // tiles in a block, rows layout: a lane reads the words of its own channel, so few of them
constexpr int kColumnsWindow = 64;  // ... columns layout: one for each lane of a wave
constexpr int kRowsOfLane = 8;      // columns layout: rows of a lane
constexpr int kWaves = 8;           // of a workgroup, at most
constexpr int64_t kFewRows = 1024;  // rows layout, forward: up to here 4 rows a lane
// rows layout: rows of a lane; fewer where the data, a gate for each channel, a second factor of a row or the backward pass's second operand take
// the registers (backward, bf16, 16413 x 2048: 83 us with 16 rows, 106 with 32; forward 61 and 58).  FEW: calls of
// a few rows, where the unrolled walk of 16 spends its time fetching instructions
template <typename T, int FORM, bool SHARED, bool UNIFORM, bool BACKWARD, bool FEW>
constexpr int kRowsOf = FEW ? 4 : UNIFORM && SHARED && !BACKWARD && FORM != FR_GATE_STATIONARY && sizeof(wide_t<T>) == 4 ? 32 : 16;

__device__ __forceinline__ void put_word(unsigned long long* p, unsigned long long w)
{
    __hip_atomic_store(p, w == kUnset ? 0x7fffffff7fffffffull : w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ unsigned long long get_word(const unsigned long long* p)
{
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename S>
constexpr int kMapWords = sizeof(S) == 8 ? 2 : 1;

__device__ __forceinline__ void put_state(unsigned long long* p, double v) { put_word(p, (unsigned long long)__double_as_longlong(v)); }
__device__ __forceinline__ void put_state(unsigned long long* p, float v) { put_word(p, __float_as_uint(v)); }
__device__ __forceinline__ bool get_state(const unsigned long long* p, double& v)
{
    const unsigned long long w = get_word(p);
    v = __longlong_as_double((long long)w);
    return w != kUnset;
}
__device__ __forceinline__ bool get_state(const unsigned long long* p, float& v)
{
    const unsigned long long w = get_word(p);
    v = __uint_as_float((unsigned)w);
    return w != kUnset;
}
// A bound that a running chip never meets.  A wait that does leaves NaN in its results and raises the context's word for lost waits, which the
// host reads when it next waits or calls (lost_waits).
constexpr int kPolls = 1 << 22;
__device__ __forceinline__ void raise_lost(const RecArgs& a) { __hip_atomic_store(a.lost, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM); }

// the workgroup's tile and channel group: in order of arrival where tiles wait for one another
__device__ __forceinline__ unsigned claim_tile(const RecArgs& a, unsigned* slot)
{
    if (a.tiles == 1) return blockIdx.x;
    if (threadIdx.x == 0) *slot = atomicAdd((unsigned*)a.ticket, 1u) + 1u;  // (the counter starts from all ones too)
    __syncthreads();
    return *slot;
}

// the map of a stretch of rows; cut: a sequence begins in it, and nothing in front of it counts (an A of 0 would turn an infinite state
// of the sequence before into a NaN of this one)
//
// A is a product of gates that may leave the type's range where no state does: gates beyond 1 over many rows.  What such an infinite A is
// multiplied by may be 0 row by row -- a state of 0, or an A of 0 in front of it (a gate of 0 forgets) -- and then stays 0: the rows' own
// values are in H, and inf * 0 would be a NaN of none of them.  Where every lane joins maps it does so without these looks (CHECKED = false) and
// once more with them if a NaN came out: they took 4 % of 4194307 x 4 f64 rows.
template <bool CHECKED, typename S>
__device__ __forceinline__ S apply(S A, S state, S H)
{
    return CHECKED && state == S(0) ? H : A * state + H;
}
template <bool CHECKED, typename S>
__device__ __forceinline__ S chain(S first, S then)
{
    return CHECKED && first == S(0) ? first : first * then;
}
template <typename S>
struct Map {
    S A, H;
    bool cut;
    __device__ __forceinline__ bool nan() const { return A != A || H != H; }
    template <bool CHECKED>
    __device__ __forceinline__ S of(S state) const
    {
        return cut ? H : apply<CHECKED>(A, state, H);
    }
};
// first p, then q
template <bool CHECKED, typename S>
__device__ __forceinline__ Map<S> join(const Map<S>& p, const Map<S>& q)
{
    return {chain<CHECKED>(p.A, q.A), q.template of<CHECKED>(p.H), p.cut || q.cut};
}
// joins without the looks for zeros, and once more with them where the first way says that a NaN came out
template <class F>
__device__ __forceinline__ void joined(F&& work)
{
    if (__any(work(std::false_type()))) work(std::true_type());
}
template <typename S>
__device__ __forceinline__ Map<S> shift_up(const Map<S>& m, int step)
{
    return {__shfl_up(m.A, step), __shfl_up(m.H, step), (bool)__shfl_up((int)m.cut, step)};
}

__device__ __forceinline__ void publish(unsigned long long* p, const Map<double>& m)
{
    const unsigned long long a = m.cut ? kCut : m.A != m.A ? 0x7ff8000000000000ull : (unsigned long long)__double_as_longlong(m.A);
    put_word(p, a);
    put_word(p + 1, (unsigned long long)__double_as_longlong(m.H));
}
__device__ __forceinline__ void publish(unsigned long long* p, const Map<float>& m)
{
    const unsigned a = m.cut ? kCut32 : m.A != m.A ? 0x7fc00000u : __float_as_uint(m.A);
    put_word(p, (unsigned long long)a << 32 | __float_as_uint(m.H));
}
__device__ __forceinline__ bool published(const unsigned long long* p, Map<double>& m)
{
    const unsigned long long a = get_word(p), h = get_word(p + 1);
    m = {__longlong_as_double((long long)a), __longlong_as_double((long long)h), a == kCut};
    return a != kUnset && h != kUnset;
}
__device__ __forceinline__ bool published(const unsigned long long* p, Map<float>& m)
{
    const unsigned long long w = get_word(p);
    m = {__uint_as_float((unsigned)(w >> 32)), __uint_as_float((unsigned)w), (unsigned)(w >> 32) == kCut32};
    return w != kUnset;
}

// Where sequences begin and end among the rows [b, e) of a stretch of R rows from row0 (both lie inside all sequences): bits by steps of the
// walk, up or down the stretch, and the sequence's number for each such step.  Most stretches lie inside one sequence and end the search with
// the first look.
template <int R, bool BACKWARD>
__device__ __forceinline__ void find_edges(const RecArgs& a, int64_t lo, int64_t hi, int64_t row0, int64_t b, int64_t e, unsigned& enters, unsigned& leaves, int* number)
{
    int64_t s = 0, first = lo, next = hi;  // (the rows of all sequences: those of the only one)
    if (a.nseq > 1) {
        s = seq_of(a, b);
        first = seq_row(a, s);
        next = seq_row(a, s + 1);
    }
    for (;;) {
        const int up = (int)(first - row0), down = (int)(next - 1 - row0);
        if (first >= b && first < e) {
            const int i = BACKWARD ? R - 1 - up : up;
            (BACKWARD ? leaves : enters) |= 1u << i;
            number[i] = (int)s;
        }
        if (next > e || next <= b || next <= first) break;  // (less than b or first: offsets out of order)
        const int i = BACKWARD ? R - 1 - down : down;
        (BACKWARD ? enters : leaves) |= 1u << i;
        number[i] = (int)s;
        if (next == e) break;
        first = next;
        do next = ++s + 1 <= a.nseq ? seq_row(a, s + 1) : a.n + 1;
        while (next <= first);
        if (s >= a.nseq) break;
    }
}

// For a whole wave, rows [b, e) the same in every lane: `base` is the sequence that holds row b, lane l gets the first row of sequence base + l
// (beyond the last sequence: a row that is never reached).  64 offsets a look: two looks for 4096 sequences.
__device__ __forceinline__ int64_t wave_sequences(const RecArgs& a, int64_t b, int64_t& base)
{
    const int lane = threadIdx.x & 63;
    int64_t span = a.nseq;
    base = 0;
    while (span > 1) {
        const int64_t stride = (span + 63) >> 6, i = base + lane * stride;
        const int64_t v = seq_row(a, i < base + span ? i : base);
        const int below = __popcll(__ballot(i < base + span && v <= b));
        const int64_t skip = (below > 0 ? below - 1 : 0) * stride;
        base += skip;
        span = span - skip < stride ? span - skip : stride;
    }
    const int64_t v = seq_row(a, base + lane <= a.nseq ? base + lane : a.nseq);
    return base + lane <= a.nseq ? v : a.n + 1;
}
// whether a sequence begins or ends among the rows; many: in more places than a wave holds
__device__ __forceinline__ bool wave_edges(int64_t first, int64_t b, int64_t e, bool& many)
{
    many = __shfl(first, 63) <= e;
    return __any(first >= b && first <= e);
}
// find_edges for a whole wave
template <int R, bool BACKWARD>
__device__ __forceinline__ void find_wave_edges(const RecArgs& a, int64_t lo, int64_t hi, int64_t row0, int64_t b, int64_t e, unsigned& enters, unsigned& leaves, int* number)
{
    if (a.nseq <= 1) {
        find_edges<R, BACKWARD>(a, lo, hi, row0, b, e, enters, leaves, number);
        return;
    }
    int64_t base;
    const int64_t first = wave_sequences(a, b, base);
    bool many;
    if (!wave_edges(first, b, e, many)) return;
    if (many) {
        find_edges<R, BACKWARD>(a, lo, hi, row0, b, e, enters, leaves, number);
        return;
    }
#pragma unroll 1
    for (int64_t r = b; r < e; ++r) {
        const int up = (int)(r - row0), i = BACKWARD ? R - 1 - up : up;
        const bool begins = __any(first == r), ends = __any(first == r + 1);
        if (begins) (BACKWARD ? leaves : enters) |= 1u << i;
        if (ends) (BACKWARD ? enters : leaves) |= 1u << i;
        if (begins || ends) number[i] = (int)(base + __popcll(__ballot(first <= r)) - 1);
    }
}

// ---- rows side by side (FR_LAYOUT_ROWMAJOR) --------------------------------------------------------------------------------------------
//
// A lane holds V neighbouring channels of R rows in registers, so the data are read once; 2^lanes lanes stand side by side across the channels,
// a wave holds 64 >> lanes such stretches of rows and the workgroup's waves the rows after them.  UNIFORM: a wave holds one stretch
// (64 channel lanes), so rows, their addresses and what begins and ends in them are the same for the whole wave and cost no vector
// instruction; a stretch inside one sequence then runs without a branch.
//
// bf16, a gate for 128 channels, 37 sequences of 16413 rows x 2048 channels: backward 203 MB in 96 us on inputs that change from call to
// call, 2.1 TB/s; 84 on the same ones (with vector addresses and edges looked for in every row 113 and more).  Vector instructions issue in
// 22 % of that.  The rest is the wait for the maps in front and the tail: a workgroup of 8 waves fills the
// registers of its CU, so loading, waiting and storing take turns.  3, 4 and 6 waves, windows of 8 and 32 tiles and 128 registers a lane were no
// faster.  Rows of fewer than 64 channels, or of channels that share a gate in pairs, are further off: a lane holds one channel there, 2 bytes
// of a 16-bit type (2^23 elements of f16: 36 to 50 MB in 49 to 70 us).  24 sequences of one row: 11 us, where a small launch takes 4; offsets,
// rows, maps and given states are trips to memory one after the other, on four workgroups.

template <typename T, int FORM, int V, bool SHARED, bool BACKWARD, bool UNIFORM, bool FEW>
__global__ __launch_bounds__(512) void rec_rows_kernel(const RecArgs a)
{
    using S = wide_t<T>;
    constexpr int R = kRowsOf<T, FORM, SHARED, UNIFORM, BACKWARD, FEW>;
    constexpr int BATCH = R < 8 ? R : 8;
    __shared__ unsigned slot;
    __shared__ S mapA[kWaves][V][64], mapH[kWaves][V][64], front[V][64];
    __shared__ int mapC[kWaves][V][64];
    __shared__ int sequence[UNIFORM ? kWaves : kWaves * 64][R];  // of a stretch's rows that begin or end one
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int across = UNIFORM ? 64 : 1 << a.lanes, cl = UNIFORM ? lane : lane & (across - 1), group = UNIFORM ? 0 : lane >> a.lanes, groups = UNIFORM ? 1 : 64 >> a.lanes;
    const unsigned item = __builtin_amdgcn_readfirstlane(claim_tile(a, &slot));
    const int64_t pos = item / (unsigned)a.blocks;  // tiles in the order of the walk
    const unsigned c = ((item % (unsigned)a.blocks) * across + cl) * V;
    const bool live = c < a.d;
    const unsigned cc = live ? c : 0;
    const int64_t lo = seq_row(a, 0), hi = seq_row(a, a.nseq);
    const int64_t stretch = pos * (waves * groups) + wave * groups + group;  // of R rows, in the order of the walk
    // rows row0 .. row0 + R - 1, walked upwards or downwards; those inside all sequences are [rb, re)
    const int64_t row0 = BACKWARD ? (a.stretches - 1 - stretch) * R : stretch * R;
    const int64_t rb = lo > row0 ? lo : row0, re = hi < row0 + R ? hi : row0 + R;
    const bool any = stretch < a.stretches && rb < re;
    auto row_at = [&](int i) { return BACKWARD ? row0 + (R - 1 - i) : row0 + i; };
    auto address_row = [&](int64_t r) { return r < 0 ? 0 : (r >= a.n ? a.n - 1 : r); };

    const T* gate = (const T*)a.gate;
    const unsigned gc0 = SHARED ? cc / (unsigned)a.width : cc;
    const T* in = (const T*)(BACKWARD ? a.dh : a.x);
    const int64_t in_r = BACKWARD ? a.dh_r : a.x_r;
    Run<T, V> raw[R];
    Run<T, V> graw[SHARED ? 1 : R];
    S ga[SHARED ? R : 1], gc[SHARED && FORM == FR_GATE_STATIONARY ? R : 1];
    if (a.n > 0) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int64_t r = address_row(row_at(i));
            raw[i] = load_run<T, V>(in + r * in_r + cc);
            if constexpr (SHARED)
                ga[i] = widen((gate + r * a.gate_r)[gc0]);
            else
                graw[i] = load_run<T, V>(gate + r * a.gate_r + gc0);
        }
    }
    if constexpr (SHARED) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const Gate<S> g = gate_of<FORM, S>(ga[i]);
            ga[i] = g.a;
            if constexpr (FORM == FR_GATE_STATIONARY) gc[i] = g.c;
        }
    }
    auto gate_at = [&](int i, int v) -> Gate<S> {
        if constexpr (SHARED) {
            if constexpr (FORM == FR_GATE_STATIONARY) return {ga[i], gc[i]};
            return {ga[i], S(1)};
        } else
            return gate_of<FORM, S>(widen(graw[i].v[v]));
    };

    // steps of the walk that are rows of a sequence, that enter one, and that leave one
    unsigned valid = 0, enters = 0, leaves = 0;
    int* seq = sequence[wave * groups + group];
    if (any) {
        const int first = BACKWARD ? (int)(row0 + R - re) : (int)(rb - row0), count = (int)(re - rb);
        valid = (count >= 32 ? ~0u : (1u << count) - 1u) << first;
        if constexpr (UNIFORM)
            find_wave_edges<R, BACKWARD>(a, lo, hi, row0, rb, re, enters, leaves, seq);
        else
            find_edges<R, BACKWARD>(a, lo, hi, row0, rb, re, enters, leaves, seq);
    }
    if constexpr (UNIFORM) {
        valid = __builtin_amdgcn_readfirstlane(valid);
        enters = __builtin_amdgcn_readfirstlane(enters);
        leaves = __builtin_amdgcn_readfirstlane(leaves);
    }
    constexpr unsigned ALL = R == 32 ? ~0u : (1u << (R & 31)) - 1u;
    const bool plain = UNIFORM && valid == ALL && (enters | leaves) == 0;
    const S* edge = (const S*)(BACKWARD ? a.dlast : a.h0);  // the state a sequence is entered with
    const int64_t edge_r = BACKWARD ? a.dlast_r : a.h0_r;

    // one row: the state of a channel moves on; returns G (backward) or h (forward)
    auto step = [&](const Gate<S>& g, S u, S& state) -> S {
        if constexpr (BACKWARD) {
            const S G = u + state;
            state = g.a * G;
            return G;
        } else {
            state = g.a * state + (FORM == FR_GATE_STATIONARY ? g.c * u : u);
            return state;
        }
    };

    S state[V];
    if (a.tiles > 1 || groups > 1 || waves > 1) {  // (uniform) the map of the thread's rows, then the state in front of them
        Map<S> m[V];
#pragma unroll
        for (int v = 0; v < V; ++v) m[v] = {S(1), S(0), false};
        auto reduce = [&](auto edges) {
#pragma unroll
            for (int i = 0; i < R; ++i) {
                if (decltype(edges)::value && !(valid >> i & 1)) continue;
                if (decltype(edges)::value && (enters >> i & 1)) {
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        // (what stands in front of the last entry does not come through)
                        m[v].H = edge && live && !(enters >> i >> 1) ? edge[seq[i] * edge_r + c + v] : S(0);
                        m[v].cut = true;
                    }
                }
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const Gate<S> g = gate_at(i, v);
                    step(g, widen(raw[i].v[v]), m[v].H);
                    if (!SHARED || v == 0) m[v].A *= g.a;
                }
            }
        };
        if (plain)
            reduce(std::false_type());
        else
            reduce(std::true_type());
        if constexpr (SHARED)
#pragma unroll
            for (int v = 1; v < V; ++v) m[v].A = m[0].A;
        // across the stretches of the wave (lanes `across` apart), then across the waves
        Map<S> before[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            before[v] = {S(1), S(0), false};
            if constexpr (!UNIFORM) {
                const Map<S> own = m[v];
                joined([&](auto checked) {
                    m[v] = own;
                    for (int d = across; d < 64; d *= 2) {
                        const Map<S> p = shift_up(m[v], d);
                        if (lane >= d) m[v] = join<decltype(checked)::value>(p, m[v]);
                    }
                    return m[v].nan();
                });
                const Map<S> p = shift_up(m[v], across);
                if (group > 0) before[v] = p;
            }
            if (group == groups - 1) {
                mapA[wave][v][cl] = m[v].A;
                mapH[wave][v][cl] = m[v].H;
                mapC[wave][v][cl] = m[v].cut;
            }
        }
        __syncthreads();
        for (int v = wave; v < V; v += waves) {
            if (lane < across) {
                const int64_t ch = ((int64_t)(item % (unsigned)a.blocks) * across + lane) * V + v;
                S st = S(0);
                if (a.tiles > 1 && ch < a.d) {
                    Map<S> all;
                    joined([&](auto checked) {
                        all = {mapA[0][v][lane], mapH[0][v][lane], mapC[0][v][lane] != 0};
                        for (int k = 1; k < waves; ++k) all = join<decltype(checked)::value>(all, Map<S>{mapA[k][v][lane], mapH[k][v][lane], mapC[k][v][lane] != 0});
                        return all.nan();
                    });
                    unsigned long long* words = (unsigned long long*)a.maps;
                    unsigned long long* states = (unsigned long long*)a.carry;
                    publish(words + (pos * a.d + ch) * kMapWords<S>, all);
                    // the maps of the block first, made one, so that only one product lies between a state's arrival and the next one's leaving
                    const int64_t block = pos / kRowsWindow, from = block * kRowsWindow;
                    const int ahead = (int)(pos - from);
                    Map<S> sum = {S(1), S(0), false};
                    bool lost = false;
                    for (int k0 = 0; k0 < ahead; k0 += 8) {
                        Map<S> seen[8];
                        for (int poll = 0;; ++poll) {
                            bool ok = true;
#pragma unroll
                            for (int k = 0; k < 8; ++k) {
                                const int64_t at = from + (k0 + k < ahead ? k0 + k : k0);
                                ok = published(words + (at * a.d + ch) * kMapWords<S>, seen[k]) && ok;
                            }
                            lost |= poll == a.polls;
                            if (ok || lost) break;
                            __builtin_amdgcn_s_sleep(1);
                        }
                        const Map<S> so_far = sum;
                        joined([&](auto checked) {
                            sum = so_far;
#pragma unroll
                            for (int k = 0; k < 8; ++k)
                                if (k0 + k < ahead) sum = join<decltype(checked)::value>(sum, seen[k]);
                            return sum.nan();
                        });
                    }
                    if (lost) sum = {S(1), S(NAN), true};
                    Map<S> onward;
                    joined([&](auto checked) {
                        onward = join<decltype(checked)::value>(sum, all);
                        return onward.nan();
                    });
                    for (int poll = 0; block > 0; ++poll) {
                        if (get_state(states + (block - 1) * a.d + ch, st)) break;
                        if (poll == a.polls) {
                            st = S(NAN);
                            lost = true;
                            break;
                        }
                    }
                    S through = S(0), front_of = S(0);
                    joined([&](auto checked) {
                        constexpr bool CHECKED = decltype(checked)::value;
                        through = onward.template of<CHECKED>(st);
                        front_of = sum.template of<CHECKED>(st);
                        return through != through || front_of != front_of;
                    });
                    if (ahead == kRowsWindow - 1) put_state(states + block * a.d + ch, through);
                    st = front_of;
                    if (lost) raise_lost(a);
                }
                front[v][lane] = st;
            }
        }
        __syncthreads();
        joined([&](auto checked) {
            constexpr bool CHECKED = decltype(checked)::value;
            bool nan = false;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                S st = front[v][cl];
                for (int k = 0; k < wave; ++k) st = Map<S>{mapA[k][v][cl], mapH[k][v][cl], mapC[k][v][cl] != 0}.template of<CHECKED>(st);
                state[v] = before[v].template of<CHECKED>(st);
                nan |= state[v] != state[v];
            }
            return nan;
        });
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v) state[v] = S(0);
    }

    // the states that the next rows' sequences are entered with: loads under a condition would be waited for one by one
    S given[BATCH][V];
    auto fetch = [&](int i0) {
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int64_t s = enters >> (i0 + i) & 1 ? seq[i0 + i] : 0;
            if (edge) {
                const Run<S, V> r = load_run<S, V>(edge + s * edge_r + cc);
#pragma unroll
                for (int v = 0; v < V; ++v) given[i][v] = r.v[v];
            } else
#pragma unroll
                for (int v = 0; v < V; ++v) given[i][v] = S(0);
        }
    };

    // the walk itself
    if constexpr (!BACKWARD) {
        T* out = (T*)a.h;
        S* last = (S*)a.last;
        auto walk = [&](auto edges) {
#pragma unroll
            for (int i = 0; i < R; ++i) {
                if (decltype(edges)::value && i % BATCH == 0) fetch(i);
                if (decltype(edges)::value && !(valid >> i & 1)) continue;
                if (decltype(edges)::value && (enters >> i & 1)) {
#pragma unroll
                    for (int v = 0; v < V; ++v) state[v] = given[i % BATCH][v];
                }
                Run<T, V> y;
#pragma unroll
                for (int v = 0; v < V; ++v) y.v[v] = narrow<T>(step(gate_at(i, v), widen(raw[i].v[v]), state[v]));
                store_run<T, V>(out + row_at(i) * a.h_r + c, y);
                if (decltype(edges)::value && last && (leaves >> i & 1)) {
                    Run<S, V> r;
#pragma unroll
                    for (int v = 0; v < V; ++v) r.v[v] = state[v];
                    store_run<S, V>(last + seq[i] * a.last_r + c, r);
                }
            }
        };
        if (live) {
            if (plain)
                walk(std::false_type());
            else
                walk(std::true_type());
        }
        if (last)  // sequences without rows end in the state they began with
            for (int64_t s0 = pos * (waves * groups) + wave * groups + group; s0 < a.nseq; s0 += a.tiles * (waves * groups))
                if (live && seq_row(a, s0 + 1) <= seq_row(a, s0))
#pragma unroll
                    for (int v = 0; v < V; ++v) last[s0 * a.last_r + c + v] = edge ? edge[s0 * edge_r + c + v] : S(0);
    } else {
        const T* hin = (const T*)a.hin;
        const T* x = (const T*)a.x;
        const S* h0 = (const S*)a.h0;
        S* dh0 = (S*)a.dh0;
        T* dx = (T*)a.dx;
        auto walk = [&](auto edges) {
#pragma unroll
            for (int i0 = 0; i0 < R; i0 += BATCH) {
                Run<T, V> hb[BATCH], xb[FORM == FR_GATE_STATIONARY ? BATCH : 1];
                if (a.dgate && a.n > 0) {
#pragma unroll
                    for (int i = 0; i < BATCH; ++i) {
                        hb[i] = load_run<T, V>(hin + address_row(row_at(i0 + i) - 1) * a.h_r + cc);
                        if constexpr (FORM == FR_GATE_STATIONARY) xb[i] = load_run<T, V>(x + address_row(row_at(i0 + i)) * a.x_r + cc);
                    }
                }
                S sum[BATCH];
                if (decltype(edges)::value) fetch(i0);
#pragma unroll
                for (int i = 0; i < BATCH; ++i) {
                    const int64_t r = row_at(i0 + i);
                    sum[i] = S(0);
                    if (decltype(edges)::value && !(valid >> (i0 + i) & 1)) continue;
                    if (decltype(edges)::value && (enters >> (i0 + i) & 1)) {
#pragma unroll
                        for (int v = 0; v < V; ++v) state[v] = given[i][v];
                    }
                    const bool first = decltype(edges)::value && (leaves >> (i0 + i) & 1);
                    Run<T, V> y, z;
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        const Gate<S> g = gate_at(i0 + i, v);
                        const S G = step(g, widen(raw[i0 + i].v[v]), state[v]);
                        y.v[v] = narrow<T>(FORM == FR_GATE_STATIONARY ? g.c * G : G);
                        if (a.dgate) {
                            S prev = widen(hb[i].v[v]);
                            if (first) prev = h0 && live ? h0[seq[i0 + i] * a.h0_r + c + v] : S(0);
                            const S dg = gate_grad<FORM, S>(g, G, prev, FORM == FR_GATE_STATIONARY ? widen(xb[FORM == FR_GATE_STATIONARY ? i : 0].v[v]) : S(0));
                            if constexpr (SHARED) {
                                sum[i] += dg;
                                if (a.sum_lanes == 0 && live) ((S*)a.part)[r * a.part_r + (c + v) * a.part_c] = dg;
                            } else
                                z.v[v] = narrow<T>(dg);
                        }
                    }
                    if (live) {
                        if (a.dx) store_run<T, V>(dx + r * a.dx_r + c, y);
                        if constexpr (!SHARED)
                            if (a.dgate) store_run<T, V>((T*)a.dgate + r * a.dg_r + c, z);
                        if (dh0 && first) {
#pragma unroll
                            for (int v = 0; v < V; ++v) dh0[seq[i0 + i] * a.dh0_r + c + v] = state[v];
                        }
                    } else
                        sum[i] = S(0);
                }
                if constexpr (SHARED) {
                    if (a.dgate && a.sum_lanes > 0) {
                        for (int d = 1; d < a.sum_lanes; d *= 2)
#pragma unroll
                            for (int i = 0; i < BATCH; ++i) sum[i] += __shfl_xor(sum[i], d);
                        if (live && (cl & (a.sum_lanes - 1)) == 0) {
#pragma unroll
                            for (int i = 0; i < BATCH; ++i) {
                                const int64_t r = row_at(i0 + i);
                                if (decltype(edges)::value && !(valid >> (i0 + i) & 1)) continue;
                                if (a.pieces == 1)
                                    ((T*)a.dgate)[r * a.dg_r + gc0] = narrow<T>(sum[i]);
                                else
                                    ((S*)a.part)[r * a.part_r + c / (64 * V)] = sum[i];
                            }
                        }
                    }
                }
            }
        };
        if (plain)
            walk(std::false_type());
        else
            walk(std::true_type());
        if (dh0)
            for (int64_t s0 = pos * (waves * groups) + wave * groups + group; s0 < a.nseq; s0 += a.tiles * (waves * groups))
                if (live && seq_row(a, s0 + 1) <= seq_row(a, s0))
#pragma unroll
                    for (int v = 0; v < V; ++v) dh0[s0 * a.dh0_r + c + v] = edge ? edge[s0 * edge_r + c + v] : S(0);
    }
}

// ---- columns one after the other (FR_LAYOUT_COLMAJOR) ----------------------------------------------------------------------------------
//
// A lane holds E neighbouring rows of up to CG channels that share their gate, a workgroup 64 E rows a wave.  The gate is read, and its
// exponential worked out, once for those channels.
//
// f64, three channels on one gate, 1000003 x 3 backward: 112 MB in 39 us on inputs that change from call to call, 2.9 TB/s (32 on the same ones,
// which the last-level cache holds); four on one, 4194307 x 4 forward: 302 MB in 111 us, 2.7 TB/s.
// Bound as the rows are, by tiles that load, wait and store in turn; 16-bit types load 16 bytes a lane and are further off (2^23 elements of
// f16, 8 columns: 50 MB in 49 us; 1000 columns of 300 sequences 66, where every lane near an edge searches the offsets).  (With blocks of 256 tiles and a map's words apart for each channel 149; 16 waves of 4
// rows a lane 99, but 44 instead of 40 where there is one channel).

template <typename T, int FORM, int CG, bool BACKWARD>
__global__ __launch_bounds__(512) void rec_columns_kernel(const RecArgs a)
{
    using S = wide_t<T>;
    constexpr int E = kRowsOfLane;
    __shared__ unsigned slot;
    __shared__ S mapA[kWaves], mapH[CG][kWaves], front[CG];
    __shared__ int mapC[kWaves];
    __shared__ int sequence[64 * kWaves][E + 1];  // of a lane's rows that begin or end one (a stride that spreads the banks)
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const unsigned item = __builtin_amdgcn_readfirstlane(claim_tile(a, &slot));
    const int64_t pos = item / a.blocks;
    const int64_t block = item % a.blocks, q = block / a.pieces, piece = block % a.pieces;
    const int64_t c0 = q * a.width + piece * CG;
    const int ng = (int)(a.width - piece * CG < CG ? a.width - piece * CG : CG);
    const int64_t lo = seq_row(a, 0), hi = seq_row(a, a.nseq);
    const int64_t run = pos * blockDim.x + threadIdx.x;  // runs of E rows, in the order of the walk
    const int64_t row0 = BACKWARD ? (a.stretches - 1 - run) * E : run * E;
    const bool there = run < a.stretches;
    const int64_t rb = lo > row0 ? lo : row0, re = hi < row0 + E ? hi : row0 + E;
    const bool any = there && rb < re;
    const bool full = any && re - rb == E;
    // step i of the walk is element at(i) of the run
    auto at = [](int i) { return BACKWARD ? E - 1 - i : i; };

    auto load = [&](const T* p) {  // E elements of a column from row0; rows that are not there: 0
        Run<T, E> r;
        p += row0;  // (outside the branches: an address worked out in one took registers that a load of the other was still to fill, and waited)
        if (there && row0 + E <= a.n)
            r = load_run<T, E>(p);
        else
#pragma unroll
            for (int i = 0; i < E; ++i) r.v[i] = there && row0 + i < a.n ? p[i] : narrow<T>(S(0));
        return r;
    };

    S ga[E], gc[FORM == FR_GATE_STATIONARY ? E : 1], u[CG][E];
    {
        const Run<T, E> g = load((const T*)a.gate + q * a.gate_c);
        Run<T, E> in[CG];
#pragma unroll
        for (int j = 0; j < CG; ++j)
            if (j < ng) in[j] = load((const T*)(BACKWARD ? a.dh : a.x) + (c0 + j) * (BACKWARD ? a.dh_c : a.x_c));
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const Gate<S> v = gate_of<FORM, S>(widen(g.v[at(i)]));
            ga[i] = v.a;
            if constexpr (FORM == FR_GATE_STATIONARY) gc[i] = v.c;
#pragma unroll
            for (int j = 0; j < CG; ++j) {
                u[j][i] = j < ng ? widen(in[j].v[at(i)]) : S(0);
                if constexpr (FORM == FR_GATE_STATIONARY && !BACKWARD) u[j][i] *= v.c;
            }
        }
    }
    // rows that enter a sequence (bit i: step i), with the state they enter it with added to their input, and rows that leave one
    unsigned enters = 0, leaves = 0;
    unsigned valid = 0;
#pragma unroll
    for (int i = 0; i < E; ++i)
        if (any && row0 + at(i) >= rb && row0 + at(i) < re) valid |= 1u << i;
    const S* edge = (const S*)(BACKWARD ? a.dlast : a.h0);
    const int64_t edge_c = BACKWARD ? a.dlast_c : a.h0_c;
    int* seq = sequence[threadIdx.x];
    bool edges = true;
    if (a.nseq > 1) {  // most waves lie inside one sequence
        const int64_t w0 = pos * blockDim.x + wave * 64, w1 = w0 + 64 < a.stretches ? w0 + 64 : a.stretches;
        const int64_t r0 = BACKWARD ? (a.stretches - w1) * E : w0 * E, r1 = BACKWARD ? (a.stretches - w0) * E : w1 * E;
        const int64_t b = r0 > lo ? r0 : lo, e = r1 < hi ? r1 : hi;
        edges = false;
        if (b < e) {
            int64_t base;
            const int64_t first = wave_sequences(a, b, base);
            bool many;
            edges = wave_edges(first, b, e, many) || many;
        }
    }
    if (any && edges) find_edges<E, BACKWARD>(a, lo, hi, row0, rb, re, enters, leaves, seq);
    if (enters && edge) {
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (enters >> i & 1)
#pragma unroll
                for (int j = 0; j < CG; ++j)
                    if (j < ng) {
                        const S h = edge[seq[i] + (c0 + j) * edge_c];
                        u[j][i] = BACKWARD ? u[j][i] + h : ga[i] * h + u[j][i];
                    }
    }
    // a row's result from the state in front of it, and the state behind it
    auto step = [&](int i, S in, S state, S& through) -> S {
        const bool cut = enters >> i & 1;
        if constexpr (BACKWARD) {
            const S G = cut ? in : in + state;
            through = ga[i] * G;
            return G;
        } else {
            const S h = cut ? in : ga[i] * state + in;
            through = h;
            return h;
        }
    };

    // the map of the lane's rows (the channels share its factor), of the rows of the lanes before it, and of the wave
    S A, H[CG];
    bool cut;
    joined([&](auto checked) {
        constexpr bool CHECKED = decltype(checked)::value;
        A = S(1), cut = enters != 0;
#pragma unroll
        for (int j = 0; j < CG; ++j) H[j] = S(0);
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (valid >> i & 1) {
#pragma unroll
                for (int j = 0; j < CG; ++j) step(i, u[j][i], H[j], H[j]);
                A *= ga[i];
            }
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const S pa = __shfl_up(A, d);
            const bool pc = __shfl_up((int)cut, d);
#pragma unroll
            for (int j = 0; j < CG; ++j) {
                const S ph = __shfl_up(H[j], d);
                if (lane >= d && !cut) H[j] = apply<CHECKED>(A, ph, H[j]);
            }
            if (lane >= d) {
                A = chain<CHECKED>(pa, A);
                cut = cut || pc;
            }
        }
        bool nan = A != A;
#pragma unroll
        for (int j = 0; j < CG; ++j) nan |= H[j] != H[j];
        return nan;
    });
    if (lane == 63) {
        mapA[wave] = A;
        mapC[wave] = cut;
#pragma unroll
        for (int j = 0; j < CG; ++j) mapH[j][wave] = H[j];
    }
    A = __shfl_up(A, 1);
    cut = __shfl_up((int)cut, 1);
#pragma unroll
    for (int j = 0; j < CG; ++j) H[j] = __shfl_up(H[j], 1);
    if (lane == 0) {
        A = S(1), cut = false;
#pragma unroll
        for (int j = 0; j < CG; ++j) H[j] = S(0);
    }
    __syncthreads();
    for (int j = wave; j < ng; j += waves) {
        S st = S(0);
        if (a.tiles > 1) {
            // (one lane's joins here and below: the looks for zeros cost less than a second way)
            Map<S> all = {mapA[0], mapH[j][0], mapC[0] != 0};
            for (int k = 1; k < waves; ++k) all = join<true>(all, Map<S>{mapA[k], mapH[j][k], mapC[k] != 0});
            // (a channel's words lie side by side: a wave reads the window's in a few lines)
            unsigned long long* words = (unsigned long long*)a.maps + (c0 + j) * a.tiles * kMapWords<S>;
            unsigned long long* states = (unsigned long long*)a.carry + (c0 + j) * (a.tiles / kColumnsWindow + 1);
            if (lane == 0) publish(words + pos * kMapWords<S>, all);
            // the maps of the window first, made one, so that only one product lies between a state's arrival and the next one's leaving
            const int64_t window = pos / kColumnsWindow, from = window * kColumnsWindow;
            const int ahead = (int)(pos - from);
            Map<S> m = {S(1), S(0), false};
            bool lost = false;
            for (int poll = 0;; ++poll) {
                const bool ok = lane >= ahead || published(words + (from + lane) * kMapWords<S>, m);
                lost = poll == a.polls;
                if (__all(ok) || lost) break;
                __builtin_amdgcn_s_sleep(2);
            }
            if (lane >= ahead) m = {S(1), S(0), false};
            if (lost) m = {S(1), S(NAN), true};
#pragma unroll
            for (int d = 1; d < 64; d *= 2) {
                const Map<S> p = shift_up(m, d);
                if (lane >= d) m = join<true>(p, m);
            }
            m = {__shfl(m.A, 63), __shfl(m.H, 63), (bool)__shfl((int)m.cut, 63)};
            const Map<S> through = join<true>(m, all);
            for (int poll = 0; window > 0; ++poll) {
                if (get_state(states + window - 1, st)) break;
                if (poll == a.polls) {
                    st = S(NAN);
                    lost = true;
                    break;
                }
                __builtin_amdgcn_s_sleep(1);
            }
            if (ahead == kColumnsWindow - 1 && lane == 0) put_state(states + window, through.template of<true>(st));
            st = m.template of<true>(st);
            if (lost && lane == 0) raise_lost(a);
        }
        if (lane == 0) front[j] = st;
    }
    __syncthreads();
    S state[CG];
    joined([&](auto checked) {
        constexpr bool CHECKED = decltype(checked)::value;
        bool nan = false;
#pragma unroll
        for (int j = 0; j < CG; ++j) {
            if (j >= ng) continue;
            S st = front[j];
            for (int k = 0; k < wave; ++k) st = Map<S>{mapA[k], mapH[j][k], mapC[k] != 0}.template of<CHECKED>(st);
            state[j] = cut ? H[j] : apply<CHECKED>(A, st, H[j]);
            nan |= state[j] != state[j];
        }
        return nan;
    });

    if constexpr (!BACKWARD) {
        S* last = (S*)a.last;
#pragma unroll
        for (int j = 0; j < CG; ++j) {
            if (j >= ng || !any) continue;
            T* out = (T*)a.h + (c0 + j) * a.h_c + row0;
            Run<T, E> y;
#pragma unroll
            for (int i = 0; i < E; ++i) {
                if (valid >> i & 1) {
                    y.v[at(i)] = narrow<T>(step(i, u[j][i], state[j], state[j]));
                    if (!full) out[at(i)] = y.v[at(i)];
                    if (last && (leaves >> i & 1)) last[seq[i] + (c0 + j) * a.last_c] = state[j];
                }
            }
            if (full) store_run<T, E>(out, y);
        }
        if (last)
            for (int64_t s0 = pos * blockDim.x + threadIdx.x; s0 < a.nseq; s0 += a.tiles * blockDim.x)
                if (seq_row(a, s0 + 1) <= seq_row(a, s0))
                    for (int j = 0; j < ng; ++j) last[s0 + (c0 + j) * a.last_c] = edge ? edge[s0 + (c0 + j) * edge_c] : S(0);
    } else {
        const S* h0 = (const S*)a.h0;
        S* dh0 = (S*)a.dh0;
        S dg[E];
#pragma unroll
        for (int i = 0; i < E; ++i) dg[i] = S(0);
#pragma unroll
        for (int j = 0; j < CG; ++j) {
            if (j >= ng || !any) continue;
            const int64_t ch = c0 + j;
            S prev[E];  // of step i: the state in front of its row
            Run<T, E> xr;
            if (a.dgate) {
                const T* hin = (const T*)a.hin + ch * a.h_c + row0 - 1;
                if (row0 > 0 && row0 + E <= a.n) {
                    const Run<T, E> hr = load_run<T, E>(hin);
#pragma unroll
                    for (int i = 0; i < E; ++i) prev[i] = widen(hr.v[at(i)]);
                } else {
#pragma unroll
                    for (int i = 0; i < E; ++i) prev[i] = row0 + at(i) > 0 && row0 + at(i) <= a.n ? widen(hin[at(i)]) : S(0);
                }
                if constexpr (FORM == FR_GATE_STATIONARY) xr = load((const T*)a.x + ch * a.x_c);
            }
            T* dx = (T*)a.dx + ch * a.dx_c + row0;
            Run<T, E> y;
#pragma unroll
            for (int i = 0; i < E; ++i) {
                if (valid >> i & 1) {
                    const S G = step(i, u[j][i], state[j], state[j]);
                    Gate<S> g = {ga[i], S(1)};
                    if constexpr (FORM == FR_GATE_STATIONARY) g.c = gc[i];
                    y.v[at(i)] = narrow<T>(FORM == FR_GATE_STATIONARY ? g.c * G : G);
                    if (!full && a.dx) dx[at(i)] = y.v[at(i)];
                    const bool first = leaves >> i & 1;
                    if (a.dgate) {
                        const S before = first ? (h0 ? h0[seq[i] + ch * a.h0_c] : S(0)) : prev[i];
                        S x = S(0);
                        if constexpr (FORM == FR_GATE_STATIONARY) x = widen(xr.v[at(i)]);
                        dg[i] += gate_grad<FORM, S>(g, G, before, x);
                    }
                    if (dh0 && first) dh0[seq[i] + ch * a.dh0_c] = state[j];
                }
            }
            if (full && a.dx) store_run<T, E>(dx, y);
        }
        if (a.dgate && any) {
            if (a.pieces == 1) {
                T* out = (T*)a.dgate + q * a.dg_c + row0;
                Run<T, E> y;
#pragma unroll
                for (int i = 0; i < E; ++i) y.v[at(i)] = narrow<T>(dg[i]);
                if (full)
                    store_run<T, E>(out, y);
                else
#pragma unroll
                    for (int i = 0; i < E; ++i)
                        if (valid >> i & 1) out[at(i)] = y.v[at(i)];
            } else {
                S* out = (S*)a.part + block * a.part_c + row0;
#pragma unroll
                for (int i = 0; i < E; ++i)
                    if (valid >> i & 1) out[at(i)] = dg[i];
            }
        }
        if (dh0)
            for (int64_t s0 = pos * blockDim.x + threadIdx.x; s0 < a.nseq; s0 += a.tiles * blockDim.x)
                if (seq_row(a, s0 + 1) <= seq_row(a, s0))
                    for (int j = 0; j < ng; ++j) dh0[s0 + (c0 + j) * a.dh0_c] = edge ? edge[s0 + (c0 + j) * edge_c] : S(0);
    }
}

// The sum of a gate's parts, as many as it has channels where their number fits no wave: thousands of terms that may all round the same way.
// Parts of 32 bits are summed in 64; of 64 bits each addition's error is kept and added at the end (two-sum).  Either way the sum adds a
// few roundings whatever the number of parts, as the tree over a wave's lanes does.
template <typename S>
struct Total;
template <>
struct Total<float> {
    double v = 0.0;
    __device__ __forceinline__ void add(float x) { v += (double)x; }
    __device__ __forceinline__ float get() const { return (float)v; }
};
template <>
struct Total<double> {
    double v = 0.0, rest = 0.0;
    __device__ __forceinline__ void add(double x)
    {
        const double s = v + x, b = s - v;
        rest += (v - (s - b)) + (x - b);
        v = s;
    }
    __device__ __forceinline__ double get() const { return isfinite(v) ? v + rest : v; }
};

// dgate of a shared gate from its parts, in one order on every run
template <typename T>
__global__ __launch_bounds__(256) void rec_heads_kernel(const RecArgs a)
{
    using S = wide_t<T>;
    const int64_t lo = seq_row(a, 0), hi = seq_row(a, a.nseq), step = (int64_t)gridDim.x * blockDim.x;
    for (int64_t id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; id < a.n * a.cols; id += step) {
        const int64_t r = a.part_r == 1 ? id % a.n : id / a.cols, q = a.part_r == 1 ? id / a.n : id % a.cols;
        if (r < lo || r >= hi) continue;
        const S* p = (const S*)a.part + r * a.part_r + q * a.pieces * a.part_c;
        Total<S> sum[4];  // (four chains: an addition and its error take four dependent instructions)
        int64_t i = 0;
        for (; i + 4 <= a.pieces; i += 4)
#pragma unroll
            for (int k = 0; k < 4; ++k) sum[k].add(p[(i + k) * a.part_c]);
        for (; i < a.pieces; ++i) sum[0].add(p[i * a.part_c]);
        ((T*)a.dgate)[r * a.dg_r + q * a.dg_c] = narrow<T>((sum[0].get() + sum[1].get()) + (sum[2].get() + sum[3].get()));
    }
}

// ---- host side ----------------------------------------------------------------------------------------------------------------------

// The workgroups along the rows, and the memory that passes states between them (none for a single one)
template <typename T>
static int rec_prepare(fr_ctx* ctx, RecArgs& a, int64_t rows, int64_t stretches_of_wave, int most, int64_t window, int64_t parts, OpWorkspace& ws, int* waves)
{
    using S = wide_t<T>;
    a.stretches = (a.n + rows - 1) / rows;
    int64_t w = (a.stretches + stretches_of_wave - 1) / stretches_of_wave;
    *waves = (int)(w < 1 ? 1 : (w > most ? most : w));
    a.tiles = (a.stretches + *waves * stretches_of_wave - 1) / (*waves * stretches_of_wave);
    if (a.tiles < 1) a.tiles = 1;
    if (a.tiles * a.blocks * 64 * *waves > 0xffffffffLL) return set_err(ctx, FR_SHAPE, "%lld rows of %lld channels are too many for one call", (long long)a.n, (long long)a.d);
    const int64_t maps = a.tiles * a.d * kMapWords<S>, states = (a.tiles / window + 1) * a.d;
    const int64_t words = a.tiles > 1 ? 1 + maps + states : 0;
    if (words + parts == 0) return FR_OK;
    FR_TRY(ws.get((size_t)(words * 8 + parts * (int64_t)sizeof(S))));
    a.lost = ctx->dev_status + 1, a.polls = ctx->test_wait_polls >= 0 ? ctx->test_wait_polls : kPolls;
    unsigned long long* p = (unsigned long long*)ws.p;
    a.ticket = p;
    a.maps = p + 1;
    a.carry = p + 1 + maps;
    a.part = p + words;
    return words ? launch_unset(ctx, p, words) : FR_OK;
}

template <typename T, int FORM, int V, bool SHARED>
static int rec_rows(fr_ctx* ctx, RecArgs& a, bool backward, OpWorkspace& ws)
{
    a.lanes = 0;
    while (a.lanes < 6 && (V << a.lanes) < a.d) ++a.lanes;
    const int64_t across = 1 << a.lanes, span = across * V;
    a.blocks = (a.d + span - 1) / span;
    a.pieces = 1, a.sum_lanes = 0;
    int64_t parts = 0;
    if (SHARED && backward && a.dgate) {
        const int64_t lanes = a.width / V;
        if (a.cols == 1 && a.blocks == 1)
            a.sum_lanes = (int)across;
        else if (a.lanes == 6 && a.width % span == 0)
            a.sum_lanes = 64, a.pieces = a.width / span;
        else if (lanes <= across && (lanes & (lanes - 1)) == 0)
            a.sum_lanes = (int)lanes;
        else
            a.pieces = a.width;
        if (a.pieces > 1) {
            a.part_r = a.cols * a.pieces, a.part_c = 1;
            parts = a.n * a.part_r;
        }
    }
    int waves;
    const bool few = !backward && a.lanes == 6 && a.n <= kFewRows;
    const int64_t rows = few ? kRowsOf<T, FORM, SHARED, true, false, true> : backward || a.lanes < 6 ? kRowsOf<T, FORM, SHARED, true, true, false> : kRowsOf<T, FORM, SHARED, true, false, false>;
    FR_TRY(rec_prepare<T>(ctx, a, rows, 64 / across, kWaves, kRowsWindow, parts, ws, &waves));
    const dim3 grid((unsigned)(a.tiles * a.blocks)), block(64 * waves);
    auto launch = [&](auto uniform) {
        constexpr bool U = decltype(uniform)::value;
        if (backward)
            hipLaunchKernelGGL((rec_rows_kernel<T, FORM, V, SHARED, true, U, false>), grid, block, 0, ctx->ls, a);
        else
            hipLaunchKernelGGL((rec_rows_kernel<T, FORM, V, SHARED, false, U, false>), grid, block, 0, ctx->ls, a);
    };
    if (few)
        hipLaunchKernelGGL((rec_rows_kernel<T, FORM, V, SHARED, false, true, true>), grid, block, 0, ctx->ls, a);
    else if constexpr (V == 1) {
        if (a.lanes == 6)
            launch(std::true_type());
        else
            launch(std::false_type());
    } else if constexpr (SHARED || sizeof(T) == 2)  // (two channels of 32 bits with a gate each: few rows only)
        launch(std::true_type());
    return FR_OK;
}

template <typename T, int FORM, int CG>
static int rec_columns(fr_ctx* ctx, RecArgs& a, bool backward, OpWorkspace& ws)
{
    a.pieces = (a.width + CG - 1) / CG;
    a.blocks = a.cols * a.pieces;
    const bool join = backward && a.dgate && a.pieces > 1;
    a.part_r = 1, a.part_c = a.n;
    int waves;
    FR_TRY(rec_prepare<T>(ctx, a, kRowsOfLane, 64, kWaves, kColumnsWindow, join ? a.blocks * a.n : 0, ws, &waves));
    const dim3 grid((unsigned)(a.tiles * a.blocks)), block(64 * waves);
    if (backward)
        hipLaunchKernelGGL((rec_columns_kernel<T, FORM, CG, true>), grid, block, 0, ctx->ls, a);
    else
        hipLaunchKernelGGL((rec_columns_kernel<T, FORM, CG, false>), grid, block, 0, ctx->ls, a);
    return FR_OK;
}

// one row after the other in memory: a single channel of a rows layout is a column
static bool rec_is_column(const RecArgs& a)
{
    return a.d == 1 && a.gate_r == 1 && (!a.x || a.x_r == 1) && (!a.h0 || a.h0_r == 1) && (!a.h || a.h_r == 1) && (!a.last || a.last_r == 1) && (!a.hin || a.h_r == 1) &&
           (!a.dh || a.dh_r == 1) && (!a.dlast || a.dlast_r == 1) && (!a.dgate || a.dg_r == 1) && (!a.dx || a.dx_r == 1) && (!a.dh0 || a.dh0_r == 1);
}

template <typename T, int FORM>
static int rec_launch(fr_ctx* ctx, RecArgs& a, int layout, bool backward, OpWorkspace& ws)
{
    // A lane of 8 bytes of channels fetches fewer, longer lines and works a shared gate out once; a lane of one channel makes more workgroups
    // and keeps more rows' data in flight.  Wide once the call is large enough to fill the chip that way, and for few rows, where the
    // tiles are few either way (bf16, us wide / narrow, shared gate: 4096 x 256 forward 22 / 19, backward 25 / 21; 16384 x 512 26 / 29 and 37 /
    // 48; 16413 x 2048 backward 83 / 168.  A gate a channel: 4096 x 1024 24 / 23 and 33 / 29; 65536 x 256 64 / 56 and 76 / 75; 16384 x 1024
    // 49 / 53 and 64 / 72; 1024 x 2048 forward 17 / 26.  f32, a gate a channel: 16384 x 1024 59 / 54 and 87 / 84, 32768 x 1024
    // 106 / 100 and 152 / 151; shared 16384 x 512 27 / 30 and 41 / 48).
    constexpr int WIDE = 8 / (int)sizeof(T);
    const bool few = !backward && a.n <= kFewRows, fits = WIDE > 1 && a.d >= 64 * WIDE && a.d % WIDE == 0 && (a.width == 1 || a.width % WIDE == 0);
    const bool wide = fits && (few || (a.width > 1 ? a.n * a.d >= 1 << 22 : sizeof(T) == 2 && a.d >= 128 * WIDE && a.n * a.d >= 1 << 23));
    if (layout == FR_LAYOUT_COLMAJOR || rec_is_column(a)) {
        if (a.width == 1)
            FR_TRY((rec_columns<T, FORM, 1>(ctx, a, backward, ws)));
        else if (a.width == 2)
            FR_TRY((rec_columns<T, FORM, 2>(ctx, a, backward, ws)));
        else
            FR_TRY((rec_columns<T, FORM, 4>(ctx, a, backward, ws)));
    } else if (wide) {
        if (a.width == 1)
            FR_TRY((rec_rows<T, FORM, WIDE, false>(ctx, a, backward, ws)));
        else
            FR_TRY((rec_rows<T, FORM, WIDE, true>(ctx, a, backward, ws)));
    } else if (a.width == 1)
        FR_TRY((rec_rows<T, FORM, 1, false>(ctx, a, backward, ws)));
    else
        FR_TRY((rec_rows<T, FORM, 1, true>(ctx, a, backward, ws)));
    if (backward && a.dgate && a.pieces > 1 && a.n > 0)
        hipLaunchKernelGGL((rec_heads_kernel<T>), dim3(blocks_upto(a.n * a.cols)), dim3(256), 0, ctx->ls, a);
    FR_HIP(ctx, hipGetLastError());
    return FR_OK;
}

template <typename T>
int rec_run(fr_ctx* ctx, RecArgs& a, int layout, int form, bool backward, OpWorkspace& ws)
{
    switch (form) {
    case FR_GATE_VALUE: return rec_launch<T, FR_GATE_VALUE>(ctx, a, layout, backward, ws);
    case FR_GATE_LOG: return rec_launch<T, FR_GATE_LOG>(ctx, a, layout, backward, ws);
    default: return rec_launch<T, FR_GATE_STATIONARY>(ctx, a, layout, backward, ws);
    }
}

}  // namespace fr
