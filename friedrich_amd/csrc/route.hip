// route.hip -- the router in front of local experts: a score for each expert, the k best of each row, their weights; and its backward pass.
//
// Scores and the order of the experts are worked out in 64 bits whatever the logits' type: which of two experts is taken must not hang on a
// rounding that another program would make otherwise.
#include "kprog_device.hpp"
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
    const void* dweights;
    void* dlogits;
    int64_t l_r, l_c, e_r, e_c, w_r, w_c, dl_r, dl_c;  // element (row, column) at row * _r + column * _c
    int* partial;  // counts of each workgroup, or null: none asked for
    int *again, *agains;  // rows that a workgroup leaves to be done again, `room` each, and their number
    int64_t room;
    // a row is held by 2^lanes lanes, `each` neighbouring experts a lane; in a rows layout they are neighbouring lanes, in a columns layout
    // neighbouring lanes hold neighbouring rows
    int lanes, each;
    bool rows;
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

// how often the rows of a workgroup chose each expert: in LDS, then to memory (counting in memory would send every slot to a few lines)
__device__ __forceinline__ void seen_clear(const RouteArgs& a, int* seen)
{
    if (!a.partial) return;
    for (int e = threadIdx.x; e < a.experts; e += blockDim.x) seen[e] = 0;
    __syncthreads();
}
__device__ __forceinline__ void seen_store(const RouteArgs& a, const int* seen)
{
    if (!a.partial) return;
    __syncthreads();
    for (int e = threadIdx.x; e < a.experts; e += blockDim.x) a.partial[(int64_t)blockIdx.x * a.experts + e] = seen[e];
}
// 16 experts a workgroup, 64 workgroups of the first launch at a time
__global__ __launch_bounds__(1024) void route_counts_kernel(const int* __restrict__ partial, int64_t blocks, int experts, int64_t* __restrict__ counts)
{
    __shared__ int64_t sums[64][17];
    const int c = threadIdx.x & 15, row = threadIdx.x >> 4, e = blockIdx.x * 16 + c;
    int64_t sum = 0;
    if (e < experts)
#pragma unroll 4
        for (int64_t b = row; b < blocks; b += 64) sum += partial[b * experts + e];
    sums[row][c] = sum;
    __syncthreads();
    for (int half = 32; half > 0; half /= 2) {
        if (row < half) sums[row][c] += sums[row + half][c];
        __syncthreads();
    }
    if (row == 0 && e < experts) counts[e] = sums[0][c];
}

// Any number of slots and any groups: one wave holds a row, lane l the experts l, l + 64, ...; the best is found slot by slot.
template <typename T, int J, bool SIGMOID>
__device__ __forceinline__ void route_row(const RouteArgs& a, int64_t row, int* seen)
{
    using W = wide_t<T>;
    const int lane = threadIdx.x & 63;
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
        if (a.partial && mine >= 0) atomicAdd(&seen[mine], 1);
    }
}

template <typename T, int J, bool SIGMOID>
__global__ __launch_bounds__(256) void route_general_kernel(const RouteArgs a)
{
    __shared__ int seen[kRouteMaxExperts];
    seen_clear(a, seen);
    for (int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); row < a.n; row += (int64_t)gridDim.x * 4) route_row<T, J, SIGMOID>(a, row, seen);
    seen_store(a, seen);
}

// ---- up to 8 slots: a few lanes a row --------------------------------------------------------------------------------------------------
//
// Each lane orders its own experts in registers and the lanes of a row merge their lists pairwise.  The order is first worked out from 32-bit
// keys: a key becomes a double, which has 29 bits to spare, and carries its expert's index in its last ten (of equal keys the lower index is
// the larger double), so that exchanging two entries is one maximum and one minimum.  Keys that are logits of 32 bits or less are exact.  Others
// are 2^-19 (1 + |key|) from the 64-bit value or nearer: a row in which two keys that matter lie closer together, or where a key is not finite,
// is left to a second launch, which gives it a wave and orders it in 64 bits.  (64-bit keys throughout took 2430 instructions for four rows of 256 experts, 770 of them
// in the sigmoids, and 157 us for 65536 rows; this takes about 1200, and 84 us with the second launch and the counts.  They issue in just
// under half of the first launch's 68 us: 196 registers leave two waves a SIMD to cover each other's waits, and 226 of the code's 1628 vector
// instructions move spilled scalars.)  A bias that closes an expert makes every row one to be done again: 418 us.

__device__ __forceinline__ double at_bits(unsigned long long b) { return __longlong_as_double((long long)b); }
__device__ __forceinline__ unsigned long long bits_of(double v) { return (unsigned long long)__double_as_longlong(v); }
constexpr double kFar = 0x1p1000;  // stands for an infinity: beyond every 32-bit key, and its last bits are zero

__device__ __forceinline__ int index_of(double key)
{
    const unsigned long long b = bits_of(key);
    return (int)(((int)(b >> 32) >> 31 ^ (int)b ^ 1023) & 1023);
}

// (the instructions by themselves: no NaN comes here, and the compiler would quiet signalling ones before each)
__device__ __forceinline__ double largest(double a, double b)
{
    double r;
    asm("v_max_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
__device__ __forceinline__ double smallest(double a, double b)
{
    double r;
    asm("v_min_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
__device__ __forceinline__ double with_index(float key, int e)
{
    const double v = largest(smallest((double)(key + 0.0f), kFar), -kFar);  // (-0 orders like 0)
    const unsigned long long b = bits_of(v);
    return at_bits(b | (unsigned)(((int)(b >> 32) >> 31 & 1023) ^ (e ^ 1023)));
}
__device__ __forceinline__ void exchange(double& a, double& b)
{
    const double hi = largest(a, b), lo = smallest(a, b);
    a = hi;
    b = lo;
}
template <int K>
__device__ __forceinline__ void order(double (&v)[K])  // descending
{
    if constexpr (K == 2) exchange(v[0], v[1]);
    if constexpr (K == 8) {
        constexpr int N[19][2] = {{0, 2}, {1, 3}, {4, 6}, {5, 7}, {0, 4}, {1, 5}, {2, 6}, {3, 7}, {0, 1}, {2, 3}, {4, 5}, {6, 7}, {2, 4}, {3, 5}, {1, 4}, {3, 6}, {1, 2}, {3, 4}, {5, 6}};
#pragma unroll
        for (int i = 0; i < 19; ++i) exchange(v[N[i][0]], v[N[i][1]]);
    }
}
// the K largest of two descending lists
template <int K>
__device__ __forceinline__ void merge(double (&v)[K], const double (&w)[K])
{
#pragma unroll
    for (int i = 0; i < K; ++i) v[i] = largest(v[i], w[K - 1 - i]);
#pragma unroll
    for (int d = K / 2; d > 0; d /= 2)
#pragma unroll
        for (int i = 0; i < K; ++i)
            if (!(i & d)) exchange(v[i], v[i + d]);
}

// What a lane holds of a row: experts e0 .. e0 + each - 1, -inf behind the last
template <typename T, int C>
struct Held {
    int part, parts, step;  // its place among the row's lanes, their number, and how far apart neighbours are in the wave
    int64_t row;
    int e0, count;
    __device__ __forceinline__ Held(const RouteArgs& a, int64_t turn)
    {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        parts = 1 << a.lanes;
        const int held = 64 >> a.lanes;  // rows of a wave
        part = a.rows ? lane & (parts - 1) : lane >> (6 - a.lanes);
        step = a.rows ? 1 : held;
        row = (turn * 4 + wave) * held + (a.rows ? lane >> a.lanes : lane & (held - 1));
        e0 = part * a.each;
        count = a.experts - e0 < a.each ? a.experts - e0 : a.each;
    }
    // the logits, -inf behind the last expert; rows behind the last read it again
    __device__ __forceinline__ void load(const RouteArgs& a, T (&v)[C]) const
    {
        const T* p = (const T*)a.logits + (row < a.n ? row : a.n - 1) * a.l_r;
        if (a.l_c == 1 && count == C) {
            const Run<T, C> r = load_run<T, C>(p + e0);
#pragma unroll
            for (int c = 0; c < C; ++c) v[c] = r.v[c];
        } else {
#pragma unroll
            for (int c = 0; c < C; ++c) v[c] = p[(int64_t)(c < count ? e0 + c : a.experts - 1) * a.l_c];
#pragma unroll
            for (int c = 0; c < C; ++c) v[c] = c < count ? v[c] : narrow<T>((wide_t<T>)-INFINITY);
        }
    }
    template <typename V>
    __device__ __forceinline__ V lane_sum(V v) const
    {
        for (int i = 1; i < parts; i *= 2) v += __shfl_xor(v, i * step);
        return v;
    }
    template <typename V>
    __device__ __forceinline__ V lane_max(V v) const
    {
        for (int i = 1; i < parts; i *= 2) {
            const V o = __shfl_xor(v, i * step);
            v = o > v ? o : v;
        }
        return v;
    }
    __device__ __forceinline__ bool lane_any(bool v) const
    {
        int w = v;
        for (int i = 1; i < parts; i *= 2) w |= __shfl_xor(w, i * step);
        return w != 0;
    }
    // a value of another lane of the row
    template <typename V>
    __device__ __forceinline__ V from(V v, int p) const
    {
        return __shfl(v, (int)(threadIdx.x & 63) + (p - part) * step);
    }
};

// the score of a logit; top and inverse: of the row, softmax only
template <bool SIGMOID>
__device__ __forceinline__ double score_of(double v, double top, double inverse)
{
    if constexpr (SIGMOID) return 1.0 / (1.0 + exp_fast(-v));
    return top == -INFINITY ? 0.0 : exp_fast(v - top) * inverse;
}

// How many groups are better than the lane's own, from the two largest keys of each lane; near: another group's value lies within `by` of it
template <typename V, typename T, int C>
__device__ __forceinline__ int groups_ahead(const RouteArgs& a, const Held<T, C>& at, V best, V second, V by, bool& near)
{
    const int lanes = a.experts / a.groups / a.each, mine = at.part / lanes;
    for (int i = 1; i < lanes; i *= 2) {
        const V ob = __shfl_xor(best, i * at.step), os = __shfl_xor(second, i * at.step);
        const V low = ob > best ? best : ob, high = os > second ? os : second;
        best = ob > best ? ob : best;
        second = low > high ? low : high;
    }
    const V value = second == -INFINITY ? best : best + second;
    int better = 0;
    for (int g = 0; g < a.groups; ++g) {
        const V v = at.from(value, g * lanes);
        better += v > value || (v == value && g < mine);
        near |= g != mine && v > -INFINITY && fabs(v - value) < by * (V(1) + fabs(value));
    }
    return better;
}

template <typename T, int C, int K, bool SIGMOID>
__global__ __launch_bounds__(256, 2) void route_lists_kernel(const RouteArgs a)
{
    using W = wide_t<T>;
    __shared__ int seen[kRouteMaxExperts];
    __shared__ int agains;
    seen_clear(a, seen);
    if (threadIdx.x == 0) agains = 0;
    __syncthreads();
    const int64_t turns = (a.n + (256 >> a.lanes) - 1) / (256 >> a.lanes);
    const bool grouped = a.top_groups < a.groups;
    const bool scored = a.bias || grouped;  // the order needs the scores
    // Error of a 32-bit score, of at most 1: the exponential is good to 2 ulp and |x| 2^-23 of its argument x, which a sigmoid's slope turns into
    // at most 2^-22 altogether; a softmax adds the rounding of the sum of its up to 16 terms a lane, 2^-20.  Adding a bias rounds twice.  x is a
    // logit (sigmoid, where |x| is paid for by the slope) or its distance from the row's largest, taken in the wide type: that of two
    // rounded logits would be off by a part of the logits, which a row may have as large as it likes.
    constexpr float kNear = SIGMOID ? 0x1p-21f : 0x1p-19f;
    const float near_key = a.bias ? 2.0f * kNear : 0.0f;  // for two keys, times 1 + |key| (f64 logits rounded to 32 bits keep their order)
    const bool exact = sizeof(T) < 8 && !a.bias;
    float bias[C];  // of the lane's experts, the same in every turn
    bool wild = false, rounded = false;  // a bias that 32 bits do not hold at all, or not exactly
    {
        const Held<T, C> at(a, blockIdx.x);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const double b = a.bias ? a.bias[at.e0 + c < a.experts ? at.e0 + c : a.experts - 1] : 0.0;
            bias[c] = (float)b;
            wild |= !(fabs(b) < 1e30);
            rounded |= (double)bias[c] != b;
        }
        rounded = at.lane_any(rounded);
    }
    for (int64_t turn = blockIdx.x; turn < turns; turn += gridDim.x) {
        const Held<T, C> at(a, turn);
        T raw[C];
        at.load(a, raw);
        float key[C];
        W top = -INFINITY;
        bool bad = false;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const W v = widen(raw[c]);
            bad |= v != v;
            top = v > top ? v : top;
            key[c] = (float)v;
        }
        bool odd = wild;
        if constexpr (sizeof(T) == 8)  // (what 32 bits would turn into a closed expert, or into one infinite key among others)
#pragma unroll
            for (int c = 0; c < C; ++c) odd |= isinf(key[c]) && !isinf(raw[c]);
        double inverse = 1.0;
        float about = 1.0f;  // 1 / the sum of exponentials in 32 bits
        if constexpr (!SIGMOID) {
            top = at.lane_max(top);
            bad |= top == (W)INFINITY;
            if (!a.renormalise) {  // weights are shares of all
                double sum = 0.0;
#pragma unroll
                for (int c = 0; c < C; ++c) sum += top > -INFINITY ? exp_fast((double)widen(raw[c]) - (double)top) : 0.0;
                sum = at.lane_sum(sum);
                inverse = sum > 0.0 ? 1.0 / sum : 0.0;
                about = (float)inverse;
            } else if (scored) {
                float sum = 0.0f;
#pragma unroll
                for (int c = 0; c < C; ++c) sum += top > -INFINITY ? __expf((float)(widen(raw[c]) - top)) : 0.0f;
                sum = at.lane_sum(sum);
                about = sum > 0.0f ? 1.0f / sum : 0.0f;
            }
        }
        bad = at.lane_any(bad);
        if (scored) {
            float rank[C], best = -INFINITY, second = -INFINITY;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const float sc = SIGMOID ? __builtin_amdgcn_rcpf(1.0f + __expf(-key[c])) : __expf((float)(widen(raw[c]) - top)) * about;
                rank[c] = key[c] == -INFINITY ? key[c] : sc + bias[c];
                second = fmaxf(second, fminf(best, rank[c]));
                best = fmaxf(best, rank[c]);
            }
            bool kept = true;
            if (grouped) kept = groups_ahead(a, at, best, second, 4 * kNear, odd) < a.top_groups;  // (two keys in a value)
#pragma unroll
            for (int c = 0; c < C; ++c) key[c] = !kept ? -INFINITY : (a.bias ? rank[c] : key[c]);  // (a key may be infinite: nothing is added to it)
        }
        double list[K];
#pragma unroll
        for (int c0 = 0; c0 < C; c0 += K) {
            double next[K];
#pragma unroll
            for (int i = 0; i < K; ++i) next[i] = with_index(c0 + i < C ? key[c0 + i < C ? c0 + i : 0] : -INFINITY, at.e0 + c0 + i);
            order(next);
            if (c0 == 0) {
#pragma unroll
                for (int i = 0; i < K; ++i) list[i] = next[i];
            } else
                merge(list, next);
        }
        for (int d = 1; d < at.parts; d *= 2) {
            double other[K];
#pragma unroll
            for (int i = 0; i < K; ++i) other[i] = __shfl_xor(list[i], d * at.step);
            merge(list, other);
        }
        // lane i of the row takes slot i
        double mine = list[0], last = list[0];
#pragma unroll
        for (int i = 1; i < K; ++i) {
            mine = at.part == i ? list[i] : mine;
            last = a.k - 1 == i ? list[i] : last;
        }
        const bool slot = at.part < a.k;
        int e = !slot || mine <= -kFar ? -1 : index_of(mine);
        const T* logits = (const T*)a.logits + (at.row < a.n ? at.row : a.n - 1) * a.l_r;
        const double v = (double)widen(logits[(int64_t)(e < 0 ? 0 : e) * a.l_c]);
        if (!exact) {
            // two slots too near each other, or an expert behind the last slot too near it -- unless they are alike in logit and bias, and
            // their indices order them
            const float b = a.bias && e >= 0 ? (float)a.bias[e] : 0.0f;
            const int next = at.part + 1 < a.k ? at.part + 1 : at.part, end = a.k - 1;
            const double below = at.from(mine, next), v_below = at.from(v, next), v_last = at.from(v, end);
            const float b_below = at.from(b, next), b_last = at.from(b, end);
            odd |= e >= 0 && next != at.part && !((float)mine - (float)below > near_key * (1.0f + fabsf((float)mine))) && (v != v_below || b != b_below || rounded);
            const float cut = (float)last, low = cut - near_key * (1.0f + fabsf(cut));
            int reach = 0;
#pragma unroll
            for (int c = 0; c < C; ++c) reach += key[c] >= low;
            if (__any(at.lane_sum(reach) > a.k && last > -kFar)) {
                const int e_last = index_of(last);
                bool rival = false;
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    const bool behind = key[c] < cut || (key[c] == cut && at.e0 + c > e_last);
                    rival |= behind && key[c] >= low && key[c] != -INFINITY && ((double)widen(raw[c]) != v_last || bias[c] != b_last || rounded);
                }
                odd |= rival && last > -kFar;
            }
        }
        odd = at.lane_any(odd) && !bad && at.row < a.n;
        if (odd && at.part == 0) a.again[blockIdx.x * a.room + atomicAdd(&agains, 1)] = (int)at.row;  // (in any order: rows are rows)
        const double score = e < 0 ? 0.0 : score_of<SIGMOID>(v, (double)top, inverse);
        const double total = at.lane_sum(score);
        if (at.row < a.n && slot && !odd) {
            const double w = bad ? __builtin_nan("") : a.renormalise ? (total > 0.0 ? score / total : 0.0) : score;
            a.chosen[at.row * a.e_r + at.part * a.e_c] = bad ? -1 : e;
            ((W*)a.weights)[at.row * a.w_r + at.part * a.w_c] = (W)(w * a.scale);
            if (a.partial && e >= 0 && !bad) atomicAdd(&seen[e], 1);
        }
    }
    __syncthreads();
    if (a.agains && threadIdx.x == 0) a.agains[blockIdx.x] = agains;
    seen_store(a, seen);
}

// the rows that a workgroup of the first launch left, counted with its others
template <typename T, int J, bool SIGMOID>
__global__ __launch_bounds__(256) void route_again_kernel(const RouteArgs a)
{
    const int count = a.agains[blockIdx.x];
    for (int i = threadIdx.x >> 6; i < count; i += 4) route_row<T, J, SIGMOID>(a, a.again[blockIdx.x * a.room + i], a.partial ? a.partial + (int64_t)blockIdx.x * a.experts : nullptr);
}

// Each lane writes its experts' gradients as if none of them had been chosen and then, over it, those of the experts that were.  32768 x 128
// bf16, k = 4: 15 to 16 us alone and 14 in a row of calls, 1.3 TB/s of the 17.8 MB that it reads and writes; vector instructions issue in
// two thirds of that, and of the code's 1940 a quarter are moves between registers (the two-address multiply-adds of the series) and a fifth the
// exponentials of the row.  With the slots' number not known when compiled, 1.5 us more.  33 rows of 16: 4 us.
template <typename T, int C, int K, bool SIGMOID>
__global__ __launch_bounds__(256) void route_backward_kernel(const RouteArgs a)
{
    using W = wide_t<T>;
    const Held<T, C> at(a, blockIdx.x);
    T raw[C];
    at.load(a, raw);
    double score[C], top = -INFINITY, inverse = 1.0;
    bool bad = false;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        score[c] = (double)widen(raw[c]);
        bad |= score[c] != score[c];
        top = fmax(top, score[c]);
    }
    const bool dense = !SIGMOID && !a.renormalise;  // every expert's score takes part
    if constexpr (!SIGMOID) {
        top = at.lane_max(top);
        bad |= top == INFINITY;
        if (dense) {
            double sum = 0.0;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                score[c] = top > -INFINITY ? exp_fast(score[c] - top) : 0.0;
                sum += score[c];
            }
            sum = at.lane_sum(sum);
            inverse = sum > 0.0 ? 1.0 / sum : 0.0;
        }
    }
    bad = at.lane_any(bad);
    const int64_t row = at.row < a.n ? at.row : a.n - 1;
    const T* logits = (const T*)a.logits + row * a.l_r;
    const int* chosen = a.chosen + row * a.e_r;
    const W* dweights = (const W*)a.dweights + row * a.w_r;
    double total = 0.0, pull = 0.0;
    int expert[K > 0 ? K : 1];
    double slot[K > 0 ? K : 1], grad[K > 0 ? K : 1];
    if constexpr (K > 0) {  // up to K slots: every lane holds them all
#pragma unroll
        for (int i = 0; i < K; ++i) {
            const int at_i = i < a.k ? i : a.k - 1, e = chosen[at_i * a.e_c];
            grad[i] = a.scale * (double)dweights[at_i * a.w_c];
            expert[i] = i < a.k && e >= 0 && e < a.experts ? e : -1;
        }
        double v[K];
#pragma unroll
        for (int i = 0; i < K; ++i) v[i] = (double)widen(logits[(int64_t)(expert[i] < 0 ? 0 : expert[i]) * a.l_c]);
#pragma unroll
        for (int i = 0; i < K; ++i) {
            slot[i] = expert[i] < 0 ? 0.0 : score_of<SIGMOID>(v[i], top, inverse);
            total += slot[i];
            pull += expert[i] < 0 ? 0.0 : slot[i] * grad[i];
        }
    } else {  // lane i of the row takes slots i, i + parts, ...
        for (int i = at.part; i < a.k; i += at.parts) {
            const int e = chosen[i * a.e_c];
            if (e < 0 || e >= a.experts) continue;
            const double sc = score_of<SIGMOID>((double)widen(logits[(int64_t)e * a.l_c]), top, inverse);
            total += sc;
            pull += sc * (a.scale * (double)dweights[i * a.w_c]);
        }
        total = at.lane_sum(total);
        pull = at.lane_sum(pull);
    }
    // renormalised: dscore_i = (dw_i - sum_j w_j dw_j) / total; softmax adds  - sum_j dscore_j score_j, which is 0 there and `pull` otherwise
    const double mean = a.renormalise ? (total > 0.0 ? pull / total : 0.0) : pull;
    const double by = a.renormalise ? (total > 0.0 ? 1.0 / total : 0.0) : 1.0;
    if (at.row >= a.n || at.count <= 0) return;
    T* out = (T*)a.dlogits + at.row * a.dl_r;
    Run<T, C> r;
#pragma unroll
    for (int c = 0; c < C; ++c) r.v[c] = narrow<T>((W)(bad ? __builtin_nan("") : dense ? -(score[c] * inverse) * mean : 0.0));
    if (a.dl_c == 1 && at.count == C)
        store_run<T, C>(out + at.e0, r);
    else
#pragma unroll
        for (int c = 0; c < C; ++c)
            if (c < at.count) out[(int64_t)(at.e0 + c) * a.dl_c] = r.v[c];
    if (bad) return;
    auto write = [&](int e, double sc, double dw) {
        const double g = SIGMOID ? dw * sc * (1.0 - sc) : sc * (a.renormalise ? dw : dw - mean);
        out[(int64_t)e * a.dl_c] = narrow<T>((W)g);
    };
    // over it, the gradient of all the slots that name an expert, written by the first of them
    if constexpr (K > 0) {
#pragma unroll
        for (int i = 0; i < K; ++i) {
            double dw = 0.0;
            bool first = true;
#pragma unroll
            for (int j = 0; j < K; ++j) {
                const bool alike = expert[j] == expert[i];
                dw += alike ? (a.renormalise ? (grad[j] - mean) * by : grad[j]) : 0.0;
                if (j < i) first = first && !alike;
            }
            if (first && expert[i] >= at.e0 && expert[i] < at.e0 + at.count) write(expert[i], slot[i], dw);
        }
    } else
        for (int i = 0; i < a.k; ++i) {
            const int e = chosen[i * a.e_c];
            if (e < at.e0 || e >= at.e0 + at.count) continue;
            double dw = 0.0;
            bool first = true;
            for (int j = 0; j < a.k; ++j) {
                if (chosen[j * a.e_c] != e) continue;
                first = first && j >= i;
                const double g = a.scale * (double)dweights[j * a.w_c];
                dw += a.renormalise ? (g - mean) * by : g;
            }
            if (first) write(e, score_of<SIGMOID>((double)widen(logits[(int64_t)e * a.l_c]), top, inverse), dw);
        }
}

template <typename T, int J>
static void general_launch(fr_ctx* ctx, const RouteArgs& a, bool sigmoid, dim3 grid)
{
    const dim3 block(256);
    if (sigmoid)
        hipLaunchKernelGGL((route_general_kernel<T, J, true>), grid, block, 0, ctx->ls, a);
    else
        hipLaunchKernelGGL((route_general_kernel<T, J, false>), grid, block, 0, ctx->ls, a);
}
template <typename T, int J>
static void again_launch(fr_ctx* ctx, const RouteArgs& a, bool sigmoid, int64_t grid)
{
    if (sigmoid)
        hipLaunchKernelGGL((route_again_kernel<T, J, true>), dim3((unsigned)grid), dim3(256), 0, ctx->ls, a);
    else
        hipLaunchKernelGGL((route_again_kernel<T, J, false>), dim3((unsigned)grid), dim3(256), 0, ctx->ls, a);
}
template <typename T, int C, bool SIGMOID>
static void lists_launch(fr_ctx* ctx, const RouteArgs& a, bool backward, dim3 grid)
{
    const dim3 block(256);
    if (backward && a.k <= 2)
        hipLaunchKernelGGL((route_backward_kernel<T, C, 2, SIGMOID>), grid, block, 0, ctx->ls, a);
    else if (backward && a.k <= 4)
        hipLaunchKernelGGL((route_backward_kernel<T, C, 4, SIGMOID>), grid, block, 0, ctx->ls, a);
    else if (backward && a.k <= 8)
        hipLaunchKernelGGL((route_backward_kernel<T, C, 8, SIGMOID>), grid, block, 0, ctx->ls, a);
    else if (backward)
        hipLaunchKernelGGL((route_backward_kernel<T, C, 0, SIGMOID>), grid, block, 0, ctx->ls, a);
    else if (a.k <= 2)
        hipLaunchKernelGGL((route_lists_kernel<T, C, 2, SIGMOID>), grid, block, 0, ctx->ls, a);
    else
        hipLaunchKernelGGL((route_lists_kernel<T, C, 8, SIGMOID>), grid, block, 0, ctx->ls, a);
}

template <typename T>
static int route_launch(fr_ctx* ctx, RouteArgs& a, int score, bool backward, int64_t* counts)
{
    const bool sigmoid = score == FR_SCORE_SIGMOID;
    // 16 experts a lane; 4 (and more lanes to merge) where the rows do not give every SIMD a wave otherwise
    a.lanes = backward ? 0 : a.k <= 2 ? 1 : 3;  // (a lane for each slot)
    while (a.experts > (16 << a.lanes)) ++a.lanes;
    if (a.experts <= 256 && (a.n << a.lanes) < (int64_t)ctx->num_cus * 4 * 64)
        while (a.lanes < 6 && a.experts > (4 << a.lanes)) ++a.lanes;
    a.each = (a.experts + (1 << a.lanes) - 1) >> a.lanes;
    const int64_t turns = (a.n + (256 >> a.lanes) - 1) / (256 >> a.lanes);
    // Lists: up to 8 slots, and groups that are whole lanes.  Keys that are not exact need the second launch, which is worth it from 16384 rows
    // on (256 experts, 8 slots, a bias: 8192 rows 38 us against 29 by the general kernel, 32768 rows 49 against 92; without a bias
    // 13 against 15 at 2048 rows and 29 against 93 at 32768).
    bool lists = a.k <= 8;
    if (a.top_groups < a.groups) {
        const int size = a.experts / a.groups, lanes = size / a.each;
        lists = lists && size % a.each == 0 && (lanes & (lanes - 1)) == 0;
    }
    bool second = !backward && (sizeof(T) == 8 || a.bias || a.top_groups < a.groups);
    if (second && a.n < 16384) lists = false;
    second = second && lists;
    int64_t blocks = turns;
    OpWorkspace ws(ctx);
    if (!backward) {
        if (!lists) blocks = (a.n + 3) / 4;
        if (blocks > (int64_t)ctx->num_cus * 4) blocks = (int64_t)ctx->num_cus * 4;  // (what is resident at four waves a SIMD)
        a.room = (turns + blocks - 1) / blocks * (256 >> a.lanes);
        const int64_t counting = counts ? blocks * a.experts : 0, redoing = second ? blocks * (a.room + 1) : 0;
        if (counting + redoing) {
            FR_TRY(ws.get((size_t)(4 * (counting + redoing))));
            if (counts) a.partial = (int*)ws.p;
            if (second) a.agains = (int*)ws.p + counting, a.again = a.agains + blocks;
        }
    }
    const dim3 grid((unsigned)blocks);
    if (!backward && !lists) {
        if (a.experts <= 64)
            general_launch<T, 1>(ctx, a, sigmoid, grid);
        else if (a.experts <= 256)
            general_launch<T, 4>(ctx, a, sigmoid, grid);
        else
            general_launch<T, 16>(ctx, a, sigmoid, grid);
    } else if (a.each <= 4) {
        if (sigmoid)
            lists_launch<T, 4, true>(ctx, a, backward, grid);
        else
            lists_launch<T, 4, false>(ctx, a, backward, grid);
    } else if (sigmoid)
        lists_launch<T, 16, true>(ctx, a, backward, grid);
    else
        lists_launch<T, 16, false>(ctx, a, backward, grid);
    if (second) {
        if (a.experts <= 256)
            again_launch<T, 4>(ctx, a, sigmoid, blocks);
        else
            again_launch<T, 16>(ctx, a, sigmoid, blocks);
    }
    if (!backward && counts) hipLaunchKernelGGL(route_counts_kernel, dim3((unsigned)((a.experts + 15) / 16)), dim3(1024), 0, ctx->ls, a.partial, blocks, a.experts, counts);
    FR_HIP(ctx, hipGetLastError());
    return FR_OK;
}

static int route_dispatch(fr_ctx* ctx, RouteArgs& a, int dtype, int score, bool backward, int64_t* counts = nullptr)
{
    switch (dtype) {
    case FR_F64: return route_launch<double>(ctx, a, score, backward, counts);
    case FR_F32: return route_launch<float>(ctx, a, score, backward, counts);
    case FR_BF16: return route_launch<__hip_bfloat16>(ctx, a, score, backward, counts);
    default: return route_launch<__half>(ctx, a, score, backward, counts);
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
        a.logits = ol.dev, a.bias = ob.as<double>(), a.chosen = oe.as<int>(), a.weights = ow.dev, a.rows = layout == FR_LAYOUT_ROWMAJOR;
        route_strides(layout, ol.ld, a.l_r, a.l_c);
        route_strides(layout, oe.ld, a.e_r, a.e_c);
        route_strides(layout, ow.ld, a.w_r, a.w_c);
        if (n > 0)
            FR_TRY(route_dispatch(ctx, a, dtype, score, false, oc.as<int64_t>()));
        else if (counts)
            hipLaunchKernelGGL(route_counts_kernel, dim3((unsigned)((n_experts + 15) / 16)), dim3(1024), 0, ctx->ls, (const int*)nullptr, (int64_t)0, (int)n_experts, oc.as<int64_t>());
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
        a.logits = ol.dev, a.chosen = oe.as<int>(), a.dweights = ow.dev, a.dlogits = od.dev, a.groups = a.top_groups = 1, a.rows = layout == FR_LAYOUT_ROWMAJOR;
        route_strides(layout, ol.ld, a.l_r, a.l_c);
        route_strides(layout, oe.ld, a.e_r, a.e_c);
        route_strides(layout, ow.ld, a.w_r, a.w_c);
        route_strides(layout, od.ld, a.dl_r, a.dl_c);
        FR_TRY(route_dispatch(ctx, a, dtype, score, true));
        return od.commit();
    });
}

}  // extern "C"
