// Filtered sampling of one id per row of logits (include/speaksense.h ss_sample_rows) for gfx950: one workgroup per row.
//
// With max = the row's largest logit and c = log2(e) / t, id i weighs 2^((x_i - max) c), held as an integer W_i = round(w_i 2^S), S = 62 - ceil(log2 n_vocab)
// (at most 51): every sum of a row fits 62 bits and is exact, so neither the order of the atomics nor the split over waves can change a result, and a running
// sum is compared with u times the total exactly.  The exponential is evaluated in double: 2^y = 2^(k/1024) 2^r, k = round(1024 y), |r| <= 1/2048, the
// first factor from a table, the second from its series up to r^2 (the next term is below 7e-12 of it).
//
// top-k and top-p are both "keep an id while the measure of the better ones stays below a target", the measure being 1 or W: a histogram over
// 2048 equal steps of the logit finds the step in which the target is crossed, the ids of that step are gathered into LDS and ranked there exactly by
// (logit, id).  A step that holds more ids than the list (equal or crowded logits) is cut again by the bits of its keys until the ids fit or are all
// equal; equal ids are then taken in the order of their number.
//
// Passes over the row, which stays in L2 after the first: the largest logit; k up to 512: one more for the ids above a bound; other k and top_p: the histogram and
// the step's ids; a row that a list does not hold: the kept weights.  Bound by the vector instructions of those passes on the one CU that a row has (the double
// exponential and the LDS atomic of an id are some 40 of them: about 13 of the 21 us of a row of 51866), then by its chain of barriers: 51866 float32 logits, 1 row 21 us, 160 rows without a filter 26, with k = 40 26, with
// top_p 0.9 at t = 1 58 (mixed settings 54: 620 GB/s), 512 rows of 128000 bfloat16 85 without a filter (1.5 TB/s), mixed 145.
#include <algorithm>
#include <type_traits>

#include "ops.h"
#include "wave_ops.h"

namespace ss {
namespace {

typedef unsigned long long u64;
constexpr int kThreads = 1024, kWaves = kThreads / 64, kBins = 2048, kList = 1024;
constexpr float kInf = __builtin_huge_valf();
__device__ __forceinline__ unsigned order_key(float x) {   // larger number <=> larger key
    const unsigned u = __float_as_uint(x + 0.0f);           // -0 -> +0: equal numbers get equal keys
    return u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}

struct Entry { unsigned key; int id; u64 w; };
__device__ __forceinline__ bool better(unsigned ka, int ia, unsigned kb, int ib) { return ka > kb || (ka == kb && ia < ib); }

template <typename T> struct Row {
    static constexpr int VEC = 16 / (int)sizeof(T), GROUP = 64 * VEC;
    typedef T V __attribute__((ext_vector_type(VEC), aligned(sizeof(T))));
    const T* p;
    int n, groups;
    // this lane's VEC consecutive ids of group g, as they lie in memory; a lane that the row's end cuts reads nothing here
    __device__ __forceinline__ V fetch(int g, int lane) const {
        const int i0 = g * GROUP + lane * VEC;
        V v{};
        if (i0 + VEC <= n) v = *(const V*)(p + i0);
        return v;
    }
    // their values x[], NaN as it is; ids behind the row are masked; returns the first id
    __device__ __forceinline__ int values(int g, int lane, V v, float* x) const {
        const int i0 = g * GROUP + lane * VEC;
        if (i0 + VEC <= n) {
#pragma unroll
            for (int e = 0; e < VEC; e++) x[e] = (float)v[e];
        } else {
#pragma unroll
            for (int e = 0; e < VEC; e++) x[e] = i0 + e < n ? (float)p[i0 + e] : -kInf;
        }
        return i0;
    }
    __device__ __forceinline__ int load(int g, int lane, float* x) const { return values(g, lane, fetch(g, lane), x); }
};

struct Weight {                    // w(x) 2^S in double and as an integer
    const double* table;           // LDS: 2^(j/1024 + S)
    double top, c, least;          // y = (x - top) c; below `least` (-150 at least) w 2^S is less than 2^-16 and counts as that, which rounds to 0
    __device__ __forceinline__ double scaled(float x) const {
        const double y = fmax(((double)x - top) * c, least);
        constexpr double magic = 6755399441055744.0 / 1024.0;            // 1.5 2^52 / 1024: adding it rounds y to a multiple of 1/1024
        const double z = y + magic;
        const int k = (int)(unsigned)__double_as_longlong(z);            // low word of the mantissa: 1024 y, rounded, two's complement
        const double r = y - (z - magic);
        constexpr double L1 = 0.693147180559945309417, L2 = 0.240226506959100712333;
        const double q = r * fma(r, L2, L1);
        const double t = table[k & 1023];
        const double s = __hiloint2double(__double2hiint(t) + ((k >> 10) << 20), __double2loint(t));  // the exponent: least + S <= k / 1024 + S <= 51
        return fma(s, q, s);
    }
    static __device__ __forceinline__ u64 integer(double s) {            // round(s), 0 <= s <= 2^51
        return (u64)__double_as_longlong(s + 4503599627370496.0) & 0x000fffffffffffffull;
    }
};

template <int CTRL> __device__ __forceinline__ u64 add_dpp64(u64 v) {
    const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)v, CTRL, 0xf, 0xf, false);
    const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)(v >> 32), CTRL, 0xf, 0xf, false);
    return v + ((u64)hi << 32 | lo);
}
__device__ __forceinline__ u64 lane64(u64 v, int l) {
    return (u64)(unsigned)__builtin_amdgcn_readlane((int)(unsigned)(v >> 32), l) << 32 | (unsigned)__builtin_amdgcn_readlane((int)(unsigned)v, l);
}
// on the VALU (a shuffle is a round trip through LDS); the same in every lane
__device__ __forceinline__ u64 wave_sum64(u64 v) {
    v = add_dpp64<kDppRor8>(v);
    v = add_dpp64<kDppRor4>(v);
    v = add_dpp64<kDppXor2>(v);
    v = add_dpp64<kDppXor1>(v);
    return (lane64(v, 0) + lane64(v, 16)) + (lane64(v, 32) + lane64(v, 48));
}
__device__ __forceinline__ u64 wave_scan64(u64 v, int lane) {            // inclusive
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const u64 t = (u64)__shfl_up((unsigned long long)v, o);
        if (lane >= o) v += t;
    }
    return v;
}

struct Shared {
    double table[1024];
    u64 hist[kBins];
    Entry list[kList];             // the ids of the step in which a target is crossed
    Entry kept[kList];             // the ids of that step and of the better ones, if they fit
    u64 wave64[kWaves];
    float wave_f[2][kWaves];
    u64 found_base;
    unsigned found_key, key_lo, key_hi;
    int found, found_id, n_list, n_kept, best;
};

// 1024 threads a row: with 512, two rows a CU, 8 rows of 51866 take 27 us instead of 22, 160 filtered rows 75 instead of 54, 512 of 128000 193 instead of 157;
// only rows without a filter gain (512 of 128000: 77 against 83).
template <typename T>
__global__ __launch_bounds__(kThreads) void sample_rows_kernel(ss_sample_rows_args a, int S) {
    constexpr int THREADS = kThreads, WAVES = kWaves, BPT = kBins / THREADS;
    static_assert(kList == THREADS, "one candidate a thread");
    __shared__ Shared sh;
    extern __shared__ __attribute__((aligned(16))) char dyn[];
    u64* mass = (u64*)dyn;                                               // [groups] measure of each group's kept ids
    typedef Row<T> R;
    constexpr int VEC = R::VEC, AHEAD = 4;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), row = blockIdx.x;
    R r{(const T*)a.logits + (long)row * a.row_stride, a.n_vocab, (a.n_vocab + R::GROUP - 1) / R::GROUP};

    // f(group, first id of the lane, its VEC logits) over the wave's groups, the loads of the next AHEAD groups in flight.  f appears once in a rolled
    // loop: a workgroup runs through its code only a few times, and instruction fetches cost more than the moves between the buffers.
    // (inlined by force, as the passes below: a call keeps this kernel's variables in memory, 55 us for one row of 128000 instead of 35)
    auto over_row = [&](auto f) __attribute__((always_inline)) {
        typename R::V v[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; i++) v[i] = r.fetch(wave + i * WAVES, lane);
#pragma unroll 1
        for (int g = wave; g < r.groups; g += WAVES) {
            float x[VEC];
            const int i0 = r.values(g, lane, v[0], x);
#pragma unroll
            for (int i = 0; i + 1 < AHEAD; i++) v[i] = v[i + 1];
            v[AHEAD - 1] = r.fetch(g + AHEAD * WAVES, lane);
            f(g, i0, x);
        }
    };

    // the largest logit; the smallest unmasked one of a sample (it only scales the histograms' steps)
    float mine = -kInf, low = kInf;
    over_row([&](int g, int, const float* x) {
#pragma unroll
        for (int e = 0; e < VEC; e++) mine = fmaxf(mine, x[e]);          // passes over NaN
        if (g == wave)
#pragma unroll
            for (int e = 0; e < VEC; e++) low = fminf(low, x[e] > -kInf ? x[e] : kInf);
    });
    for (int i = tid; i < 1024; i += THREADS) sh.table[i] = exp2(i * (1.0 / 1024.0) + S);
    {
        const float wt = wave_max(mine), wl = -wave_max(-low);
        if (lane == 0) { sh.wave_f[0][wave] = wt; sh.wave_f[1][wave] = wl; }
        if (tid == 0) sh.best = 0x7fffffff;
    }
    __syncthreads();
    float top = -kInf;
    low = kInf;
    for (int w = 0; w < WAVES; w++) { top = fmaxf(top, sh.wave_f[0][w]); low = fminf(low, sh.wave_f[1][w]); }
    if (top == -kInf) {                                                   // every id is masked
        if (tid == 0) {
            a.id[row] = -1;
            if (a.p) a.p[row] = 0.0f;
            if (a.logprob) a.logprob[row] = -kInf;
            if (a.n_kept) a.n_kept[row] = 0;
        }
        return;
    }
    auto block_sum64 = [&](u64 v) {
        v = wave_sum64(v);
        __syncthreads();
        if (lane == 0) sh.wave64[wave] = v;
        __syncthreads();
        u64 t = 0;
        for (int w = 0; w < WAVES; w++) t += sh.wave64[w];
        __syncthreads();
        return t;
    };
    // one wave: the id at place `need` (from 1) among the ids that `is` says yes to, counted in order of id; mass[] holds their number in each group
    auto nth = [&](u64 need, auto is) {
        u64 run = 0;
        int at = 0;
        for (; at < r.groups - 1 && run + mass[at] < need; at++) run += mass[at];
        float x[VEC];
        const int i0 = r.load(at, lane, x);
        u64 n = 0;
#pragma unroll
        for (int e = 0; e < VEC; e++) n += is(x[e], i0 + e);
        const u64 inc = run + wave_scan64(n, lane);
        if (inc - n < need && need <= inc) {
            n = inc - n;
#pragma unroll
            for (int e = 0; e < VEC; e++)
                if (is(x[e], i0 + e) && ++n == need) sh.found_id = i0 + e;
        }
    };
    auto count_groups = [&](auto is) __attribute__((always_inline)) {
        over_row([&](int g, int i0, const float* x) {
            u64 n = 0;
#pragma unroll
            for (int e = 0; e < VEC; e++) n += is(x[e], i0 + e);
            n = wave_sum64(n);
            if (lane == 0) mass[g] = n;
        });
        __syncthreads();
    };

    const float t_row = a.temperature ? a.temperature[row] : 1.0f;
    const bool greedy = !(t_row > 0.0f);
    // an infinite or vanishing t must not meet a difference of 0 or infinity
    const double c = fmax(fmin(1.44269504088896340736 / (greedy ? 1.0 : (double)t_row), 1e300), 1e-300);
    const double one = ldexp(1.0, S);
    Weight wt{sh.table, (double)top, c, -(double)(S + 16)};
    const int k_row = a.top_k ? a.top_k[row] : 0;
    const float p_row = a.top_p ? a.top_p[row] : 1.0f;
    const bool by_k = !greedy && k_row > 0 && k_row < a.n_vocab, by_p = !greedy && p_row < 1.0f;
    float m_row = a.min_p ? fminf(a.min_p[row], 1.0f) : 0.0f;
    if (a.min_p && !(a.min_p[row] == a.min_p[row])) m_row = 0.0f;
    const bool by_m = !greedy && m_row > 0.0f;
    const double m_scaled = (double)m_row * one;
    if (by_m) wt.least = fmin(wt.least, log2((double)m_row) - 1.0);      // weights around min_p have to be told apart, however small it is

    // the sum of all weights, for logprob: of float32 exponentials where some pass goes over the whole row and needs no exact ones, else exact
    float part = 0.0f;
    double whole = 0.0;
    bool summed = false;
    const float cf = (float)c;
    const bool plain = c > 1e-30 && c < 1e30;                             // float32 takes it
    auto add_parts = [&](const float* x) {                                // NaN counts as masked: fmaxf passes over it
        if (plain)
#pragma unroll
            for (int e = 0; e < VEC; e++) part += __builtin_amdgcn_exp2f(fmaxf((x[e] - top) * cf, -kInf));
        else
#pragma unroll
            for (int e = 0; e < VEC; e++) part += __builtin_amdgcn_exp2f(fmaxf((float)((double)(x[e] - top) * c), -kInf));
    };
    auto sum_parts = [&]() {
        const double s = (double)wave_sum(part);
        __syncthreads();
        if (lane == 0) sh.wave64[wave] = (u64)__double_as_longlong(s);
        __syncthreads();
        whole = 0.0;
        for (int w = 0; w < WAVES; w++) whole += __longlong_as_double((long long)sh.wave64[w]);
        __syncthreads();
    };
    if (top == kInf) {                                                    // ids at +inf share all weight, the others are masked
        auto is = [&](float x, int) { return x == kInf; };
        u64 n = 0;
        count_groups(is);
        for (int g = tid; g < r.groups; g += THREADS) n += mass[g];
        n = block_sum64(n);
        u64 m = greedy ? 1 : by_k ? min(n, (u64)k_row) : n;
        if (by_p) m = max((u64)1, (u64)ceil((double)fmaxf(p_row, 0.0f) * (double)m));
        const double u = a.u[row];
        const u64 j = !greedy && u > 0.0 ? (u64)fmin(u * (double)m, (double)m) : 0;
        if (wave == 0) nth(min(j, m - 1) + 1, is);
        __syncthreads();                                                  // some lane has left found_id
        if (tid == 0) {
            a.id[row] = sh.found_id;
            if (a.p) a.p[row] = (float)(1.0 / (double)m);
            if (a.logprob) a.logprob[row] = (float)-log((double)n);
            if (a.n_kept) a.n_kept[row] = (int)m;
        }
        return;
    }
    if (greedy) {
        over_row([&](int, int i0, const float* x) {
            if (a.logprob) add_parts(x);
#pragma unroll
            for (int e = 0; e < VEC; e++)
                if (x[e] == top) atomicMin(&sh.best, i0 + e);
        });
        if (a.logprob) sum_parts();
        __syncthreads();
        if (tid == 0) {
            a.id[row] = sh.best;
            if (a.p) a.p[row] = 1.0f;
            if (a.logprob) a.logprob[row] = (float)-log(whole);
            if (a.n_kept) a.n_kept[row] = 1;
        }
        return;
    }

    float thr = -kInf;                                                    // kept: x > thr, or x == thr and id <= thr_id
    int thr_id = -1;
    auto alive = [&](float x, int id) { return x > thr || (x == thr && id <= thr_id); };
    // (a span beyond 64 is the work of a mask of some lowest number: the histogram's steps are for the logits above it.
    // With 2 % of the ids at float32's lowest and steps up to it, k = 40 of 160 rows took 141 us instead of 26)
    low = low < top ? fmaxf(low, top - 64.0f) : top - 64.0f;              // (the sample may be all masked)
    const float steps = low < top ? (float)(kBins - 1) / (top - low) : 0.0f;
    auto bin_of = [&](float x) { return (int)fminf(fmaxf((top - x) * steps, 0.0f), (float)(kBins - 1)); };   // NaN: 0
    auto value_of = [&](unsigned key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); };

    // counts need 32 bits of a bin: half the LDS traffic
    auto bin_at = [&](auto by_mass, int i) -> u64 { return decltype(by_mass)::value ? sh.hist[i] : (u64)((const unsigned*)sh.hist)[i]; };
    auto add = [&](auto by_mass, int bin, float x) {
        if constexpr (decltype(by_mass)::value) atomicAdd(&sh.hist[bin], Weight::integer(wt.scaled(x)));
        else atomicAdd((unsigned*)sh.hist + bin, 1u);
    };
    auto clear = [&]() {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < BPT; i++) sh.hist[BPT * tid + i] = 0;
        if (tid == 0) { sh.n_list = 0; sh.key_lo = 0xffffffffu; sh.key_hi = 0; sh.found = -1; }
        __syncthreads();
    };
    auto my_bins = [&](auto by_mass) {
        u64 s = 0;
#pragma unroll
        for (int i = 0; i < BPT; i++) s += bin_at(by_mass, BPT * tid + i);
        return s;
    };
    // finds the crossing of `target` in hist (bins in order from the best): bin in sh.found, measure before it in sh.found_base
    auto cross = [&](auto by_mass, u64 base, u64 target) {
        const u64 own = my_bins(by_mass), inc = wave_scan64(own, lane);
        if (lane == 63) sh.wave64[wave] = inc;
        __syncthreads();
        u64 before = base + inc - own;
        for (int w = 0; w < wave; w++) before += sh.wave64[w];
#pragma unroll
        for (int i = 0; i < BPT; i++) {
            const u64 h = bin_at(by_mass, BPT * tid + i);
            if (before < target && target <= before + h) { sh.found = BPT * tid + i; sh.found_base = before; }
            before += h;
        }
        __syncthreads();
    };
    const std::integral_constant<bool, false> by_count{};
    const std::integral_constant<bool, true> by_mass{};

    bool listed = false;               // sh.kept holds every id that is still kept (and others, that `alive` rules out)
    // the ids of the histogram's steps 0 .. b - 1 into sh.kept, those of step b into sh.list with their measure.  Almost every id falls to one comparison
    // with a bound below them all
    auto list_steps = [&](auto mode, int b) __attribute__((always_inline)) {
        // (b + 1) / steps and what float32 may be off; the last step holds all that lies below it too
        const float reach = b >= kBins - 1 ? -kInf : top - (float)(b + 2) / steps - fabsf(top) * 4e-7f - 1e-37f;
        __syncthreads();
        if (tid == 0) { sh.n_kept = 0; sh.n_list = 0; sh.key_lo = 0xffffffffu; sh.key_hi = 0; }
        __syncthreads();
        unsigned key_lo = 0xffffffffu, key_hi = 0;
        const bool sum = a.logprob && by_k && !summed;
        over_row([&](int, int i0, const float* x) {
            if (sum) add_parts(x);
            float m = x[0];
#pragma unroll
            for (int e = 1; e < VEC; e++) m = fmaxf(m, x[e]);
            if (!__ballot(m >= reach)) return;
            const bool full = *(volatile int*)&sh.n_kept > kList;         // of no use any more
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                if (!(x[e] >= reach && x[e] > -kInf)) continue;
                const int bin = bin_of(x[e]);
                const unsigned key = order_key(x[e]);
                if (bin == b) {
                    const int at = atomicAdd(&sh.n_list, 1);
                    if (at < kList) sh.list[at] = Entry{key, i0 + e, decltype(mode)::value ? Weight::integer(wt.scaled(x[e])) : 1};
                    key_lo = min(key_lo, key);
                    key_hi = max(key_hi, key);
                } else if (bin < b && !full) {
                    const int at = atomicAdd(&sh.n_kept, 1);
                    if (at < kList) sh.kept[at] = Entry{key, i0 + e, 0};
                }
            }
        });
        if (key_lo <= key_hi) { atomicMin(&sh.key_lo, key_lo); atomicMax(&sh.key_hi, key_hi); }
        if (sum) { sum_parts(); summed = true; }
        __syncthreads();
    };
    // narrows (thr, thr_id) to the ids whose better ones measure less than the target, from sh.kept or from the row.  target 0: top_p of the measure's total.
    // `complete`: the source holds every id that (thr, thr_id) keeps, so that there may be nothing to narrow.  b >= 0: the target is known to be crossed
    // in step b, `base` lies before it
    auto select = [&](auto mode, auto from_list, u64 target, bool complete, int b, u64 base) __attribute__((always_inline)) {
        constexpr bool MASS = decltype(mode)::value, LIST = decltype(from_list)::value;
        auto measure = [&](float x) -> u64 { return MASS ? Weight::integer(wt.scaled(x)) : 1; };
        const int n_from = LIST ? sh.n_kept : 0;
        auto each = [&](auto f) __attribute__((always_inline)) {                                         // f(logit, id) of every id still kept
            if constexpr (LIST) {
                for (int i = tid; i < n_from; i += THREADS) {
                    const float x = value_of(sh.kept[i].key);
                    if (alive(x, sh.kept[i].id)) f(x, sh.kept[i].id);
                }
            } else
                over_row([&](int, int i0, const float* x) {
#pragma unroll
                    for (int e = 0; e < VEC; e++)
                        if (alive(x[e], i0 + e)) f(x[e], i0 + e);
                });
        };
        auto take = [&](float x, int id) {                                // into the list of candidates
            const unsigned key = order_key(x);
            const int at = atomicAdd(&sh.n_list, 1);
            if (at < kList) sh.list[at] = Entry{key, id, measure(x)};
            atomicMin(&sh.key_lo, key);
            atomicMax(&sh.key_hi, key);
        };
        if (b < 0) {
            clear();
            each([&](float x, int) { add(mode, bin_of(x), x); });
            __syncthreads();
            const u64 total = block_sum64(my_bins(mode));
            if (target == 0) target = max((u64)1, (u64)ceil((double)fmaxf(p_row, 0.0f) * (double)total));
            if (target >= total && complete) return;
            target = min(target, total);
            cross(mode, 0, target);
            b = sh.found; base = sh.found_base;
        }
        const bool fresh = thr == -kInf;                                  // nothing is ruled out yet: the row's steps are what is kept
        if (!LIST && fresh) list_steps(mode, b);
        else {
            each([&](float x, int id) { if (bin_of(x) == b) take(x, id); });
            __syncthreads();
        }
        for (bool first = true;; first = false) {
            const int n = sh.n_list;
            const unsigned lo = sh.key_lo, hi = sh.key_hi;
            __syncthreads();
            if (n <= kList) {
                // rank them: 64 ids a wave, the ids that they are compared with shared out over the waves that are left (512 rows of 128000: 157 -> 145 us)
                sh.hist[tid] = 0;
                const int per = (n + 63) / 64, parts = WAVES / per, part = wave / per, i = (wave - part * per) * 64 + lane;
                __syncthreads();
                if (part < parts && i < n) {
                    const Entry me = sh.list[i];
                    u64 before = 0;
                    for (int j = part; j < n; j += parts)
                        if (better(sh.list[j].key, sh.list[j].id, me.key, me.id)) before += sh.list[j].w;
                    atomicAdd(&sh.hist[i], before);
                }
                __syncthreads();
                if (tid < n) {
                    const Entry me = sh.list[tid];
                    const u64 before = base + sh.hist[tid];
                    if (before < target && target <= before + me.w) { sh.found_key = me.key; sh.found_id = me.id; }
                }
                __syncthreads();
                thr = value_of(sh.found_key); thr_id = sh.found_id;
                if (!LIST && fresh && first) {                            // the candidates that stay join the better steps
                    for (int i = tid; i < n; i += THREADS)
                        if (alive(value_of(sh.list[i].key), sh.list[i].id)) {
                            const int at = atomicAdd(&sh.n_kept, 1);
                            if (at < kList) sh.kept[at] = sh.list[i];
                        }
                    __syncthreads();
                    listed = sh.n_kept <= kList;
                }
                return;
            }
            if constexpr (LIST) return;                                   // never: a list's ids fit
            if (lo == hi) {                                               // equal logits: the first `need` of them by id
                const float tie = value_of(lo);
                const u64 m = measure(tie), need = (target - base + m - 1) / m;
                auto is = [&](float x, int id) { return x == tie && alive(tie, id); };
                count_groups(is);
                if (wave == 0) nth(need, is);
                __syncthreads();
                thr = tie; thr_id = sh.found_id;
                return;
            }
            const int shift = max(0, 32 - __clz(hi - lo) - 11);
            auto in_reach = [&](auto f) {                                 // f(logit, id, key) of the kept ids with keys from lo to hi.  One id at a time: rare
#pragma unroll 1
                for (int i = tid; i < r.n; i += THREADS) {
                    const float x = (float)r.p[i];
                    const unsigned key = order_key(x);
                    if (key >= lo && key <= hi && alive(x, i)) f(x, i, key);
                }
            };
            clear();
            in_reach([&](float x, int, unsigned key) { add(mode, (int)((hi - key) >> shift), x); });
            __syncthreads();
            cross(mode, base, target);
            b = sh.found; base = sh.found_base;
            in_reach([&](float x, int id, unsigned key) { if ((int)((hi - key) >> shift) == b) take(x, id); });
            __syncthreads();
        }
    };
    const std::integral_constant<bool, true> from_list{};
    const std::integral_constant<bool, false> from_row{};
    if (by_k) {
        // the k-th largest of the threads' largest logits bounds the k-th largest of all from below.  For k of half the threads about 0.7 THREADS ids of a
        // random row lie above it: the list takes them, and they are all that is looked at from here on
        if (2 * k_row <= THREADS) {
            clear();
            if (mine > -kInf) add(by_count, bin_of(mine), mine);
            __syncthreads();
            if (block_sum64(my_bins(by_count)) >= (u64)k_row) {
                cross(by_count, 0, (u64)k_row);
                list_steps(by_count, sh.found + 1);
                listed = sh.n_kept <= kList;
            }
        }
        if (listed) select(by_count, from_list, (u64)k_row, false, -1, 0);
        else select(by_count, from_row, (u64)k_row, true, -1, 0);
    }
    if (by_p) {
        if (listed) select(by_mass, from_list, 0, true, -1, 0);
        else if (by_k) select(by_mass, from_row, 0, true, -1, 0);
        else {
            // masked ids and NaN weigh 0: no test
            clear();
            over_row([&](int, int, const float* x) {
#pragma unroll
                for (int e = 0; e < VEC; e++) add(by_mass, bin_of(x[e]), x[e]);
            });
            __syncthreads();
            const u64 total = block_sum64(my_bins(by_mass)), target = max((u64)1, (u64)ceil((double)fmaxf(p_row, 0.0f) * (double)total));
            whole = (double)total / one;
            if (target < total) {
                cross(by_mass, 0, target);
                select(by_mass, from_row, target, true, sh.found, sh.found_base);
            }
        }
    }

    // the kept ids' weights, group by group
    auto kept = [&](float x, int id, u64* w) {
        if (!alive(x, id)) return false;
        const double s = wt.scaled(x);
        *w = Weight::integer(s);
        return !by_m || s >= m_scaled || x == top;
    };
    __syncthreads();
    u64 total = 0;
    int n_kept = 0;
    if (listed) {
        for (int g = tid; g < r.groups; g += THREADS) mass[g] = 0;
        __syncthreads();
        for (int i = tid; i < sh.n_kept; i += THREADS) {
            const Entry e = sh.kept[i];
            u64 w;
            if (kept(value_of(e.key), e.id, &w)) { total += w; n_kept++; atomicAdd(&mass[e.id / R::GROUP], w); }
        }
    } else {
        const bool add_whole = a.logprob && !summed && (by_k || (by_m && !by_p)), plain_row = !by_k && !by_p && !by_m;
        over_row([&](int g, int i0, const float* x) {
            u64 s = 0;
            if (add_whole) add_parts(x);
            if (plain_row) {                                              // masked ids and NaN weigh 0
#pragma unroll
                for (int e = 0; e < VEC; e++) { s += Weight::integer(wt.scaled(x[e])); n_kept += x[e] > -kInf; }
            } else {
#pragma unroll
                for (int e = 0; e < VEC; e++) {
                    u64 w;
                    if (kept(x[e], i0 + e, &w)) { s += w; n_kept++; }
                }
            }
            total += s;
            s = wave_sum64(s);
            if (lane == 0) mass[g] = s;
        });
        if (add_whole) sum_parts();
    }
    total = block_sum64(total);
    n_kept = (int)block_sum64((u64)n_kept);

    if (wave != 0) return;
    const double u = a.u[row];
    u64 target = u > 0.0 ? (u64)fmin(u * (double)total, (double)total) : 0;
    if (target >= total) target = total - 1;                              // drawn: the first id whose running sum exceeds target
    u64 run = 0;
    int at = 0;
    for (int g0 = 0; g0 < r.groups; g0 += 64) {                           // 64 groups a step
        const u64 m = g0 + lane < r.groups ? mass[g0 + lane] : 0, inc = run + wave_scan64(m, lane);
        const u64 hit = __ballot(inc > target);
        if (hit) {
            const int l = __ffsll((unsigned long long)hit) - 1;
            at = g0 + l;
            run = (u64)__shfl((unsigned long long)(inc - m), l);
            break;
        }
        run = (u64)__shfl((unsigned long long)inc, 63);
    }
    float x[VEC];
    const int i0 = r.load(at, lane, x);
    u64 w[VEC], s = 0;
#pragma unroll
    for (int e = 0; e < VEC; e++) {
        if (!kept(x[e], i0 + e, &w[e])) w[e] = 0;
        s += w[e];
    }
    const u64 inc = run + wave_scan64(s, lane);
    if (inc > target && inc - s <= target) {
        u64 z = inc - s;
        bool done = false;
#pragma unroll
        for (int e = 0; e < VEC; e++) {
            z += w[e];
            if (!done && z > target) {
                done = true;
                a.id[row] = i0 + e;
                if (a.p) a.p[row] = (float)((double)w[e] / (double)total);
                if (a.logprob) {
                    const double d = ((double)x[e] - (double)top) * c * 0.693147180559945309417;
                    const double z0 = by_k || by_p || by_m ? whole : (double)total / one;
                    a.logprob[row] = (float)(d - log(z0));
                }
                if (a.n_kept) a.n_kept[row] = n_kept;
            }
        }
    }
}

}  // namespace

void launch_sample_rows(const ss_sample_rows_args& a, hipStream_t st) {
    if (a.n_rows == 0) return;
    int bits = 0;
    while ((1 << bits) < a.n_vocab) bits++;
    const int S = std::min(51, 62 - bits);
    auto go = [&](auto t) {
        typedef decltype(t) T;
        const int groups = (a.n_vocab + Row<T>::GROUP - 1) / Row<T>::GROUP;
        constexpr int most = (1 << 20) / Row<T>::GROUP * 8;
        static_assert(sizeof(Shared) + most <= 160 * 1024, "LDS of a workgroup: 57,648 bytes and 8 a group");
        static std::atomic<uint64_t> once{0};
        once_per_device(once, [&] { SS_HIP(hipFuncSetAttribute((const void*)sample_rows_kernel<T>, hipFuncAttributeMaxDynamicSharedMemorySize, most)); });
        sample_rows_kernel<T><<<a.n_rows, kThreads, (size_t)groups * 8, st>>>(a, S);
    };
    if (a.dtype == SS_DTYPE_F32) go(0.0f);
    else if (a.dtype == SS_DTYPE_F16) go(f16());
    else go(bf16());
    SS_LAUNCH_CHECK();
}

}  // namespace ss
