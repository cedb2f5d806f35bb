// Filtered sampling of one id per row of logits (include/speaksense.h ss_sample_rows) for gfx950: one workgroup per row.
//
// With max = the row's largest logit and c = log2(e) / t, id i weighs 2^((x_i - max) c), held as an integer W_i = round(w_i 2^S), S = 62 - ceil(log2 n_vocab)
// (at most 51): every sum of a row fits 62 bits and is exact, so neither the order of the atomics nor the split over waves can change a result, and a running
// sum is compared with u times the total exactly.  The exponential is evaluated in double: 2^y = 2^(k/256) 2^r, k = round(256 y), |r| <= 1/512, the first
// factor from a table, the second from its series up to r^4 (the next term is 2e-17).
//
// top-k and top-p are both "keep an id while the measure of the better ones stays below a target", the measure being 1 or W: a histogram over
// 2048 equal steps of the logit finds the step in which the target is crossed, the ids of that step are gathered into LDS and ranked there exactly by
// (logit, id).  A step that holds more ids than the list (equal or crowded logits) is cut again by the bits of its keys until the ids fit or are all
// equal; equal ids are then taken in the order of their number.
#include <algorithm>
#include <type_traits>

#include "ops.h"
#include "wave_ops.h"

namespace ss {
namespace {

typedef unsigned long long u64;
constexpr int kWaves = 16, kThreads = 64 * kWaves, kBins = 2048, kList = 1024;
constexpr float kInf = __builtin_huge_valf();
constexpr unsigned kKeyNegInf = 0x007fffffu;     // order_key(-inf): every masked id has this key or a lower one

__device__ __forceinline__ unsigned order_key(float x) {   // larger number <=> larger key
    const unsigned u = __float_as_uint(x);
    return u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}

struct Entry { unsigned key; int id; u64 w; };
__device__ __forceinline__ bool better(unsigned ka, int ia, unsigned kb, int ib) { return ka > kb || (ka == kb && ia < ib); }

template <typename T> struct Row {
    static constexpr int VEC = 16 / (int)sizeof(T), GROUP = 64 * VEC;
    typedef T V __attribute__((ext_vector_type(VEC), aligned(sizeof(T))));
    const T* p;
    int n, groups;
    bool inf_row;                  // the largest logit is +inf: only those ids count, all alike
    __device__ __forceinline__ float clean(T v) const {
        float x = (float)v + 0.0f;                       // -0 -> +0: equal numbers get equal keys
        x = x != x ? -kInf : x;
        return inf_row ? (x == kInf ? 0.0f : -kInf) : x;
    }
    // this lane's VEC consecutive ids of group g: x[], first id returned; ids behind the row are masked
    __device__ __forceinline__ int load(int g, int lane, float* x) const {
        const int i0 = g * GROUP + lane * VEC;
        if (i0 + VEC <= n) {
            const V v = *(const V*)(p + i0);
#pragma unroll
            for (int e = 0; e < VEC; e++) x[e] = clean(v[e]);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; e++) x[e] = i0 + e < n ? clean(p[i0 + e]) : -kInf;
        }
        return i0;
    }
};

struct Weight {                    // w(x) in double and as an integer
    const double* table;           // LDS: 2^(j/256)
    double max, c, one;            // one = 2^S
    int S;
    __device__ __forceinline__ double scaled(float x) const {            // w 2^S
        const double y = fmax(((double)x - max) * c, -1000.0);
        constexpr double magic = 6755399441055744.0 / 256.0;             // 1.5 2^52 / 256: adding it rounds y to a multiple of 1/256
        const double z = y + magic;
        const int k = (int)(unsigned)__double_as_longlong(z);            // low word of the mantissa: 256 y, rounded, two's complement
        const double r = y - (z - magic);
        constexpr double L1 = 0.693147180559945309417, L2 = 0.240226506959100712333, L3 = 0.0555041086648215799532, L4 = 0.00961812910762847716198;
        const double q = r * (L1 + r * (L2 + r * (L3 + r * L4)));
        const double t = table[k & 255];
        return ldexp(t + t * q, (k >> 8) + S);
    }
    static __device__ __forceinline__ u64 integer(double s) {            // round(s), 0 <= s <= 2^51
        return (u64)__double_as_longlong(s + 4503599627370496.0) & 0x000fffffffffffffull;
    }
};

__device__ __forceinline__ u64 shfl_xor64(u64 v, int o) { return (u64)__shfl_xor((unsigned long long)v, o); }
__device__ __forceinline__ u64 wave_sum64(u64 v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += shfl_xor64(v, o);
    return v;
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
    double table[256];
    u64 hist[kBins];
    Entry list[kList];
    u64 wave64[kWaves + 1];
    float wave_f[3][kWaves];
    int wave_i[kWaves];
    u64 found_base;
    unsigned found_key, key_lo, key_hi;
    int found, found_id, n_list;
};

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_rows_kernel(ss_sample_rows_args a, int S) {
    __shared__ Shared sh;
    extern __shared__ __attribute__((aligned(16))) char dyn[];
    u64* mass = (u64*)dyn;                                               // [groups] measure of each group's kept ids
    typedef Row<T> R;
    constexpr int VEC = R::VEC;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), row = blockIdx.x;
    R r{(const T*)a.logits + (long)row * a.row_stride, a.n_vocab, (a.n_vocab + R::GROUP - 1) / R::GROUP, false};
    for (int i = tid; i < 256; i += kThreads) sh.table[i] = exp2(i * (1.0 / 256.0));

    // the largest logit (lowest id), the smallest unmasked one
    float top = -kInf, low = kInf;
    int best = 0x7fffffff;
    for (int g = wave; g < r.groups; g += kWaves) {
        float x[VEC];
        const int i0 = r.load(g, lane, x);
#pragma unroll
        for (int e = 0; e < VEC; e++) {
            if (x[e] > top) { top = x[e]; best = i0 + e; }
            if (x[e] > -kInf) low = fminf(low, x[e]);
        }
    }
    {
        const float wt = wave_max(top);
        int wb = top == wt ? best : 0x7fffffff;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) wb = min(wb, __shfl_xor(wb, o));
        const float wl = -wave_max(-low);
        if (lane == 0) { sh.wave_f[0][wave] = wt; sh.wave_i[wave] = wb; sh.wave_f[1][wave] = wl; }
    }
    __syncthreads();
    top = -kInf; best = 0x7fffffff; low = kInf;
    for (int w = 0; w < kWaves; w++) {
        const float t = sh.wave_f[0][w];
        const int b = sh.wave_i[w];
        if (t > top) { top = t; best = b; } else if (t == top) best = min(best, b);
        low = fminf(low, sh.wave_f[1][w]);
    }
    if (top == -kInf) {                                                   // every id is masked
        if (tid == 0) {
            a.id[row] = -1;
            if (a.p) a.p[row] = 0.0f;
            if (a.logprob) a.logprob[row] = -kInf;
            if (a.n_kept) a.n_kept[row] = 0;
        }
        return;
    }
    if (top == kInf) { r.inf_row = true; top = low = 0.0f; }

    const float t_row = a.temperature ? a.temperature[row] : 1.0f;
    const bool greedy = !(t_row > 0.0f);
    // an infinite or vanishing t must not meet a difference of 0 or infinity
    const double c = fmax(fmin(1.44269504088896340736 / (greedy ? 1.0 : (double)t_row), 1e300), 1e-300);
    const Weight wt{sh.table, (double)top, c, ldexp(1.0, S), S};
    const int k_row = a.top_k ? a.top_k[row] : 0;
    const float p_row = a.top_p ? a.top_p[row] : 1.0f;
    const bool by_k = !greedy && k_row > 0 && k_row < a.n_vocab, by_p = !greedy && p_row < 1.0f;
    float m_row = a.min_p ? fminf(a.min_p[row], 1.0f) : 0.0f;
    if (a.min_p && !(a.min_p[row] == a.min_p[row])) m_row = 0.0f;
    const bool by_m = !greedy && m_row > 0.0f;
    const double m_scaled = (double)m_row * wt.one;

    // the sum of all weights, for logprob, where the exact total of the kept ones is not that
    double whole = 0.0;
    auto block_sum = [&](float v) {
        const double s = (double)wave_sum(v);
        __syncthreads();
        if (lane == 0) sh.wave64[wave] = (u64)__double_as_longlong(s);
        __syncthreads();
        double z = 0.0;
        for (int w = 0; w < kWaves; w++) z += __longlong_as_double((long long)sh.wave64[w]);
        return z;
    };
    if (a.logprob && (greedy || by_k || by_p || by_m)) {
        float s = 0.0f;
        for (int g = wave; g < r.groups; g += kWaves) {
            float x[VEC];
            r.load(g, lane, x);
#pragma unroll
            for (int e = 0; e < VEC; e++) s += __builtin_amdgcn_exp2f((float)((double)(x[e] - top) * c));
        }
        whole = block_sum(s);
    }
    if (greedy) {
        if (tid == 0) {
            a.id[row] = best;
            if (a.p) a.p[row] = 1.0f;
            if (a.logprob) a.logprob[row] = (float)-log(whole);
            if (a.n_kept) a.n_kept[row] = 1;
        }
        return;
    }
    __syncthreads();                                                      // the table

    unsigned thr = kKeyNegInf;                                            // kept: key > thr, or key == thr and id <= thr_id
    int thr_id = -1;
    auto alive = [&](unsigned key, int id) { return key > thr || (key == thr && id <= thr_id); };
    const float steps = low < top ? (float)(kBins - 1) / (top - low) : 0.0f;
    auto bin_of = [&](float x) { return min((int)((top - x) * steps), kBins - 1); };

    // finds the crossing of `target` in hist (bins in order from the best): bin in sh.found, measure before it in sh.found_base; the total is returned
    auto total_of_hist = [&]() {
        u64 v = sh.hist[2 * tid] + sh.hist[2 * tid + 1];
        v = wave_sum64(v);
        if (lane == 0) sh.wave64[wave] = v;
        __syncthreads();
        u64 t = 0;
        for (int w = 0; w < kWaves; w++) t += sh.wave64[w];
        __syncthreads();
        return t;
    };
    auto cross = [&](u64 base, u64 target) {
        const u64 h0 = sh.hist[2 * tid], h1 = sh.hist[2 * tid + 1];
        const u64 inc = wave_scan64(h0 + h1, lane);
        if (lane == 63) sh.wave64[wave] = inc;
        __syncthreads();
        u64 before = base + inc - (h0 + h1);
        for (int w = 0; w < wave; w++) before += sh.wave64[w];
        if (before < target && target <= before + h0) { sh.found = 2 * tid; sh.found_base = before; }
        before += h0;
        if (before < target && target <= before + h1) { sh.found = 2 * tid + 1; sh.found_base = before; }
        __syncthreads();
    };
    // narrows (thr, thr_id) to the ids whose better ones measure less than the target
    auto select = [&](auto by_mass, u64 count) {
        constexpr bool MASS = decltype(by_mass)::value;
        auto measure = [&](float x) -> u64 { return MASS ? Weight::integer(wt.scaled(x)) : 1; };
        auto fill = [&](auto bin) {                                       // bin(x, key): bin or -1
            __syncthreads();
            sh.hist[2 * tid] = 0; sh.hist[2 * tid + 1] = 0;
            if (tid == 0) { sh.n_list = 0; sh.key_lo = 0xffffffffu; sh.key_hi = 0; sh.found = -1; }
            __syncthreads();
            for (int g = wave; g < r.groups; g += kWaves) {
                float x[VEC];
                const int i0 = r.load(g, lane, x);
#pragma unroll
                for (int e = 0; e < VEC; e++) {
                    const unsigned key = order_key(x[e]);
                    if (!alive(key, i0 + e)) continue;
                    const int b = bin(x[e], key);
                    if (b >= 0) atomicAdd(&sh.hist[b], measure(x[e]));
                }
            }
            __syncthreads();
        };
        auto gather = [&](auto in) {
            for (int g = wave; g < r.groups; g += kWaves) {
                float x[VEC];
                const int i0 = r.load(g, lane, x);
#pragma unroll
                for (int e = 0; e < VEC; e++) {
                    const unsigned key = order_key(x[e]);
                    if (!alive(key, i0 + e) || !in(x[e], key)) continue;
                    const int at = atomicAdd(&sh.n_list, 1);
                    if (at < kList) sh.list[at] = Entry{key, i0 + e, measure(x[e])};
                    atomicMin(&sh.key_lo, key);
                    atomicMax(&sh.key_hi, key);
                }
            }
            __syncthreads();
        };
        fill([&](float x, unsigned) { return bin_of(x); });
        const u64 total = total_of_hist();
        u64 target = count;
        if constexpr (MASS) target = max((u64)1, (u64)ceil((double)fmaxf(p_row, 0.0f) * (double)total));
        if (target >= total) return;                                      // all of them
        cross(0, target);
        int b = sh.found;
        u64 base = sh.found_base;
        gather([&](float x, unsigned) { return bin_of(x) == b; });
        for (;;) {
            const int n = sh.n_list;
            const unsigned lo = sh.key_lo, hi = sh.key_hi;
            __syncthreads();
            if (n <= kList) {
                for (int i = tid; i < n; i += kThreads) {
                    const Entry me = sh.list[i];
                    u64 before = base;
                    for (int j = 0; j < n; j++)
                        if (better(sh.list[j].key, sh.list[j].id, me.key, me.id)) before += sh.list[j].w;
                    if (before < target && target <= before + me.w) { sh.found_key = me.key; sh.found_id = me.id; }
                }
                __syncthreads();
                thr = sh.found_key; thr_id = sh.found_id;
                return;
            }
            if (lo == hi) {                                               // equal logits: the first `need` of them by id
                const float x0 = __uint_as_float(lo & 0x80000000u ? lo ^ 0x80000000u : ~lo);
                const u64 m = measure(x0), need = (target - base + m - 1) / m;
                auto ties = [&](int g) {                                  // this lane's ties of group g
                    float x[VEC];
                    const int i0 = r.load(g, lane, x);
                    int n = 0;
#pragma unroll
                    for (int e = 0; e < VEC; e++) n += order_key(x[e]) == lo && alive(lo, i0 + e);
                    return n;
                };
                for (int g = wave; g < r.groups; g += kWaves) {
                    const u64 n = wave_sum64((u64)ties(g));
                    if (lane == 0) mass[g] = n;
                }
                __syncthreads();
                if (wave == 0) {
                    u64 run = 0;
                    int at = 0;
                    for (; at < r.groups - 1 && run + mass[at] < need; at++) run += mass[at];
                    const u64 mine = (u64)ties(at), inc = run + wave_scan64(mine, lane);
                    if (inc - mine < need && need <= inc) {
                        float x[VEC];
                        const int i0 = r.load(at, lane, x);
                        u64 n = inc - mine;
#pragma unroll
                        for (int e = 0; e < VEC; e++)
                            if (order_key(x[e]) == lo && alive(lo, i0 + e) && ++n == need) sh.found_id = i0 + e;
                    }
                }
                __syncthreads();
                thr = lo; thr_id = sh.found_id;
                return;
            }
            const int shift = max(0, 32 - __clz(hi - lo) - 11);
            fill([&](float, unsigned key) { return key < lo || key > hi ? -1 : (int)((hi - key) >> shift); });
            cross(base, target);
            b = sh.found; base = sh.found_base;
            gather([&](float, unsigned key) { return key >= lo && key <= hi && (int)((hi - key) >> shift) == b; });
        }
    };
    if (by_k) select(std::integral_constant<bool, false>(), (u64)k_row);
    if (by_p) select(std::integral_constant<bool, true>(), 0);

    // the kept ids' weights, group by group
    auto kept = [&](float x, int id, u64* w) {
        if (!alive(order_key(x), id)) return false;
        const double s = wt.scaled(x);
        *w = Weight::integer(s);
        return !by_m || s >= m_scaled;
    };
    __syncthreads();
    u64 total = 0;
    int n_kept = 0;
    for (int g = wave; g < r.groups; g += kWaves) {
        float x[VEC];
        const int i0 = r.load(g, lane, x);
        u64 s = 0;
#pragma unroll
        for (int e = 0; e < VEC; e++) {
            u64 w;
            if (kept(x[e], i0 + e, &w)) { s += w; n_kept++; }
        }
        s = wave_sum64(s);
        if (lane == 0) mass[g] = s;
        total += s;
    }
    n_kept = (int)wave_sum((float)n_kept);                                // < 2^24: exact
    if (lane == 0) { sh.wave64[wave] = total; sh.wave_i[wave] = n_kept; }
    __syncthreads();
    total = 0; n_kept = 0;
    for (int w = 0; w < kWaves; w++) { total += sh.wave64[w]; n_kept += sh.wave_i[w]; }

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
                    const double d = ((double)x[e] - wt.max) * c * 0.693147180559945309417;
                    const double z0 = by_k || by_p || by_m ? whole : (double)total / wt.one;
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
        constexpr int most = (1 << 20) / Row<T>::GROUP * 8;               // beside ~35 KB of static LDS
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
