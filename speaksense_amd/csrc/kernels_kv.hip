// Paged key / value cache for gfx950: append with quantisation, read back, attention of a chunk of new tokens.
//
// Cache of one layer: k and v are [n_pages][n_kv_heads][page_size][head_dim] codes, one scale per (page, head, row) beside 8-bit codes:
//   same   f16 / bf16 as the tokens
//   e4m3   code = RNE_e4m3(x 2^(127 - e)), e = E8M0 byte with amax / 2^(e - 127) <= 448 (the format of the fp8 engine's cross cache)
//   int8   s = amax / 127 (IEEE), code = rint(x / s)
// A row with an infinity (and no NaN): its infinities hold the largest code under the exponent 253 (448 2^126 is an infinity) or the scale s = infinity (code 0
// of the finite elements times that is a NaN).
// A sequence s of the step has n_s = q_start[s + 1] - q_start[s] new tokens, the last n_s of its kv_len[s] positions; position p lies in row
// p % page_size of page page_table[s][p / page_size].  Every index that comes from device memory is checked here before it is used: a page number
// outside [0, n_pages) holds nothing (its keys are masked, reads give zeros, writes are dropped), spans of q_start outside the token rows are empty.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "gemm_common.h"
#include "ops.h"
#include "wave_ops.h"

namespace ss {
namespace {

// LDS of the tile kernel: pitches of a key and of a value row (16-bit elements), bytes of one stage.  The 16 key rows that a wave's lanes read 16 bytes of
// each start on 16 different groups of 4 banks, the 8 value rows that 32 lanes read 32 bytes of on 8 different groups of 8.
template <int D> constexpr int kKeyPitch = 2 * D + 16;
template <int D> constexpr int kValuePitch = 2 * D + 32;
template <int D> constexpr int kTileBuf = 64 * (kKeyPitch<D> + kValuePitch<D>) + 528;   // + 64 key scales, 64 relative value scales, sref, its move

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

enum { K_F16 = 0, K_BF16 = 1, K_E4M3 = 2, K_I8 = 3 };   // what the cache holds

struct KvArgs {
    char *k, *v, *ks, *vs;
    unsigned page_bytes, sc_stride;      // between pages: bytes of codes, elements of scales (the host has checked that they fit)
    const int *table, *q_start, *kv_len;
    long table_stride;
    int n_pages, page_shift, H, max_pages, n_seqs, n_tokens;
};

// a + page * pitch: one multiply-add of 32 x 32 + 64 bits
__device__ __forceinline__ char* page_ptr(char* a, int page, unsigned pitch) { return a + (unsigned long)(unsigned)page * pitch; }

struct Span { int q0, n_new, len, pos0; };   // first token row, new tokens, positions held, position of the first new token
__device__ __forceinline__ Span seq_span(const KvArgs& a, int s) {
    Span r;
    r.q0 = a.q_start[s];
    const int q1 = a.q_start[s + 1];
    r.n_new = r.q0 >= 0 && q1 > r.q0 && q1 <= a.n_tokens ? q1 - r.q0 : 0;
    const int held = max(a.kv_len[s], 0);
    r.len = min(held, a.max_pages << a.page_shift);      // the host has checked that the product fits 31 bits
    r.pos0 = held - r.n_new;
    return r;
}
__device__ __forceinline__ int page_at(const KvArgs& a, int s, int page) {   // page index inside the sequence -> page of the cache, or -1
    if (page < 0 || page >= a.max_pages) return -1;
    const int p = a.table[(long)s * a.table_stride + page];
    return p < 0 || p >= a.n_pages ? -1 : p;
}
// The sequence of token row t: 64 boundaries a step.  Any contents of q_start give an index in [-1, n_seqs]; the caller checks the span itself.
__device__ __forceinline__ int find_seq(const int* qs, int n_seqs, int t) {
    const int lane = threadIdx.x & 63;
    int lo = 0, len = n_seqs + 1;
    while (len > 64) {
        const int step = (len + 63) >> 6, i = (lane + 1) * step - 1;
        const bool below = i < len && qs[lo + i] <= t;
        const int c = __popcll(__ballot(below));
        lo += c * step;
        len = min(step, len - c * step);
    }
    const bool below = lane < len && qs[lo + lane] <= t;
    return lo + __popcll(__ballot(below)) - 1;
}

// ---------------------------------------------------------------------------------------------
// append / read.  A workgroup looks up where `per` consecutive token rows lie (one lane each, into LDS), then its threads run over their per x 2 H key and value
// rows, 16 (append) or 8 (read) elements a lane.  Bound by HBM: 2 bytes of tokens and 1 or 2 of codes per element, once each; looking up costs four dependent loads, so a
// workgroup takes several rows as soon as there are enough to fill the card (kv_rows_per_group).  96 ragged prompts of 20 heads of 64 into int8: 17.5 us, 4.9 TB/s;
// 32 windows of 1500 keys back from e4m3: 64 us, 5.8 TB/s; a step of 8 tokens: 3.6 us, those loads.
// ---------------------------------------------------------------------------------------------
constexpr int kMostRows = 16;      // token rows of a workgroup

// place[i] of token row t0 + i: its row of the cache (page * page_size + row in page), -1 on no page, -2 of no sequence
__device__ __forceinline__ void find_places(const KvArgs& a, int t0, int per, long* place) {
    if (threadIdx.x < 64) {
        const int lane = threadIdx.x, t = t0 + lane;
        int s = find_seq(a.q_start, a.n_seqs, t0);
        if (lane < per) {
            long at = -2;
            if (t < a.n_tokens) {
                s = max(s, 0);
                while (s < a.n_seqs && a.q_start[s + 1] <= t) s++;       // from the first row's sequence on
                if (s < a.n_seqs) {
                    const Span sp = seq_span(a, s);
                    if (t >= sp.q0 && t < sp.q0 + sp.n_new) {
                        const int pos = sp.pos0 + (t - sp.q0), page = pos < 0 ? -1 : page_at(a, s, pos >> a.page_shift);
                        at = page < 0 ? -1 : ((long)page << a.page_shift) + (pos & ((1 << a.page_shift) - 1));
                    }
                }
            }
            place[lane] = at;
        }
    }
    __syncthreads();
}
template <int LPR> __device__ __forceinline__ unsigned lanes_umax(unsigned v) {   // over the LPR lanes of a row
#define SS_DPP_UMAX(CTRL) v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false))
    SS_DPP_UMAX(kDppXor1); SS_DPP_UMAX(kDppXor2);
    if (LPR == 8) SS_DPP_UMAX(kDppHalfMirror);
#undef SS_DPP_UMAX
    return v;
}
// item -> (key or value head, token row, PER elements), the elements first and the heads last: a head's rows of neighbouring positions touch in a page, so
// neighbouring lanes read or write whole lines of it (with the tokens last: 64-byte pieces, the read of 32 windows 104 us instead of 93)
template <int D, int PER> struct Item {
    static constexpr int LPR = D / PER;
    int i, h, c;                   // token row of the workgroup, head, piece of PER elements
    bool is_v;
    __device__ __forceinline__ Item(int item, int shift, int H) {
        const int r = item / LPR;
        c = item % LPR;
        i = r & ((1 << shift) - 1);
        h = r >> shift;
        is_v = h >= H;
        if (is_v) h -= H;
    }
};
__device__ __forceinline__ float i8_at(unsigned w, int i) { return (float)(int)(signed char)(w >> (8 * i)); }

template <typename T, int KIND, int D>
__global__ __launch_bounds__(256) void kv_append_kernel(KvArgs a, int shift, const T* __restrict__ kn, long k_row, long k_head, const T* __restrict__ vn, long v_row, long v_head) {
    typedef typename Mfma<T>::V8 V8;
    __shared__ long place[kMostRows];
    const int t0 = blockIdx.x << shift;
    find_places(a, t0, 1 << shift, place);
    const int items = (2 * a.H * Item<D, 16>::LPR) << shift, mask = (1 << a.page_shift) - 1;
    for (int item = blockIdx.y * 256 + threadIdx.x; item < items; item += gridDim.y * 256) {
        const Item<D, 16> it(item, shift, a.H);
        const long at = place[it.i];
        if (at < 0) continue;                            // the lanes of a row agree
        const int t = t0 + it.i;
        const T* src = (it.is_v ? vn + (long)t * v_row + (long)it.h * v_head : kn + (long)t * k_row + (long)it.h * k_head) + it.c * 16;
        const V8 x[2] = {*(const V8*)src, *(const V8*)(src + 8)};
        const int page = (int)(at >> a.page_shift);
        const long slot = ((long)it.h << a.page_shift) + (at & mask);            // row inside the page
        char* dst = page_ptr(it.is_v ? a.v : a.k, page, a.page_bytes);
        if constexpr (KIND == K_F16 || KIND == K_BF16) {
            *(V8*)(dst + (slot * D + it.c * 16) * 2) = x[0];
            *(V8*)(dst + (slot * D + it.c * 16 + 8) * 2) = x[1];
        } else {
            float f[16];
            unsigned top = 0;      // the largest magnitude as bits: a NaN outranks every number, so a row that holds one reads back as NaN
#pragma unroll
            for (int i = 0; i < 16; i++) { f[i] = (float)x[i >> 3][i & 7]; top = max(top, __float_as_uint(f[i]) & 0x7fffffffu); }
            top = lanes_umax<D / 16>(top);
            const bool infinite = top == 0x7f800000u;
            u32x4 code;
            char* sc = it.is_v ? a.vs : a.ks;
            const long sat = (long)((unsigned long)(unsigned)page * a.sc_stride) + slot;
            if constexpr (KIND == K_E4M3) {
                const int e = infinite ? 253 : e8m0_for_amax(__uint_as_float(top));
                const float m = pow2_neg_of_e8m0(e);
#pragma unroll
                for (int i = 0; i < 16; i++) f[i] *= m;
                if (infinite)
#pragma unroll
                    for (int i = 0; i < 16; i++) f[i] = fminf(fmaxf(f[i], -448.0f), 448.0f);
#pragma unroll
                for (int i = 0; i < 4; i++) code[i] = pack_e4m3x4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]);
                if (it.c == 0) sc[sat] = (char)e;
            } else {
                const float s8 = __uint_as_float(top) / 127.0f, by = s8 > 0.0f ? s8 : 1.0f;
                // x / s as IEEE rounds it (ties of the code depend on it, and of 16-bit rows one element in 400 lies on a tie): from the correctly rounded
                // reciprocal of the row, two corrections by the exact remainder, 5 instructions an element instead of the division's 11
                const float r = 1.0f / by;
                float q[16];
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    float y = f[i] * r;
                    y = fmaf(fmaf(-by, y, f[i]), r, y);
                    y = fmaf(fmaf(-by, y, f[i]), r, y);
                    q[i] = rintf(y);
                }
                if (__ballot(!(s8 < 1e30f) || by < 1e-30f)) {    // remainders out of float's range; an infinity; a NaN
                    asm volatile("");
                    const bool finite = top < 0x7f800000u;
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const float whole = fminf(fmaxf(rintf(f[i] / by), -127.0f), 127.0f), end = fabsf(f[i]) < __builtin_huge_valf() ? 0.0f : copysignf(127.0f, f[i]);
                        q[i] = finite ? whole : end;
                    }
                }
                unsigned b[16];
#pragma unroll
                for (int i = 0; i < 16; i++) b[i] = (unsigned)(int)q[i] & 0xffu;
#pragma unroll
                for (int i = 0; i < 4; i++) code[i] = b[4 * i] | b[4 * i + 1] << 8 | b[4 * i + 2] << 16 | b[4 * i + 3] << 24;
                if (it.c == 0) ((float*)sc)[sat] = s8;
            }
            *(u32x4*)(dst + slot * D + it.c * 16) = code;
        }
    }
}

// NT: results of more than kNtBytes leave past the caches, which could not hold them for their reader anyway (245 MB: 64 instead of 83 us from 8 bits, 77
// instead of 102 from 16; at 31 MB there is no difference, and the reader finds them cached).  8 elements a lane: each store instruction
// writes whole lines (16, two stores each: 94 us).
constexpr long kNtBytes = 128l << 20;
template <typename T, int KIND, int D, bool NT>
__global__ __launch_bounds__(256) void kv_read_kernel(KvArgs a, int shift, T* __restrict__ ko, long k_row, long k_head, T* __restrict__ vo, long v_row, long v_head) {
    typedef typename Mfma<T>::V8 V8;
    __shared__ long place[kMostRows];
    const int t0 = blockIdx.x << shift;
    find_places(a, t0, 1 << shift, place);
    const int items = (2 * a.H * Item<D, 8>::LPR) << shift, mask = (1 << a.page_shift) - 1;
#pragma unroll 4
    for (int item = blockIdx.y * 256 + threadIdx.x; item < items; item += gridDim.y * 256) {
        const Item<D, 8> it(item, shift, a.H);
        const long at = place[it.i];
        if (at == -2) continue;
        V8 x;
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = (T)0.0f;
        if (at >= 0) {
            const int page = (int)(at >> a.page_shift);
            const long slot = ((long)it.h << a.page_shift) + (at & mask);
            const char* src = page_ptr(it.is_v ? a.v : a.k, page, a.page_bytes);
            if constexpr (KIND == K_F16 || KIND == K_BF16) x = *(const V8*)(src + (slot * D + it.c * 8) * 2);
            else {
                const u32x2 code = *(const u32x2*)(src + slot * D + it.c * 8);
                const char* sc = it.is_v ? a.vs : a.ks;
                const long sat = (long)((unsigned long)(unsigned)page * a.sc_stride) + slot;
                float m;
                if constexpr (KIND == K_E4M3) m = __uint_as_float((unsigned)(unsigned char)sc[sat] << 23);
                else m = ((const float*)sc)[sat];
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    float f[4];
                    if constexpr (KIND == K_E4M3) {
                        f[0] = __builtin_amdgcn_cvt_f32_fp8(code[i], 0); f[1] = __builtin_amdgcn_cvt_f32_fp8(code[i], 1);
                        f[2] = __builtin_amdgcn_cvt_f32_fp8(code[i], 2); f[3] = __builtin_amdgcn_cvt_f32_fp8(code[i], 3);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; e++) f[e] = i8_at(code[i], e);
                    }
#pragma unroll
                    for (int e = 0; e < 4; e++) x[4 * i + e] = (T)(f[e] * m);
                }
            }
        }
        const int t = t0 + it.i;
        T* dst = (it.is_v ? vo + (long)t * v_row + (long)it.h * v_head : ko + (long)t * k_row + (long)it.h * k_head) + it.c * 8;
        if constexpr (NT) __builtin_nontemporal_store(x, (V8*)dst);
        else *(V8*)dst = x;
    }
}

// ---------------------------------------------------------------------------------------------
// attention: o_q = sum_j p_qj v_j / sum_j p_qj, p_qj = exp2(x_qj - m_q), x_qj = scale log2(e) q.k_j, over j < limit_q.
//
// Both kernels compute S^T = K Q^T with mfma 16x16x32 (A = 16 keys, B = 16 query rows), so a lane owns one query row (lane & 15) and, of every 16
// keys, rows 4 g .. 4 g + 3 (g = lane >> 4).  Two such blocks give it 8 keys = its B operand of the next product O^T = V^T P^T: the contraction index
// (g, j) stands for key 16 (j >> 2) + 4 g + (j & 3) on both sides, so the probabilities never leave the registers.  The A operand of that product
// wants, per lane, 8 keys of one column; a lane reads D/16 neighbouring columns of its 8 keys (whole lines across the 16 lanes) and turns that
// little block with v_perm: MFMA number jj takes column (D/16) (lane & 15) + jj.  No transposed copy of V exists anywhere.
//
// 8-bit caches: codes enter the MFMA as f16 (exact: |code| <= 448) whatever the tokens' type; a key's scale multiplies its score in f32, a value's
// scale multiplies its probability, relative to a running power of two (sref) near the largest scale seen, so that no term leaves f16's range at the top.
// bf16 queries are brought to f16 by a power of two of their own (exact but for elements below 2^-17 of the row's largest, which keep steps of 2^-24 of it).
//
// m_q need not be the maximum, only near it: it moves when a score exceeds it by more than 2^8 (p then is at most 2^8, in f16 as in bf16), which
// leaves most tiles without a reduction across lanes and without rescaling O.
//
// At the bottom f16 holds a number in full only from 2^-14 on.  So over f16 caches all p of a row are taken 2^7 higher (l, O and p alike: the division takes it
// out; p is at most 2^(8 + 7)): a long tail of probabilities down to 2^-21 of the largest keeps its digits.  Over 8-bit caches f16 holds p v_j / sref, and sref may
// belong to a key that a row does not see or that weighs nothing there: all p of a row are taken 2^lift higher, 2^5, and where the row's largest term lies
// below 2^-8, as much more as brings it to 1, as far as float32 holds p (2^121; l is kept 2^64 lower, so that its sum stays in range too).  Terms then reach
// 2^(8 + 2 + 5) at most, and the row's largest lies at 2^-3 or above.  It is looked for only where m or sref moved and while some row of the wave is low; in
// between it can only grow.
// ---------------------------------------------------------------------------------------------
struct AttnArgs {
    const void* q; long q_row, q_head;
    void* out; long o_row, o_head;
    float* lse;                        // [n_tokens][heads] or null
    float* part; float2* part_ml;      // [n_tokens][heads][splits][D], [n_tokens][heads][splits]
    float c2;                          // |scale| * log2(e), at least the smallest normal number: a masked -inf stays one
    int neg;                           // scale < 0: the queries' signs are turned instead
    int G, causal, splits, split_keys; // query heads per key head; key ranges and their length (a multiple of 128)
    int max_new;                       // the first max_new tokens of a span are computed: the launch has room for no more, whatever q_start holds by now
    int nq;                            // tile kernel: query tiles per (sequence, head)
};

constexpr float kInf = __builtin_huge_valf();
constexpr float kSlack = 8.0f;         // log2 of the largest probability relative to m
constexpr float kRefRange = 4.0f;      // of a value's scale above sref
template <typename M, bool SCALED> constexpr float kLift = std::is_same<M, bf16>::value ? 0.0f : SCALED ? 5.0f : 7.0f;      // in log2 units
constexpr float kLow = -8.0f, kMostLift = 121.0f;     // 8-bit caches
constexpr float kDown = 0x1p-64f;      // 8-bit caches: on l

template <int KIND> struct Held;       // what the MFMA multiplies, and bytes of an element
template <> struct Held<K_F16> { typedef f16 M; static constexpr int B = 2; };
template <> struct Held<K_BF16> { typedef bf16 M; static constexpr int B = 2; };
template <> struct Held<K_E4M3> { typedef f16 M; static constexpr int B = 1; };
template <> struct Held<K_I8> { typedef f16 M; static constexpr int B = 1; };

__device__ __forceinline__ unsigned perm(unsigned hi, unsigned lo, unsigned sel) { return __builtin_amdgcn_perm(hi, lo, sel); }

// four codes -> two f16 pairs.  int8: byte u = code + 128 under the byte 0x64 is the f16 number 1024 + u; minus 1152 gives the code, exactly
__device__ __forceinline__ unsigned f16_less_1152(unsigned w) {
    const h16x2 k = {(f16)1152.0f, (f16)1152.0f};
    return __builtin_bit_cast(unsigned, __builtin_bit_cast(h16x2, w) - k);
}
template <int KIND> __device__ __forceinline__ void codes_to_f16(unsigned w, unsigned* o) {
    if constexpr (KIND == K_E4M3) {
        o[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
        o[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true));
    } else {
        w ^= 0x80808080u;
        o[0] = f16_less_1152(perm(0x64646464u, w, 0x04010400u));
        o[1] = f16_less_1152(perm(0x64646464u, w, 0x04030402u));
    }
}

// the 16 query rows of one column tile as B operands; returns the power of two that was taken out of this lane's row.  `dim0(s)`: first of the 8
// dims that this lane's group contributes to k-step s
template <typename T, typename M, int D, bool PAIRED>
__device__ __forceinline__ float load_q(const T* q, bool ok, bool neg, int g, typename Mfma<M>::V8* qf) {
    typedef typename Mfma<T>::V8 TV8;
    TV8 x[D / 32];
#pragma unroll
    for (int s = 0; s < D / 32; s++) {
        const int dim = PAIRED ? 64 * (s >> 1) + 16 * g + 8 * (s & 1) : 32 * s + 8 * g;
        if (ok) x[s] = *(const TV8*)(q + dim);
        else
#pragma unroll
            for (int i = 0; i < 8; i++) x[s][i] = (T)0.0f;
    }
    float back = 1.0f;
    if constexpr (std::is_same<T, M>::value) {
#pragma unroll
        for (int s = 0; s < D / 32; s++) qf[s] = x[s];
    } else {
        float top = 0.0f;
#pragma unroll
        for (int s = 0; s < D / 32; s++)
#pragma unroll
            for (int i = 0; i < 8; i++) top = fmaxf(top, fabsf((float)x[s][i]));
        top = rows_max(top);
        const unsigned e = min(max(__float_as_uint(top) >> 23, 1u), 253u);
        const float m = __uint_as_float((254u - e) << 23);
        back = __uint_as_float(e << 23);
#pragma unroll
        for (int s = 0; s < D / 32; s++)
#pragma unroll
            for (int i = 0; i < 8; i++) qf[s][i] = (M)((float)x[s][i] * m);
    }
    if (neg)
#pragma unroll
        for (int s = 0; s < D / 32; s++) qf[s] = -qf[s];
    return back;
}

// A operand of O^T += V^T P^T from the D/16 columns x 8 keys block a lane holds (DW dwords per key)
template <typename M, int KIND, int D> struct VBlock {
    static constexpr int DW = D / 16 * Held<KIND>::B / 4;
    unsigned w[8][DW];
    __device__ __forceinline__ void frags(typename Mfma<M>::V8* f) const {
        u32x4* o = (u32x4*)f;
        if constexpr (Held<KIND>::B == 2) {
#pragma unroll
            for (int d = 0; d < DW; d++)
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    o[2 * d][t] = perm(w[2 * t + 1][d], w[2 * t][d], 0x05040100u);
                    o[2 * d + 1][t] = perm(w[2 * t + 1][d], w[2 * t][d], 0x07060302u);
                }
        } else if constexpr (KIND == K_E4M3) {
#pragma unroll
            for (int d = 0; d < DW; d++)
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    unsigned x[2], y[2];
                    codes_to_f16<KIND>(w[2 * t][d], x);
                    codes_to_f16<KIND>(w[2 * t + 1][d], y);
#pragma unroll
                    for (int p = 0; p < 2; p++) {
                        o[4 * d + 2 * p][t] = perm(y[p], x[p], 0x05040100u);
                        o[4 * d + 2 * p + 1][t] = perm(y[p], x[p], 0x07060302u);
                    }
                }
        } else {
#pragma unroll
            for (int d = 0; d < DW; d++)
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    const unsigned x = w[2 * t][d] ^ 0x80808080u, y = w[2 * t + 1][d] ^ 0x80808080u;
                    const unsigned lo = perm(y, x, 0x05010400u), hi = perm(y, x, 0x07030602u);   // (x0 y0 x1 y1), (x2 y2 x3 y3)
                    o[4 * d][t] = f16_less_1152(perm(0x64646464u, lo, 0x04010400u));
                    o[4 * d + 1][t] = f16_less_1152(perm(0x64646464u, lo, 0x04030402u));
                    o[4 * d + 2][t] = f16_less_1152(perm(0x64646464u, hi, 0x04010400u));
                    o[4 * d + 3][t] = f16_less_1152(perm(0x64646464u, hi, 0x04030402u));
                }
        }
    }
};

// Online softmax state of one column tile (a lane's query row), and the step for 32 keys
template <typename M, bool SCALED, int D> struct Row {
    float raw = -kInf, l = 0.0f;       // m before the factor c; l: this lane's keys only, total() sums the four groups
    float big = -kInf;                 // SCALED: log2 of the row's largest term p v / sref where it was last looked for, p relative to 2^m
    f32x4 o[D / 16];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < D / 16; i++) o[i] = (f32x4){0, 0, 0, 0};
    }
    __device__ __forceinline__ float m(float c) const { return raw * c; }        // in log2 units
    __device__ __forceinline__ float lift() const {          // a whole number; l and o hold 2^lift times the sums relative to 2^m
        return kLift<M, SCALED> + (SCALED && big < kLow && big > -kInf ? fminf(ceilf(-big), kMostLift) : 0.0f);
    }
    __device__ __forceinline__ float unlift() const { return __uint_as_float((unsigned)(127 - (int)lift()) << 23); }
    __device__ __forceinline__ void sum(float w) { l = SCALED ? fmaf(w, kDown, l) : l + w; }
    __device__ __forceinline__ float total() const {          // relative to 2^m
        const float t = rows_sum(l);
        return t * unlift() * (SCALED ? 1.0f / kDown : 1.0f);
    }
    __device__ __forceinline__ void scale(float a) {
        l *= a;
#pragma unroll
        for (int i = 0; i < D / 16; i++) o[i] *= a;
    }
    __device__ __forceinline__ void add(const typename Mfma<M>::V8* vf, typename Mfma<M>::V8 p) {
#pragma unroll
        for (int i = 0; i < D / 16; i++) o[i] = Mfma<M>::mma(vf[i], p, o[i]);
    }
};
struct Gauge { bool far = false, low = false; };       // of some row of the wave: |m| is large; its largest term is small

// Scores x[QC][8] of 32 keys (-inf where masked; c > 0 brings them to log2 units) -> what probs() subtracts from x c.  `value(e)`: scale / sref of
// the key of score e; by: what sref's last move multiplied O by, 1 if it did not move.
// exp2(x c - m) is one fma and one exponential.  The fma does not round x c where m did, so every probability of the row is off by the factor
// 2^(x c - m at the maximum), at most 2^(|m| 2^-24), which the division by l takes out again but for what m's moves leave: below 2^-12 of it as far
// as |m| <= 2^12 (the scores' own float32 steps then are as large).  Beyond that (far, the same for the whole wave) the difference is formed first.
template <int QC, int NE, typename M, bool SCALED, int D, typename F>
__device__ __forceinline__ void softmax_ref(Row<M, SCALED, D>* st, Gauge& ga, float by, float (*x)[NE], const float* c, float* ref, F value) {
    float top[QC];
    bool moved = SCALED && by != 1.0f;
#pragma unroll
    for (int j = 0; j < QC; j++) {
        top[j] = x[j][0];
#pragma unroll
        for (int e = 1; e < NE; e++) top[j] = fmaxf(top[j], x[j][e]);
        const float m = st[j].m(c[j]);
        moved |= top[j] * c[j] > m + kSlack;
        ref[j] = (m == -kInf ? 0.0f : m) - kLift<M, SCALED>;
    }
    if (__ballot(moved) || ga.far || ga.low) {
        asm volatile("");              // a branch, not selects
        bool f = false, w = false;
#pragma unroll
        for (int j = 0; j < QC; j++) {                     // m up to the largest score so far, what was summed along with it
            const float old = st[j].m(c[j]);
            st[j].raw = fmaxf(st[j].raw, rows_max(top[j]));
            const float mn = st[j].m(c[j]);
            ref[j] = mn == -kInf ? 0.0f : mn;
            st[j].scale(__builtin_amdgcn_exp2f(old - ref[j]) * (SCALED ? st[j].unlift() : 1.0f));
            if (SCALED) st[j].big += old - ref[j] + __builtin_amdgcn_logf(by);       // by 0: nothing but zeros has been summed
            f |= fabsf(ref[j]) > 4096.0f;
        }
        ga.far = __ballot(f) != 0;
        if (ga.far)
#pragma unroll
            for (int j = 0; j < QC; j++) {
#pragma unroll
                for (int e = 0; e < NE; e++) x[j][e] -= st[j].raw == -kInf ? 0.0f : st[j].raw;
                ref[j] = 0.0f;
            }
        if constexpr (SCALED) {
#pragma unroll
            for (int j = 0; j < QC; j++) top[j] = -kInf;
#pragma unroll
            for (int e = 0; e < NE; e++) {
                const float v = __builtin_amdgcn_logf(value(e));
#pragma unroll
                for (int j = 0; j < QC; j++) top[j] = fmaxf(top[j], fmaf(x[j][e], c[j], v - ref[j]));
            }
#pragma unroll
            for (int j = 0; j < QC; j++) {
                st[j].big = fmaxf(st[j].big, rows_max(top[j]));
                w |= st[j].raw > -kInf && st[j].big < kLow;
                const float lift = st[j].lift();
                st[j].scale(__uint_as_float((unsigned)(127 + (int)lift) << 23));
                ref[j] -= lift;
            }
            ga.low = __ballot(w) != 0;
        } else
#pragma unroll
            for (int j = 0; j < QC; j++) ref[j] -= kLift<M, SCALED>;
    }
}
// 8 scores of a lane -> its B operand
template <typename M, bool SCALED, int D>
__device__ __forceinline__ typename Mfma<M>::V8 probs(Row<M, SCALED, D>& st, const float* x, float c, float ref, const float* v) {
    typename Mfma<M>::V8 p;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float w = __builtin_amdgcn_exp2f(fmaf(x[e], c, -ref));
        st.sum(w);
        p[e] = (M)(SCALED ? w * v[e] : w);
    }
    return p;
}

// the running power of two near the largest value scale; one per wave
struct ScaleRef {
    float ref = 0.0f;
    // of the scales of a tile, `top` the lane's largest: did it move, and what O has to be multiplied by then
    __device__ __forceinline__ bool moves(float top, float* by) {
        if (!__ballot(top > ref * kRefRange)) return false;
        const float n = fmaxf(__uint_as_float(__float_as_uint(fmaxf(wave_max(top), ref)) & 0x7f800000u), 1.17549435e-38f);   // (scales may be subnormal)
        *by = ref / n;
        ref = n;
        return true;
    }
    __device__ __forceinline__ float inv() const { return ref > 0.0f ? 1.0f / ref : 0.0f; }
};

// a finished row's output: acc[D/16] columns from `col` on of head row `out`
template <typename T, int N> __device__ __forceinline__ void store_cols(T* p, const float* x) {
    if constexpr (N == 4) {
        typename Mfma<T>::V4 y;
#pragma unroll
        for (int i = 0; i < 4; i++) y[i] = (T)x[i];
        *(typename Mfma<T>::V4*)p = y;
    } else {
        typename Mfma<T>::V8 y;
#pragma unroll
        for (int i = 0; i < 8; i++) y[i] = (T)x[i];
        *(typename Mfma<T>::V8*)p = y;
    }
}

// ---- few query rows (max_new G <= 16): grid (sequences x splits, key heads); the 4 waves of a workgroup take every fourth 32-key tile of its key
// range straight from memory into registers (the next tile's loads fly while one is computed) and merge at the end.  HBM-bound: with G <= 16 the
// MFMA issues of a tile take ~1/10 of the time its bytes need at the card's rate, so the 15 idle columns of a one-head row cost nothing.
// 4 contexts of 30001..65536 bf16 keys, 8 x 4 heads of 128: 116 us, 6.7 TB/s; 96 x 1500 e4m3 keys, 20 heads of 64: 76 us, 4.9 TB/s (74 without the rows' largest terms); a step of 8 short contexts: 9 us. ----
template <int KIND, int D> struct KvTile {
    static constexpr int B = Held<KIND>::B, KN = D * B / 64;   // 16-byte pieces of a key row per lane
    u32x4 k[2][KN];
    VBlock<typename Held<KIND>::M, KIND, D> v;
    float ks[8], vs[8];
    int page[2];

    __device__ __forceinline__ void load(const KvArgs& a, int h, int key0, int p0, int p1, int lane) {
        const int m = lane & 15, g = lane >> 4;
        page[0] = p0; page[1] = p1;
        const int mask = (1 << a.page_shift) - 1;
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const int p = max(page[b], 0), r0 = (key0 + 16 * b) & mask;     // 16 keys share a page
            const long row = ((long)h << a.page_shift) + r0;
            const char* kp = page_ptr(a.k, p, a.page_bytes) + row * (D * B);
            const char* vp = page_ptr(a.v, p, a.page_bytes) + row * (D * B);
#pragma unroll
            for (int i = 0; i < KN; i++) k[b][i] = *(const u32x4*)(kp + m * (D * B) + 64 * i + 16 * g);
            constexpr int DW = VBlock<typename Held<KIND>::M, KIND, D>::DW;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const char* src = vp + (4 * g + r) * (D * B) + m * (4 * DW);
                if constexpr (DW == 1) v.w[4 * b + r][0] = *(const unsigned*)src;
                else if constexpr (DW == 2) { const u32x2 t = *(const u32x2*)src; v.w[4 * b + r][0] = t[0]; v.w[4 * b + r][1] = t[1]; }
                else {
                    const u32x4 t = *(const u32x4*)src;
#pragma unroll
                    for (int i = 0; i < 4; i++) v.w[4 * b + r][i] = t[i];
                }
            }
            const long at = (long)((unsigned long)(unsigned)p * a.sc_stride) + row + 4 * g;
            if constexpr (KIND == K_E4M3) {
                const unsigned x = *(const unsigned*)(a.ks + at), y = *(const unsigned*)(a.vs + at);
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    ks[4 * b + r] = __uint_as_float((x >> (8 * r) & 255u) << 23);
                    vs[4 * b + r] = __uint_as_float((y >> (8 * r) & 255u) << 23);
                }
            } else if constexpr (KIND == K_I8) {
                const f32x4 x = *(const f32x4*)(a.ks + 4 * at), y = *(const f32x4*)(a.vs + 4 * at);
#pragma unroll
                for (int r = 0; r < 4; r++) { ks[4 * b + r] = x[r]; vs[4 * b + r] = y[r]; }
            }
        }
    }
};

// (launch bounds: head_dim 64 at 3 waves a SIMD, 76 us for 96 windows; at 4 it spills, 103)
template <typename T, int KIND, int D>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void kv_attn_few_kernel(KvArgs a, AttnArgs t) {
    typedef typename Held<KIND>::M M;
    typedef typename Mfma<M>::V8 V8;
    constexpr bool SCALED = Held<KIND>::B == 1;
    constexpr int N = D / 16;
    __shared__ float s_o[4][16][D];
    __shared__ float s_m[4][16], s_l[4][16], s_ref[4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
    const int h = blockIdx.y, s = blockIdx.x / t.splits, split = blockIdx.x % t.splits;
    const Span sp = seq_span(a, s);
    const int rows = min(sp.n_new, t.max_new) * t.G;       // <= 16
    if (rows == 0) return;

    const bool mine = c < rows;
    const int tok = c / t.G, row = sp.q0 + (mine ? tok : 0), head = h * t.G + (mine ? c % t.G : 0);
    const int limit = !mine ? 0 : t.causal ? max(0, min(sp.pos0 + tok + 1, sp.len)) : sp.len;     // keys this lane's query row sees
    const int full = t.causal ? max(0, min(sp.pos0 + 1, sp.len)) : sp.len;                        // keys every row sees
    V8 qf[D / 32];
    const float back = load_q<T, M, D, SCALED>((const T*)t.q + (long)row * t.q_row + (long)head * t.q_head, mine, t.neg, g, qf);
    const float c2 = fmaxf(t.c2 * back, 1.17549435e-38f);

    const int lo = split * t.split_keys, hi = split == t.splits - 1 ? sp.len : min(sp.len, lo + t.split_keys);
    const int n = hi > lo ? (hi - lo + 31) / 32 : 0, mine_n = n > wave ? (n - wave + 3) / 4 : 0;   // tiles of the range / of this wave
    Row<M, SCALED, D> st;
    st.clear();
    Gauge ga;
    ScaleRef sr;

    int ids[2] = {-1, -1};             // lane i: the pages of this wave's tile i of the current 64
    auto fetch_ids = [&](int first) {
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const int key = lo + ((first + lane) * 4 + wave) * 32 + 16 * b;
            ids[b] = first + lane < mine_n && key < hi ? page_at(a, s, key >> a.page_shift) : -1;
        }
    };
    auto load = [&](KvTile<KIND, D>& x, int i) {
        if ((i & 63) == 0) fetch_ids(i);
        x.load(a, h, lo + (i * 4 + wave) * 32, __builtin_amdgcn_readlane(ids[0], i & 63), __builtin_amdgcn_readlane(ids[1], i & 63), lane);
    };
    auto compute = [&](KvTile<KIND, D>& x, int i) {
        const int key0 = lo + (i * 4 + wave) * 32;
        float sc[8];
#pragma unroll
        for (int b = 0; b < 2; b++) {
            f32x4 z = {0, 0, 0, 0};
#pragma unroll
            for (int d = 0; d < D / 32; d++) {
                V8 kf;
                if constexpr (!SCALED) kf = __builtin_bit_cast(V8, x.k[b][d]);
                else {
                    u32x4 w;
                    unsigned o[2];
                    codes_to_f16<KIND>(x.k[b][d >> 1][2 * (d & 1)], o); w[0] = o[0]; w[1] = o[1];
                    codes_to_f16<KIND>(x.k[b][d >> 1][2 * (d & 1) + 1], o); w[2] = o[0]; w[3] = o[1];
                    kf = __builtin_bit_cast(V8, w);
                }
                z = Mfma<M>::mma(kf, qf[d], z);
            }
#pragma unroll
            for (int r = 0; r < 4; r++) sc[4 * b + r] = SCALED ? z[r] * x.ks[4 * b + r] : z[r];
        }
        if (key0 + 32 > full || x.page[0] < 0 || x.page[1] < 0) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int key = key0 + 16 * (j >> 2) + 4 * g + (j & 3);
                const bool held = key < sp.len && x.page[j >> 2] >= 0;
                if (!held || key >= limit) sc[j] = -kInf;
                if (!held) {           // whatever lies there (it may be NaN): 0 x probability 0
#pragma unroll
                    for (int d = 0; d < x.v.DW; d++) x.v.w[j][d] = 0;
                    x.vs[j] = 0.0f;
                }
            }
        }
        float by = 1.0f;
        if constexpr (SCALED) {
            const float* v = x.vs;
            if (sr.moves(fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7]))), &by))
#pragma unroll
                for (int k = 0; k < N; k++) st.o[k] *= by;
            const float inv = sr.inv();
#pragma unroll
            for (int j = 0; j < 8; j++) x.vs[j] *= inv;
        }
        float m;
        softmax_ref<1, 8>(&st, ga, by, &sc, &c2, &m, [&](int e) { return x.vs[e]; });
        const V8 p = probs(st, sc, c2, m, x.vs);
        V8 vf[N];
        x.v.frags(vf);
        st.add(vf, p);
    };
    KvTile<KIND, D> x, y;
    if (mine_n > 0) load(x, 0);
    for (int i = 0; i < mine_n; i += 2) {
        if (i + 1 < mine_n) load(y, i + 1);
        compute(x, i);
        if (i + 1 < mine_n) {
            if (i + 2 < mine_n) load(x, i + 2);
            compute(y, i + 1);
        }
    }

    // merge the four waves: sums relative to the largest m and, in 8 bits, to the largest sref (of 0 where a wave met no value but zeros)
    const float l = st.total();
    const float m = st.m(c2);
    if (lane < 16) { s_m[wave][c] = m; s_l[wave][c] = l; }
    if (SCALED && lane == 0) s_ref[wave] = sr.ref;
    __syncthreads();
    const float R = SCALED ? fmaxf(fmaxf(s_ref[0], s_ref[1]), fmaxf(s_ref[2], s_ref[3])) : 1.0f;
    float M4 = fmaxf(fmaxf(s_m[0][c], s_m[1][c]), fmaxf(s_m[2][c], s_m[3][c]));
    const float f = __builtin_amdgcn_exp2f(m - M4) * (SCALED && R > 0.0f ? sr.ref / R : 1.0f);
#pragma unroll
    for (int r = 0; r < 4; r++)
#pragma unroll
        for (int k = 0; k < N; k++) s_o[wave][c][N * (4 * g + r) + k] = M4 == -kInf ? 0.0f : st.o[k][r] * st.unlift() * f;
    __syncthreads();
    const int oc = threadIdx.x >> 4, col = (threadIdx.x & 15) * N;
    if (oc >= rows) return;
    M4 = fmaxf(fmaxf(s_m[0][oc], s_m[1][oc]), fmaxf(s_m[2][oc], s_m[3][oc]));
    float L = 0.0f, acc[N];
#pragma unroll
    for (int w = 0; w < 4; w++) L += s_l[w][oc] * (M4 == -kInf ? 1.0f : __builtin_amdgcn_exp2f(s_m[w][oc] - M4));      // m -inf: no key (l = 0), or a query of NaN (l = NaN)
#pragma unroll
    for (int k = 0; k < N; k++) acc[k] = (s_o[0][oc][col + k] + s_o[1][oc][col + k]) + (s_o[2][oc][col + k] + s_o[3][oc][col + k]);
    const int orow = sp.q0 + oc / t.G, ohead = h * t.G + oc % t.G;
    const long at = (long)orow * (a.H * t.G) + ohead;
    if (t.splits == 1) {
        const float inv = L > 0.0f ? 1.0f / L : L;         // no key: zeros (L is 0 or NaN here)
#pragma unroll
        for (int k = 0; k < N; k++) acc[k] = acc[k] * inv * R;       // (in this order: R may be the smallest normal number)
        store_cols<T, N>((T*)t.out + (long)orow * t.o_row + (long)ohead * t.o_head + col, acc);
        if (t.lse && col == 0) t.lse[at] = L > 0.0f ? (M4 + __builtin_amdgcn_logf(L)) * 0.69314718055994530942f : (L == 0.0f ? -kInf : L);
    } else {
        float* o = t.part + (at * t.splits + split) * D + col;
#pragma unroll
        for (int k = 0; k < N; k++) o[k] = acc[k] * R;
        if (col == 0) t.part_ml[at * t.splits + split] = make_float2(M4, L);
    }
}

// ---- many query rows: a workgroup of 4 waves owns 64 QC query rows of one (sequence, key head), each wave 16 QC of them; 64-key tiles of K and V go
// through LDS as 16 bits (8-bit codes are converted once, on the way in), the next tile's loads fly while one is computed, the page numbers of the one
// after that are on their way too; one barrier a tile.  V fragments come out of LDS by the transposing read (ds_read_b64_tr_b16: of each 16 lanes, lane i
// names 4 columns of row i / 4 and receives 4 rows of column i), columns 16 n + (lane & 15) for MFMA n.
// Bound by LDS (a 64-key tile is read once per wave: 106..117 B/clk for the keys, 57 for the transposing reads) and by the dependency chain of its two waves a
// SIMD: 2 chunks of 2048 x 32 query heads over 16384 int8 keys of 128: 1.21 ms, 806 TFLOP/s, 68 % of what a large bf16 product reaches here; 16-bit keys 73 %.
// Without its LDS reads it took 740 us, without the exponentials 11 % less, without the staging 22 % less (16 bit 6 %); the rows' largest terms cost 1.5 %. ----
template <typename M> __device__ __forceinline__ typename Mfma<M>::V8 read_tr(const char* p0, const char* p1) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4 lds4;
    struct { s16x4 lo, hi; } v{__builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)p0), __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)p1)};
    return __builtin_bit_cast(typename Mfma<M>::V8, v);
}

template <typename T, int KIND, int D, int QC>
// (launch bounds: head_dim 64 with two column tiles at 3 waves a SIMD, 168 registers of the 172 that it would take: bf16 prompts over int8 45 us instead of 51.
// With four, 256 registers hold all but 1 to 6 values over 8-bit caches, which spill: bf16 over int8 219 us where f16 takes 206)
__global__ __launch_bounds__(256, D == 64 && QC == 2 ? 3 : 2) void kv_attn_tile_kernel(KvArgs a, AttnArgs t) {
    typedef typename Held<KIND>::M M;
    typedef typename Mfma<M>::V8 V8;
    constexpr bool SCALED = Held<KIND>::B == 1;
    constexpr int N = D / 16, B = Held<KIND>::B;
    constexpr int KP = kKeyPitch<D>, VP = kValuePitch<D>, kBuf = kTileBuf<D>;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
    int bid = blockIdx.x;
    {   // consecutive workgroups land on different XCDs: give each XCD a contiguous range, so that the query tiles of one (sequence, head) share an L2
        const int nwg = gridDim.x, q8 = nwg / 8, r8 = nwg % 8, xcd = bid % 8, idx = bid / 8;
        bid = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + idx;
    }
    const int qb = t.nq - 1 - bid % t.nq;                  // causal: the longest first
    bid /= t.nq;
    const int split = bid % t.splits;
    bid /= t.splits;
    const int h = bid % a.H, s = bid / a.H;
    const Span sp = seq_span(a, s);
    const int rows = min(sp.n_new, t.max_new) * t.G, r0 = qb * (64 * QC);
    if (rows <= r0) return;

    const int w0 = r0 + wave * (16 * QC);                  // this wave's first query row
    int limit[QC];
    V8 qf[QC][D / 32];
    float c2[QC];
    auto row_of = [&](int i, int* head) {                  // token row and head of column tile i's row (of row 0 where there is none)
        const int q = w0 + 16 * i + c, ok = q < rows, tok = ok ? q / t.G : 0;
        *head = h * t.G + (ok ? q - tok * t.G : 0);
        return sp.q0 + tok;
    };
#pragma unroll
    for (int i = 0; i < QC; i++) {
        int head;
        const int row = row_of(i, &head);
        const bool ok = w0 + 16 * i + c < rows;
        limit[i] = !ok ? 0 : t.causal ? max(0, min(sp.pos0 + (row - sp.q0) + 1, sp.len)) : sp.len;
        c2[i] = fmaxf(t.c2 * load_q<T, M, D, false>((const T*)t.q + (long)row * t.q_row + (long)head * t.q_head, ok, t.neg, g, qf[i]), 1.17549435e-38f);
    }
    const int last = min(rows, r0 + 64 * QC) - 1;
    const int end = t.causal ? max(0, min(sp.pos0 + last / t.G + 1, sp.len)) : sp.len;            // keys any row of the workgroup sees
    const int wend = w0 >= rows ? 0 : t.causal ? max(0, min(sp.pos0 + (min(rows, w0 + 16 * QC) - 1) / t.G + 1, sp.len)) : sp.len;   // of the wave
    const int full = t.causal ? max(0, min(sp.pos0 + w0 / t.G + 1, sp.len)) : sp.len;             // keys every row of the wave sees
    const int lo = split * t.split_keys, hi = split == t.splits - 1 ? end : min(end, lo + t.split_keys);
    const int n = hi > lo ? (hi - lo + 63) / 64 : 0;

    Row<M, SCALED, D> st[QC];
#pragma unroll
    for (int i = 0; i < QC; i++) st[i].clear();
    ScaleRef sr;

    // staging: a row of codes is PR pieces of 16 bytes; thread -> rows tid / PR + p RP.  The rows that a wave's piece p touches lie in one group of 16 keys,
    // hence on one page: its address is scalar, the lane's offset the same for all pieces and tiles.
    constexpr int PR = D * B / 16, RP = 256 / PR, NP = 64 / RP;
    const int group = wave * (64 / PR) / 16;               // of piece 0
    const unsigned lane_off = (tid / PR & 15) * (D * B) + (tid % PR) * 16;
    u32x4 gk[NP], gv[NP];
    float gks = 0.0f, gvs = 0.0f;      // first wave: the scales of the tile's rows
    int hid = -1;                      // lanes 0..3: page numbers for the next fetch, of 16 keys each
    bool okay = false;                 // of the fetched tile: the scales of this lane's row lie on a page
    int bad = 0;                       // of the fetched tile: bit b = its keys 16 b .. 16 b + 15 lie on no page
    const int mask = (1 << a.page_shift) - 1;
    const long head_row = (long)h << a.page_shift;
    const int* trow = a.table + (long)s * a.table_stride;
    auto there = [&](int page) { return page >= 0 && page < a.n_pages; };
    auto ids = [&](int i) {
        const int key = lo + i * 64 + 16 * lane;
        if (lane < 4) hid = key < sp.len ? trow[key >> a.page_shift] : -1;       // key < len <= max_pages * page_size
    };
    auto fetch = [&](int i) {          // tile i; ids(i) has run
        const int key0 = lo + i * 64;
#pragma unroll
        for (int p = 0; p < NP; p++) {
            const int b = p * RP / 16 + group, id = __builtin_amdgcn_readlane(hid, b);
            const long off = (long)((unsigned long)(unsigned)(there(id) ? id : 0) * a.page_bytes) + (head_row + ((key0 + 16 * b) & mask)) * (D * B);
            gk[p] = *(const u32x4*)(a.k + off + lane_off);
            gv[p] = *(const u32x4*)(a.v + off + lane_off);
        }
        if (SCALED && wave == 0) {
            const int id = __shfl(hid, lane >> 4);
            okay = there(id) && key0 + lane < sp.len;
            const long at = (long)((unsigned long)(unsigned)(there(id) ? id : 0) * a.sc_stride) + head_row + ((key0 + lane) & mask);
            if constexpr (KIND == K_E4M3) {
                gks = __uint_as_float((unsigned)(unsigned char)a.ks[at] << 23);
                gvs = __uint_as_float((unsigned)(unsigned char)a.vs[at] << 23);
            } else { gks = ((const float*)a.ks)[at]; gvs = ((const float*)a.vs)[at]; }
        }
        bad = 0;
#pragma unroll
        for (int b = 0; b < 4; b++) bad |= key0 + 16 * b < sp.len && !there(__builtin_amdgcn_readlane(hid, b)) ? 1 << b : 0;
    };
    auto put = [&](int i, char* buf) { // what fetch(i) brought
        const int key0 = lo + i * 64;
        if (key0 + 64 > sp.len || bad) {                   // values of no key: whatever lies there must not meet a probability of 0
            asm volatile("");
#pragma unroll
            for (int p = 0; p < NP; p++) {
                const int r = tid / PR + p * RP;
                if (key0 + r >= sp.len || (bad >> (r >> 4) & 1)) gv[p] = (u32x4){0, 0, 0, 0};
            }
        }
#pragma unroll
        for (int p = 0; p < NP; p++) {
            const int r = tid / PR + p * RP;
            char *kd = buf + r * KP, *vd = buf + 64 * KP + r * VP;
            if constexpr (!SCALED) {
                *(u32x4*)(kd + (tid % PR) * 16) = gk[p];
                *(u32x4*)(vd + (tid % PR) * 16) = gv[p];
            } else {
                u32x4 x[2];
                unsigned o[2];
#pragma unroll
                for (int w = 0; w < 4; w++) { codes_to_f16<KIND>(gk[p][w], o); x[w >> 1][2 * (w & 1)] = o[0]; x[w >> 1][2 * (w & 1) + 1] = o[1]; }
                *(u32x4*)(kd + (tid % PR) * 32) = x[0];
                *(u32x4*)(kd + (tid % PR) * 32 + 16) = x[1];
#pragma unroll
                for (int w = 0; w < 4; w++) { codes_to_f16<KIND>(gv[p][w], o); x[w >> 1][2 * (w & 1)] = o[0]; x[w >> 1][2 * (w & 1) + 1] = o[1]; }
                *(u32x4*)(vd + (tid % PR) * 32) = x[0];
                *(u32x4*)(vd + (tid % PR) * 32 + 16) = x[1];
            }
        }
        if (SCALED && wave == 0) {     // the first wave keeps sref and hands out what follows from it
            float* sc = (float*)(buf + 64 * (KP + VP));
            const float v = okay ? gvs : 0.0f;
            float by = 1.0f;
            sr.moves(v, &by);
            sc[lane] = okay ? gks : 0.0f;
            sc[64 + lane] = v * sr.inv();
            if (lane == 0) { sc[128] = sr.ref; sc[129] = by; }
        }
    };
    int hole = 0;                      // `bad` of the tile that is computed
    const int koff = c * KP + g * 16, voff = 64 * KP + (4 * g + (c >> 2)) * VP + (c & 3) * 8;
    Gauge ga;
    float ref = 1.0f;                  // sref of what this wave has summed
    auto compute = [&](bool edge, const char* buf, int key0) {      // edge: some key of the tile is masked for some row of the wave
        const float* sc = (const float*)(buf + 64 * (KP + VP));
        float by = 1.0f;
        if constexpr (SCALED) {
            ref = sc[128];
            by = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(sc[129])));
            if (by != 1.0f)
#pragma unroll
                for (int j = 0; j < QC; j++)
#pragma unroll
                    for (int k = 0; k < N; k++) st[j].o[k] *= by;
        }
        // scores: the next 16 keys' fragments are on their way out of LDS while these are multiplied
        float x[QC][16];
        V8 kf[2][D / 32];
        auto read_k = [&](int b) {
#pragma unroll
            for (int d = 0; d < D / 32; d++) kf[b & 1][d] = *(const V8*)(buf + koff + 16 * b * KP + d * 64);
        };
        read_k(0);
#pragma unroll
        for (int b = 0; b < 4; b++) {
            f32x4 z[QC], ks;
            if constexpr (SCALED) ks = *(const f32x4*)(sc + 16 * b + 4 * g);
            if (b < 3) read_k(b + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < QC; j++) z[j] = (f32x4){0, 0, 0, 0};
#pragma unroll
            for (int d = 0; d < D / 32; d++)
#pragma unroll
                for (int j = 0; j < QC; j++) z[j] = Mfma<M>::mma(kf[b & 1][d], qf[j][d], z[j]);
#pragma unroll
            for (int j = 0; j < QC; j++)
#pragma unroll
                for (int r = 0; r < 4; r++) x[j][4 * b + r] = SCALED ? z[j][r] * ks[r] : z[j][r];
        }
        // values: groups of 4 column tiles of one half; a group's fragments are read while the one before is multiplied
        constexpr int NG = N / 4;
        V8 vf[2][4];
        auto read_v = [&](int grp) {
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const char* vp = buf + voff + grp / NG * 32 * VP + (grp % NG * 4 + k) * 32;
                vf[grp & 1][k] = read_tr<M>(vp, vp + 16 * VP);
            }
        };
        read_v(0);
        if (edge) {
            asm volatile("");          // a branch: the selects are not worth their time on the tiles that need none
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const int key = key0 + 16 * (e >> 2) + 4 * g + (e & 3);
                const bool gone = hole >> (e >> 2) & 1;
#pragma unroll
                for (int j = 0; j < QC; j++)
                    if (gone || key >= limit[j]) x[j][e] = -kInf;
            }
        }
        float m[QC];
        softmax_ref<QC, 16>(st, ga, by, x, c2, m, [&](int e) { return sc[64 + 16 * (e >> 2) + 4 * g + (e & 3)]; });
        float vs[2][8];
        if constexpr (SCALED)
#pragma unroll
            for (int b = 0; b < 4; b++) {
                const f32x4 y = *(const f32x4*)(sc + 64 + 16 * b + 4 * g);
#pragma unroll
                for (int r = 0; r < 4; r++) vs[b >> 1][4 * (b & 1) + r] = y[r];
            }
        V8 p[2][QC];
#pragma unroll
        for (int j = 0; j < QC; j++) p[0][j] = probs(st[j], x[j], c2[j], m[j], vs[0]);
#pragma unroll
        for (int grp = 0; grp < 2 * NG; grp++) {
            if (grp + 1 < 2 * NG) read_v(grp + 1);
            __builtin_amdgcn_sched_barrier(0);
            if (grp < NG)              // the second half's exponentials between the first half's products
#pragma unroll
                for (int j = grp * QC / NG; j < (grp + 1) * QC / NG; j++) p[1][j] = probs(st[j], x[j] + 8, c2[j], m[j], vs[1]);
#pragma unroll
            for (int k = 0; k < 4; k++)
#pragma unroll
                for (int j = 0; j < QC; j++) {
                    f32x4& o = st[j].o[grp % NG * 4 + k];
                    o = Mfma<M>::mma(vf[grp & 1][k], p[grp / NG][j], o);
                }
        }
    };
    if (n > 0) {                       // one block from here to the end of the loop: nothing older than its own loads is in flight where it begins
        ids(0);
        fetch(0);
        hole = bad;
        if (n > 1) ids(1);
        put(0, smem);
        if (n > 1) fetch(1);
        if (n > 2) ids(2);
        __syncthreads();
        for (int i = 0;;) {
            const int key0 = lo + i * 64;
            if (key0 < wend) compute(key0 + 64 > full || hole, smem + (i & 1) * kBuf, key0);
            if (++i >= n) break;
            hole = bad;
            put(i, smem + (i & 1) * kBuf);                 // last read before the barrier that ended tile i - 2
            if (i + 1 < n) fetch(i + 1);
            if (i + 2 < n) ids(i + 2);
            __syncthreads();
        }
    }
#pragma unroll
    for (int j = 0; j < QC; j++) {
        const float L = st[j].total(), mm = st[j].m(c2[j]);
        if (w0 + 16 * j + c >= rows) continue;
        int head;
        const int row = row_of(j, &head);
        const long at = (long)row * (a.H * t.G) + head;
        const float u = SCALED ? ref : 1.0f, un = st[j].unlift();
        if (t.splits == 1) {
            const float inv = L > 0.0f ? 1.0f / L : L;
            T* o = (T*)t.out + (long)row * t.o_row + (long)head * t.o_head;
#pragma unroll
            for (int k = 0; k < N; k++) {
                float y[4];
#pragma unroll
                for (int r = 0; r < 4; r++) y[r] = L == 0.0f ? 0.0f : st[j].o[k][r] * un * inv * u;
                store_cols<T, 4>(o + 16 * k + 4 * g, y);
            }
            if (t.lse && g == 0) t.lse[at] = L > 0.0f ? (mm + __builtin_amdgcn_logf(L)) * 0.69314718055994530942f : (L == 0.0f ? -kInf : L);
        } else {
            float* o = t.part + (at * t.splits + split) * D;
#pragma unroll
            for (int k = 0; k < N; k++) {
                f32x4 y = {0, 0, 0, 0};
                if (L != 0.0f) y = st[j].o[k] * un * u;
                *(f32x4*)(o + 16 * k + 4 * g) = y;
            }
            if (g == 0) t.part_ml[at * t.splits + split] = make_float2(mm, L);
        }
    }
}

// One workgroup per query row joins its key ranges: 4 waves take them in turn, 8 loads in flight each.
template <typename T, int D>
__global__ __launch_bounds__(256) void kv_attn_join_kernel(KvArgs a, AttnArgs t) {
    constexpr int E = D / 64;
    __shared__ float s_acc[4][D];
    const int heads = a.H * t.G, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long at = blockIdx.x;
    const int row = (int)(at / heads), head = (int)(at % heads);
    const int s = find_seq(a.q_start, a.n_seqs, row);
    if (s < 0 || s >= a.n_seqs) return;
    const Span sp = seq_span(a, s);
    if (row < sp.q0 || row >= sp.q0 + min(sp.n_new, t.max_new)) return;
    const float2 ml = lane < t.splits ? t.part_ml[at * t.splits + lane] : make_float2(-kInf, 0.0f);
    const float m = wave_max(ml.x), f = ml.x == -kInf ? 0.0f : __builtin_amdgcn_exp2f(ml.x - m);
    const float L = wave_sum(ml.y * f);
    float acc[E];
#pragma unroll
    for (int e = 0; e < E; e++) acc[e] = 0.0f;
    for (int i0 = wave * 8; i0 < t.splits; i0 += 32) {
        float o[8][E];
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int e = 0; e < E; e++) o[i][e] = t.part[(at * t.splits + min(i0 + i, t.splits - 1)) * D + lane * E + e];
#pragma unroll
        for (int i = 0; i < 8; i++) {                      // beyond the last range the weight is 0
            const float w = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), min(i0 + i, 63)));
#pragma unroll
            for (int e = 0; e < E; e++) acc[e] += i0 + i < t.splits ? w * o[i][e] : 0.0f;
        }
    }
#pragma unroll
    for (int e = 0; e < E; e++) s_acc[wave][lane * E + e] = acc[e];
    __syncthreads();
    if (threadIdx.x < D) {
        const int d = threadIdx.x;
        const float inv = L > 0.0f ? 1.0f / L : L;
        ((T*)t.out)[(long)row * t.o_row + (long)head * t.o_head + d] = (T)(((s_acc[0][d] + s_acc[1][d]) + (s_acc[2][d] + s_acc[3][d])) * inv);
    }
    if (t.lse && threadIdx.x == 0) t.lse[at] = L > 0.0f ? (m + __builtin_amdgcn_logf(L)) * 0.69314718055994530942f : (L == 0.0f ? -kInf : L);
}

KvArgs kv_args(const ss_kv_cache& c, const ss_kv_batch& b) {
    KvArgs a{};
    a.k = (char*)c.k; a.v = (char*)c.v; a.ks = (char*)c.k_scale; a.vs = (char*)c.v_scale;
    a.page_bytes = (unsigned)(c.page_stride * (c.kind == SS_KV_SAME ? 2 : 1));
    a.sc_stride = (unsigned)c.scale_stride;
    a.table = b.page_table; a.q_start = b.q_start; a.kv_len = b.kv_len; a.table_stride = b.table_stride;
    a.n_pages = c.n_pages; a.page_shift = __builtin_ctz((unsigned)c.page_size); a.H = c.n_kv_heads;
    a.max_pages = b.max_pages; a.n_seqs = b.n_seqs; a.n_tokens = b.n_tokens;
    return a;
}

// calls f(type tag, kind tag, dim tag) for the cache's combination
template <int V> using Int = std::integral_constant<int, V>;
template <typename F> void by_type(const ss_kv_cache& c, F f) {
    auto dim = [&](auto t, auto k) { c.head_dim == 64 ? f(t, k, Int<64>()) : f(t, k, Int<128>()); };
    const bool bf = c.dtype == SS_DTYPE_BF16;
    if (c.kind == SS_KV_SAME) { if (bf) dim(bf16(), Int<K_BF16>()); else dim(f16(), Int<K_F16>()); }
    else if (c.kind == SS_KV_E4M3) { if (bf) dim(bf16(), Int<K_E4M3>()); else dim(f16(), Int<K_E4M3>()); }
    else { if (bf) dim(bf16(), Int<K_I8>()); else dim(f16(), Int<K_I8>()); }
}

int up(long a, long b) { return (int)((a + b - 1) / b); }

}  // namespace

// log2 of the token rows of a workgroup, and workgroups side by side on them: enough workgroups to fill the card come first (small calls are all latency),
// then rows
static int kv_rows_per_group(const ss_kv_cache& c, const ss_kv_batch& b, int elements, int* side) {
    int shift = 0;
    while ((2 << shift) <= kMostRows && b.n_tokens >> (shift + 1) >= 512) shift++;
    *side = std::max(1, (int)std::min((long)up((2l * c.n_kv_heads * (c.head_dim / elements)) << shift, 256), 2048l / up(b.n_tokens, 1 << shift)));
    return shift;
}

void launch_kv_append(const ss_kv_cache& c, const ss_kv_batch& b, const ss_kv_rows& k, const ss_kv_rows& v, hipStream_t st) {
    if (b.n_tokens == 0 || b.n_seqs == 0) return;
    int side;
    const int shift = kv_rows_per_group(c, b, 16, &side);
    by_type(c, [&](auto t, auto kind, auto dim) {
        typedef decltype(t) T;
        kv_append_kernel<T, kind.value, dim.value><<<dim3(up(b.n_tokens, 1 << shift), side), 256, 0, st>>>(kv_args(c, b), shift, (const T*)k.p, k.row_stride, k.head_stride, (const T*)v.p,
                                                                                                     v.row_stride, v.head_stride);
    });
    SS_LAUNCH_CHECK();
}

void launch_kv_read(const ss_kv_cache& c, const ss_kv_batch& b, const ss_kv_rows& k, const ss_kv_rows& v, hipStream_t st) {
    if (b.n_tokens == 0 || b.n_seqs == 0) return;
    int side;
    const int shift = kv_rows_per_group(c, b, 8, &side);
    by_type(c, [&](auto t, auto kind, auto dim) {
        typedef decltype(t) T;
        auto go = [&](auto nt) {
            kv_read_kernel<T, kind.value, dim.value, nt.value><<<dim3(up(b.n_tokens, 1 << shift), side), 256, 0, st>>>(kv_args(c, b), shift, (T*)k.p, k.row_stride, k.head_stride,
                                                                                                                       (T*)v.p, v.row_stride, v.head_stride);
        };
        if (4l * b.n_tokens * c.n_kv_heads * c.head_dim > kNtBytes) go(std::true_type());
        else go(std::false_type());
    });
    SS_LAUNCH_CHECK();
}

KvPlan kv_attention_plan(const ss_kv_cache& c, const ss_kv_batch& b, int n_heads) {
    KvPlan p{};
    p.splits = 1;
    if (b.n_seqs == 0 || b.n_tokens == 0 || b.max_new == 0) return p;
    const bool join = (long)b.n_tokens * n_heads < 1 << 24;        // a workgroup a row: more than that is no grid, and fills the card without cuts
    const int G = n_heads / c.n_kv_heads;
    const long cap = (long)b.max_pages * c.page_size, keys = std::max(1l, b.max_len > 0 ? std::min((long)b.max_len, cap) : cap);
    const long rows = (long)b.max_new * G, pairs = (long)b.n_seqs * c.n_kv_heads;
    // One kernel takes the whole batch: a workgroup of the tile kernel that finds few rows leaves three waves to the loads alone.  The few-row kernel beside it for
    // the spans of up to 16 rows, with a join of its own, was slower wherever both apply: 32 spans of 1..20 rows over 448 keys 27 us against 17, over 16384 keys
    // 689 against 460
    p.tile = rows > 16;
    // Column tiles a wave.  4 read K and V out of LDS half as often, if they leave two workgroups a CU (head_dim 64, int8 codes and f16 tokens over 4096 keys:
    // 8 x 512 x 4 rows 206 us against 241, but 8 x 256 x 4 rows, one workgroup a CU, 173 against 137; over 512 keys 40 against 36.5 and 27 against 24); at head_dim
    // 128 they do not fit the registers
    const long wide = pairs * up(rows, 256);
    p.qc = rows <= 64 ? 1 : c.head_dim == 64 && rows >= 1024 && wide >= 512 ? 4 : 2;
    // As many key ranges as give the card 512 workgroups, none shorter than 512 keys (256 wanted: 1 x 128 x 4 rows over 16384 keys 87 us instead of 72; 1024 wanted:
    // 83, and 16 contexts of one token 546 instead of 504)
    const long groups = p.tile ? pairs * up(rows, 64 * p.qc) : pairs;
    const long n = !join ? 1 : std::max(1l, std::min({(512 + groups - 1) / groups, (keys + 511) / 512, 64l}));
    p.split_keys = (int)((keys + n * 128 - 1) / (n * 128) * 128);
    p.splits = (int)((keys + p.split_keys - 1) / p.split_keys);
    if (p.splits > 1) p.workspace = (int64_t)b.n_tokens * n_heads * p.splits * (c.head_dim + 2) * 4;
    return p;
}

void launch_kv_attention(const ss_kv_cache& c, const ss_kv_batch& b, const ss_kv_rows& q, int n_heads, float scale, bool causal, const ss_kv_rows& out,
                         float* lse, void* workspace, hipStream_t st) {
    if (b.n_tokens == 0 || b.n_seqs == 0 || b.max_new == 0) return;
    const KvPlan p = kv_attention_plan(c, b, n_heads);
    const KvArgs a = kv_args(c, b);
    AttnArgs t{};
    t.q = q.p; t.q_row = q.row_stride; t.q_head = q.head_stride;
    t.out = out.p; t.o_row = out.row_stride; t.o_head = out.head_stride;
    t.lse = lse; t.c2 = std::max(std::fabs(scale) * 1.44269504088896340736f, 1.17549435e-38f); t.neg = scale < 0.0f; t.G = n_heads / c.n_kv_heads; t.causal = causal; t.max_new = b.max_new;
    by_type(c, [&](auto tt, auto kind, auto dim) {
        typedef decltype(tt) T;
        constexpr int K = kind.value, D = dim.value;
        t.splits = p.splits; t.split_keys = p.split_keys;
        t.part = (float*)workspace;
        t.part_ml = (float2*)((float*)workspace + (size_t)b.n_tokens * n_heads * p.splits * D);
        if (!p.tile)
            kv_attn_few_kernel<T, K, D><<<dim3(b.n_seqs * p.splits, c.n_kv_heads), 256, 0, st>>>(a, t);
        else {
            auto go = [&](auto qc) {
                constexpr int QC = qc.value, smem = 2 * kTileBuf<D>;
                static std::atomic<uint64_t> once{0};
                once_per_device(once, [&] { SS_HIP(hipFuncSetAttribute((const void*)kv_attn_tile_kernel<T, K, D, QC>, hipFuncAttributeMaxDynamicSharedMemorySize, smem)); });
                t.nq = up((long)b.max_new * t.G, 64 * QC);
                kv_attn_tile_kernel<T, K, D, QC><<<(unsigned)((long)b.n_seqs * c.n_kv_heads * t.nq * p.splits), 256, smem, st>>>(a, t);
            };
            if (p.qc == 1) go(Int<1>());
            else if (p.qc == 2 || D == 128) go(Int<2>());
            else if constexpr (D == 64) go(Int<4>());
        }
        SS_LAUNCH_CHECK();
        if (p.splits > 1) {
            kv_attn_join_kernel<T, D><<<(unsigned)((long)b.n_tokens * n_heads), 256, 0, st>>>(a, t);
            SS_LAUNCH_CHECK();
        }
    });
}

}  // namespace ss
