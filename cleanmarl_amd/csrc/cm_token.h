// cm_token.h -- device helpers of the token-level losses (cm_token.hip): 16-byte pieces of a row of logits, running softmax sums.
#pragma once
#include "cm_common.h"
#include <float.h>
#include <math.h>

// ---------------------------------------------------------------- 16 bytes of a row
// A row may start at any multiple of its element size (odd vocabularies): the vector types carry the element's alignment only, and gfx950
// takes such global accesses as they are.
typedef unsigned tok_u4_a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned tok_u4_a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned tok_u4 __attribute__((ext_vector_type(4)));
typedef unsigned tok_u2_a1 __attribute__((ext_vector_type(2), aligned(1)));
typedef unsigned tok_u1_a1 __attribute__((aligned(1)));
typedef _Float16 tok_h2 __attribute__((ext_vector_type(2)));
typedef __bf16 tok_b2 __attribute__((ext_vector_type(2)));
typedef float tok_f2 __attribute__((ext_vector_type(2)));
typedef unsigned short tok_s2 __attribute__((ext_vector_type(2)));

struct TokF32 {
    typedef float elem;
    typedef tok_u4_a4 vec;
    static constexpr int W = 4;  // elements in 16 bytes
    static __device__ __forceinline__ float get(elem v) { return v; }
    static __device__ __forceinline__ elem put(float v) { return v; }
    static __device__ __forceinline__ void unpack(const tok_u4& r, float (&f)[W]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(r[i]);
    }
    static __device__ __forceinline__ tok_u4 pack(const float (&f)[W]) {
        tok_u4 r;
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = __float_as_uint(f[i]);
        return r;
    }
};
struct TokF16 {
    static constexpr unsigned NEG_INF = 0xfc00u;
    typedef _Float16 elem;
    typedef tok_u4_a2 vec;
    static constexpr int W = 8;
    static __device__ __forceinline__ float get(elem v) { return (float)v; }
    static __device__ __forceinline__ elem put(float v) { return (elem)v; }
    static __device__ __forceinline__ void unpack(const tok_u4& r, float (&f)[W]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const tok_h2 h = __builtin_bit_cast(tok_h2, (unsigned)r[i]);
            f[2 * i] = (float)h[0]; f[2 * i + 1] = (float)h[1];
        }
    }
    static __device__ __forceinline__ tok_u4 pack(const float (&f)[W]) {
        tok_u4 r;
#pragma unroll
        for (int i = 0; i < 4; ++i) { const tok_h2 h = {(_Float16)f[2 * i], (_Float16)f[2 * i + 1]}; r[i] = __builtin_bit_cast(unsigned, h); }
        return r;
    }
};
struct TokBF16 {
    static constexpr unsigned NEG_INF = 0xff80u;
    typedef __bf16 elem;
    typedef tok_u4_a2 vec;
    static constexpr int W = 8;
    static __device__ __forceinline__ float get(elem v) { return (float)v; }
    static __device__ __forceinline__ elem put(float v) { return (elem)v; }
    static __device__ __forceinline__ void unpack(const tok_u4& r, float (&f)[W]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(r[i] << 16); f[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u); }
    }
    static __device__ __forceinline__ tok_u4 pack(const float (&f)[W]) {  // v_cvt_pk_bf16_f32: round to nearest even
        tok_u4 r;
#pragma unroll
        for (int i = 0; i < 4; ++i) { const tok_f2 v = {f[2 * i], f[2 * i + 1]}; r[i] = __builtin_bit_cast(unsigned, __builtin_convertvector(v, tok_b2)); }
        return r;
    }
};

// W bytes of avail, as words
template <int W> struct TokAvail { unsigned a[W / 4]; };
template <int W>
__device__ __forceinline__ TokAvail<W> tok_avail(const uint8_t* av, int j) {
    TokAvail<W> r;
    if constexpr (W == 8) { const tok_u2_a1 v = *reinterpret_cast<const tok_u2_a1*>(av + j); r.a[0] = v[0]; r.a[1] = v[1]; }
    else r.a[0] = *reinterpret_cast<const tok_u1_a1*>(av + j);
    return r;
}
// elements [j, j + W) of a row, as they are in memory; places behind the vocabulary are -inf and unavailable
template <class T>
__device__ __forceinline__ tok_u4 tok_raw(const typename T::elem* row, int j, int V) {
    if (j + T::W <= V) return *reinterpret_cast<const typename T::vec*>(row + j);
    float f[T::W];
#pragma unroll
    for (int i = 0; i < T::W; ++i) { f[i] = -INFINITY; if (j + i < V) f[i] = T::get(row[j + i]); }
    return T::pack(f);
}
template <int W>
__device__ __forceinline__ TokAvail<W> tok_raw_avail(const uint8_t* av, int j, int V) {
    if (j + W <= V) return tok_avail<W>(av, j);
    TokAvail<W> r = {};
#pragma unroll
    for (int i = 0; i < W; ++i) if (j + i < V) r.a[i >> 2] |= (unsigned)av[j + i] << (8 * (i & 3));
    return r;
}
// unavailable places become -inf, whatever the memory holds there
template <int W>
__device__ __forceinline__ void tok_mask(const TokAvail<W>& a, float (&f)[W]) {
#pragma unroll
    for (int i = 0; i < W; ++i) f[i] = (a.a[i >> 2] >> (8 * (i & 3)) & 0xffu) ? f[i] : -INFINITY;
}
// the same on a packed piece
template <class T>
__device__ __forceinline__ void tok_mask_raw(const TokAvail<T::W>& a, tok_u4& r) {
    if constexpr (T::W == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = (a.a[0] >> (8 * i) & 0xffu) ? r[i] : 0xff800000u;
    } else {
        const tok_s2 inf = {(unsigned short)T::NEG_INF, (unsigned short)T::NEG_INF}, one = {1, 1};
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // two bytes -> two halves of all ones or all zeros
            const unsigned two = __builtin_amdgcn_perm(0u, a.a[i >> 1], i & 1 ? 0x0c030c02u : 0x0c010c00u);
            const tok_s2 keep = tok_s2{0, 0} - __builtin_elementwise_min(__builtin_bit_cast(tok_s2, two), one), v = __builtin_bit_cast(tok_s2, (unsigned)r[i]);
            r[i] = __builtin_bit_cast(unsigned, (v & keep) | (inf & ~keep));
        }
    }
    asm("" : "+v"(r));  // packed from here on: the compiler would keep the halves apart, in two registers
}
template <class T, bool AV>
__device__ __forceinline__ void tok_load(const typename T::elem* row, const uint8_t* av, int j, int V, float (&f)[T::W]) {
    T::unpack(tok_raw<T>(row, j, V), f);
    if constexpr (AV) tok_mask<T::W>(tok_raw_avail<T::W>(av, j, V), f);
}
// A long row is taken apart into a body of whole pieces that begin on a cache line (where a row of an odd vocabulary does not: pieces
// across lines cost a sixth of the bandwidth) and at most 127 bytes in front and 15 behind it, which the first threads take one element each.
struct TokShape {
    int head, full, edges;  // elements in front of the body, pieces in it, elements outside it
    __device__ __forceinline__ int edge(int t, int W) const { return t < head ? t : full * W + t; }                              // element of thread t < edges
    __device__ __forceinline__ int piece(int j, int W) const { return j < head || j >= head + full * W ? -1 : (j - head) / W; }  // piece of element j, -1: an edge
    __device__ __forceinline__ int edge_of(int j, int W) const { return j < head ? j : j - full * W; }
};
template <class T>
__device__ __forceinline__ TokShape tok_shape(const typename T::elem* row, int V, unsigned peel) {  // peel: 127, or 0 for none
    TokShape s;
    s.head = (int)((-(unsigned)reinterpret_cast<uintptr_t>(row) & peel) / sizeof(typename T::elem));
    s.full = (V - s.head) / T::W;
    s.edges = V - s.full * T::W;
    return s;
}
template <class T>
__device__ __forceinline__ void tok_store(typename T::elem* row, int j, int V, const float (&f)[T::W]) {
    constexpr int W = T::W;
    if (j + W <= V) {
        *reinterpret_cast<typename T::vec*>(row + j) = T::pack(f);
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i) if (j + i < V) row[j + i] = T::put(f[i]);
    }
}

// ---------------------------------------------------------------- running softmax sums
// m = max x, s = sum e^t, u = sum t2 e^t with t = (x - m) / T and t2 = t log2(e), the argument of v_exp_f32.  The difference is taken BEFORE
// the scaling: rows whose logits all sit at the type's lowest value are then uniform rows (t = 0) and not overflows, and for 16-bit
// logits the difference is nearly always exact.  m starts at -FLT_MAX and not at -inf: a row with nothing available keeps s = 0 (that is how it is
// recognised) without a NaN from inf - inf; a NaN or +inf in an available place ends in s = NaN, which is what it should do.
struct TokSum { float m, s, u; };

constexpr float TOK_LN2 = 0.6931471805599453f, TOK_FAR = -1e20f;  // products with e^t = 0 stay 0 where t2 is clamped to TOK_FAR
// 1 / T, and log2(e) / T in 64 bits and as the sum of two floats: rounded to one, it would move every logit of a row the same way, and what moves
// each log-probability by 1e-7 moves the sum over a long answer by 1e-4
// (lo > 0, so that its product with -inf is -inf)
struct TokScale { float nat, bin, lo; double full; };

__device__ __forceinline__ float tok_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// brings `a` to the larger maximum m
template <bool EN>
__device__ __forceinline__ void tok_raise(TokSum& a, float m, float bin) {
    const float d = (a.m - m) * bin, f = tok_exp2(d);
    if constexpr (EN) a.u = f * fmaf(fmaxf(d, TOK_FAR), a.s, a.u);  // sum (t + d) e^(t + d)
    a.s *= f;
    a.m = m;
}
template <bool EN>
__device__ __forceinline__ void tok_merge(TokSum& a, TokSum b, float bin) {
    const float m = fmaxf(a.m, b.m);
    tok_raise<EN>(a, m, bin);
    tok_raise<EN>(b, m, bin);
    a.s += b.s;
    if constexpr (EN) a.u += b.u;
}
template <bool EN, int W>
__device__ __forceinline__ void tok_add(TokSum& a, const float (&f)[W], float bin, float lo) {
    float m = a.m;
#pragma unroll
    for (int i = 0; i < W; ++i) m = fmaxf(m, f[i]);
    tok_raise<EN>(a, m, bin);
#pragma unroll
    for (int i = 0; i < W; ++i) {
        const float x = f[i] - m, d = fmaf(x, lo, x * bin), e = tok_exp2(d);
        a.s += e;
        if constexpr (EN) a.u = fmaf(e, fmaxf(d, TOK_FAR), a.u);
    }
}
template <bool EN, int G>
__device__ __forceinline__ void tok_group(TokSum& a, float bin) {  // over the G lanes of a group (a power of two, <= 64)
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) {
        TokSum b;
        b.m = __shfl_xor(a.m, o, 64);
        b.s = __shfl_xor(a.s, o, 64);
        b.u = EN ? __shfl_xor(a.u, o, 64) : 0.0f;
        tok_merge<EN>(a, b, bin);
    }
}
// over a workgroup of NW waves; `sh` holds NW entries and is free again when its next use has passed a barrier
template <bool EN, int NW>
__device__ __forceinline__ void tok_block(TokSum& a, float bin, TokSum* sh) {
    tok_group<EN, 64>(a, bin);
    if constexpr (NW > 1) {
        if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = a;
        __syncthreads();
        a = sh[threadIdx.x & (NW - 1)];
        tok_group<EN, NW>(a, bin);  // every group of NW lanes in the same order: one result
    }
}

// ---------------------------------------------------------------- the same, cheaper, for rows of ordinary size
// e^t = 2^(x c - M) with c = log2(e) / T: one fused multiply-add and one v_exp_f32.  M is any number near the row's maximum times c: floats have
// exponents to spare, so M follows the maximum only when that has run TOK_SLACK ahead, and the rescaling costs next to nothing.  M's own
// rounding is a factor common to every e^t of the row and cancels in e^t / s and in x c - M - log2 s.  What this form cannot do -- rows
// without a finite sum, logits so large that x c - M has no correct places, -inf beside an entropy (0 * -inf) -- shows in (M, s, u) and is done over with TokSum.
struct TokRun { float M, s, u; };
constexpr float TOK_START = -1.2676506e30f /* -2^100 */, TOK_SLACK = 16.0f, TOK_LARGE = 1048576.0f /* 2^20: the places behind x c - M are then at least 2^-4 */;

template <bool EN>
__device__ __forceinline__ void run_raise(TokRun& a, float M) {
    const float d = a.M - M, f = tok_exp2(d);
    if constexpr (EN) a.u = f * fmaf(fmaxf(d, TOK_FAR), a.s, a.u);
    a.s *= f;
    a.M = M;
}
// CLAMP: -inf among the logits is ordinary (unavailable columns), its product with e^t = 0 must not be NaN
template <bool EN, bool CLAMP, int W>
__device__ __forceinline__ void run_add(TokRun& a, const float (&f)[W], float c, float lo) {
    float m = f[0];
#pragma unroll
    for (int i = 1; i < W; ++i) m = fmaxf(m, f[i]);
    m *= c;
    if (m > a.M + TOK_SLACK) run_raise<EN>(a, m);
#pragma unroll
    for (int i = 0; i < W; ++i) {
        float t = fmaf(f[i], c, -a.M);
        t = fmaf(f[i], lo, t);
        const float e = tok_exp2(t);
        a.s += e;
        if constexpr (EN) a.u = fmaf(e, CLAMP ? fmaxf(t, TOK_FAR) : t, a.u);
    }
}
template <bool EN>
__device__ __forceinline__ void run_merge(TokRun& a, TokRun b) {
    const float M = fmaxf(a.M, b.M);
    run_raise<EN>(a, M);
    run_raise<EN>(b, M);
    a.s += b.s;
    if constexpr (EN) a.u += b.u;
}
template <bool EN, int G>
__device__ __forceinline__ void run_group(TokRun& a) {
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) {
        TokRun b;
        b.M = __shfl_xor(a.M, o, 64);
        b.s = __shfl_xor(a.s, o, 64);
        b.u = EN ? __shfl_xor(a.u, o, 64) : 0.0f;
        run_merge<EN>(a, b);
    }
}
template <bool EN, int NW>
__device__ __forceinline__ void run_block(TokRun& a, TokRun* sh) {  // sh: as in tok_block
    run_group<EN, 64>(a);
    if constexpr (NW > 1) {
        if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = a;
        __syncthreads();
        a = sh[threadIdx.x & (NW - 1)];
        run_group<EN, NW>(a);
    }
}
template <bool EN>
__device__ __forceinline__ bool run_ordinary(const TokRun& a) {
    return a.s > 0.0f && a.s < INFINITY && fabsf(a.M) <= TOK_LARGE && (!EN || fabsf(a.u) < INFINITY);
}

// The gradients do without `lo`: 2^(x c - M) / s' with the s' that makes the two agree near the maximum, where x is M / c
__device__ __forceinline__ float run_sum(const TokRun& z, const TokScale& c) { return z.s * tok_exp2(-z.M * (c.lo / c.bin)); }

// log-probability of a logit x from the row's sums: t in 64 bits (one rounding at the end), log s in 32, or in 64 for sums of many of them
__device__ __forceinline__ float run_logp(float x, float M, float logs, const TokScale& c) { return (float)(((double)x * c.full - (double)M) * 0.6931471805599453 - (double)logs); }
__device__ __forceinline__ float tok_logp(float x, float m, float logs, const TokScale& c) { return (float)(((double)x - (double)m) * c.full * 0.6931471805599453 - (double)logs); }

// ---------------------------------------------------------------- what a row's backward needs
// dx_j = a [j = token] - b p_j + h p_j (log p_j + H), all already divided by T; p_j = e^t rs, log p_j + H = t + K
struct TokGrad { float m, rs, K, a, b, h; int tok; };

template <bool HE, int W>
__device__ __forceinline__ void tok_grad_rest(const float (&f)[W], const TokGrad& g, float bin, float (&d)[W]) {  // without the token's own term
    const float brs = -g.b * g.rs, hrs = g.h * g.rs;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        const float t = (f[i] - g.m) * bin, e = tok_exp2(t);
        if constexpr (HE) d[i] = e * fmaf(hrs, fmaxf(fmaf(t, TOK_LN2, g.K), TOK_FAR), brs);  // e = 0 where t is clamped
        else d[i] = e * brs;
    }
}
template <bool HE, int W>
__device__ __forceinline__ void tok_grad(const float (&f)[W], int j, const TokGrad& g, float bin, float (&d)[W]) {
    tok_grad_rest<HE>(f, g, bin, d);
    if ((unsigned)(g.tok - j) < (unsigned)W) {
#pragma unroll
        for (int i = 0; i < W; ++i) if (j + i == g.tok) d[i] += g.a;
    }
}

// The same in the form of TokRun: 2^(x c - M) rs.  16-bit gradients take the row's factor into the exponent (its rounding there, at most
// 2^-16 of the value, is nothing beside theirs) and its sign into the packed pieces, unless M is so large that its places would be lost.
struct RunGrad { float M, brs, hrs, K, shift; unsigned sign; bool fold; };
template <class T, bool HE>
__device__ __forceinline__ RunGrad run_grad_row(float M, float s, float K, float b, float h) {
    RunGrad g;
    const float rs = 1.0f / s;
    g.M = M; g.K = K; g.brs = -b * rs; g.hrs = h * rs;
    g.shift = log2f(fabsf(b)) - log2f(s) - M;  // b = 0: -inf, and every 2^ is 0
    g.sign = (__float_as_uint(-b) >> 31) ? 0x80008000u : 0u;
    g.fold = !HE && T::W == 8 && fabsf(M) <= 128.0f && !(fabsf(g.shift) > 256.0f && b != 0.0f);
    return g;
}
template <class T, bool HE>
__device__ __forceinline__ tok_u4 run_grad(const tok_u4& raw, const RunGrad& g, float c) {
    float f[T::W], d[T::W];
    T::unpack(raw, f);
    if (!HE && T::W == 8 && g.fold) {
#pragma unroll
        for (int i = 0; i < T::W; ++i) d[i] = tok_exp2(fmaf(f[i], c, g.shift));
        tok_u4 r = T::pack(d);
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] ^= g.sign;
        return r;
    }
#pragma unroll
    for (int i = 0; i < T::W; ++i) {
        const float t = fmaf(f[i], c, -g.M), e = tok_exp2(t);
        if constexpr (HE) {
            d[i] = e * fmaf(g.hrs, fmaxf(fmaf(t, TOK_LN2, g.K), TOK_FAR), g.brs);  // e = 0 where it is clamped
        } else d[i] = e * g.brs;
    }
    return T::pack(d);
}
template <bool HE>
__device__ __forceinline__ float run_grad_one(float x, const RunGrad& g, float c) {
    const float t = fmaf(x, c, -g.M), e = tok_exp2(t);
    if constexpr (HE) return e * fmaf(g.hrs, fmaxf(fmaf(t, TOK_LN2, g.K), TOK_FAR), g.brs);
    else return e * g.brs;
}

// ---------------------------------------------------------------- arguments of every kernel of the family
enum { TOK_LOGP = 0, TOK_BWD = 1, TOK_POLICY = 2 };
constexpr int TOK_STATS = CM_NUM_STATS, TOK_MAX_GRID = 2048;

struct TokArgs {
    const void* logits; int64_t ld; const uint8_t* avail; int64_t avail_ld; const void* token; int token_bytes;
    int64_t rows; int V; TokScale c;
    float *logp, *entropy; double* logp64; float2* keep;                                     // forward: keep = (m, s), (M, -s) in the form of TokRun, s = 0 for a row that is left out
    const float2* keep_in; const float *entropy_in, *d_logp, *d_entropy;     // backward
    void* dlogits; int64_t dld;
    const float *logp_old, *adv, *logp_ref, *weight; float lo, hi, kl_coef, ent_coef; double* part;  // policy
    float *g_out, *h_out;                                                    // policy in two launches: the factors of each row for the second
    float4* split; int segs;                                                 // few long rows: partial sums (M, s, u, token's logit) of segs segments a row
    unsigned peel;                                                           // long rows: tok_shape
    float* stats;                                                            // policy: where a launch of one workgroup writes its sums; preference: see pairs
    const double* pair_part; int pairs;                                      // preference, backward: the first workgroup adds up what k_pref_pair left of each pair
    const int32_t* range_lo; const int32_t* range_hi;                        // preference: only the rows [*range_lo, *range_hi) are touched
};
constexpr int TOK_SPLIT_ROWS = 64, TOK_SPLIT_SEGS = 32;  // the most rows that are split, the most segments of one
constexpr int TOK_HELD = 1024 * 16 * 16;                 // a policy loss holds rows of up to this many bytes, at least
constexpr size_t TOK_ROW_BYTES = sizeof(float2) + 3 * sizeof(float);
constexpr size_t TOK_SPLIT_BYTES = (size_t)TOK_SPLIT_ROWS * TOK_SPLIT_SEGS * sizeof(float4);
// sums of n partial rows of statistics in a fixed order, by a workgroup of NT threads (one call per kernel)
template <int NT>
__device__ __forceinline__ void tok_sum_stats(const double* part, int n, float* stats) {
    constexpr int GROUPS = NT / TOK_STATS, BATCH = 8;
    __shared__ double sh[NT / 64][TOK_STATS];
    const int c = threadIdx.x % TOK_STATS, g = threadIdx.x / TOK_STATS;
    double s = 0.0;
    for (int i0 = g; i0 < n; i0 += GROUPS * BATCH) {  // a batch of loads in flight
        double v[BATCH];
#pragma unroll
        for (int q = 0; q < BATCH; ++q) v[q] = i0 + q * GROUPS < n ? part[(int64_t)(i0 + q * GROUPS) * TOK_STATS + c] : 0.0;
#pragma unroll
        for (int q = 0; q < BATCH; ++q) s += v[q];
    }
#pragma unroll
    for (int o = 32; o >= TOK_STATS; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) < TOK_STATS) sh[threadIdx.x >> 6][c] = s;
    __syncthreads();
    if (threadIdx.x < TOK_STATS) {
        double t = 0.0;
        for (int i = 0; i < NT / 64; ++i) t += sh[i][c];
        stats[c] = (float)t;
    }
}
// launches the kernels of one type; `scratch`: TOK_SPLIT_BYTES for partial sums (TOK_LOGP), TOK_ROW_BYTES a row (TOK_POLICY, more than
// TOK_HELD bytes of logits); returns the number of partial rows of statistics (TOK_POLICY)
int tok_launch_f32(TokArgs a, int mode, bool en, void* scratch, hipStream_t s);
int tok_launch_f16(TokArgs a, int mode, bool en, void* scratch, hipStream_t s);
int tok_launch_bf16(TokArgs a, int mode, bool en, void* scratch, hipStream_t s);
