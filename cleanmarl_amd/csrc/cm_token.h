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

// elements [j, j + W) of a row as floats; places behind the vocabulary and unavailable ones are -inf, whatever the memory holds there
template <class T, bool AV>
__device__ __forceinline__ void tok_load(const typename T::elem* __restrict__ row, const uint8_t* __restrict__ av, int j, int V, float (&f)[T::W]) {
    constexpr int W = T::W;
    if (j + W <= V) {
        const tok_u4 raw = *reinterpret_cast<const typename T::vec*>(row + j);
        T::unpack(raw, f);
        if constexpr (AV) {
            unsigned a[2];
            if constexpr (W == 8) { const tok_u2_a1 r = *reinterpret_cast<const tok_u2_a1*>(av + j); a[0] = r[0]; a[1] = r[1]; }
            else a[0] = *reinterpret_cast<const tok_u1_a1*>(av + j);
#pragma unroll
            for (int i = 0; i < W; ++i) f[i] = (a[i >> 2] >> (8 * (i & 3)) & 0xffu) ? f[i] : -INFINITY;
        }
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i) {
            f[i] = -INFINITY;
            if (j + i < V && (!AV || av[j + i])) f[i] = T::get(row[j + i]);
        }
    }
}
template <class T>
__device__ __forceinline__ void tok_store(typename T::elem* __restrict__ row, int j, int V, const float (&f)[T::W]) {
    constexpr int W = T::W;
    if (j + W <= V) {
        *reinterpret_cast<typename T::vec*>(row + j) = T::pack(f);
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i) if (j + i < V) row[j + i] = T::put(f[i]);
    }
}

// ---------------------------------------------------------------- running softmax sums
// m = max x, s = sum e^t, u = sum t e^t with t = (x - m) / T.  The difference is taken BEFORE the scaling: rows whose logits all sit at
// the type's lowest value are then uniform rows (t = 0) and not overflows, and for 16-bit logits the difference is nearly always exact.
// m starts at -FLT_MAX and not at -inf: a row with nothing available keeps s = 0 (that is how it is recognised) without a NaN from inf - inf;
// a NaN or +inf in an available place ends in s = NaN, which is what it should do.
struct TokSum { float m, s, u; };

#define TOK_LOG2E 1.4426950408889634f
struct TokScale { float nat, bin; };  // 1 / T for natural logarithms, log2(e) / T for v_exp_f32

__device__ __forceinline__ float tok_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// brings `a` to the larger maximum m
template <bool EN>
__device__ __forceinline__ void tok_raise(TokSum& a, float m, const TokScale& c) {
    const float f = tok_exp2((a.m - m) * c.bin);
    if constexpr (EN) a.u = f * fmaf(fmaxf((a.m - m) * c.nat, -1e30f), a.s, a.u);  // sum (t - d) e^(t - d); the clamp keeps 0 * inf out
    a.s *= f;
    a.m = m;
}
template <bool EN>
__device__ __forceinline__ void tok_merge(TokSum& a, TokSum b, const TokScale& c) {
    const float m = fmaxf(a.m, b.m);
    tok_raise<EN>(a, m, c);
    tok_raise<EN>(b, m, c);
    a.s += b.s;
    if constexpr (EN) a.u += b.u;
}
template <bool EN, int W>
__device__ __forceinline__ void tok_add(TokSum& a, const float (&f)[W], const TokScale& c) {
    float m = a.m;
#pragma unroll
    for (int i = 0; i < W; ++i) m = fmaxf(m, f[i]);
    tok_raise<EN>(a, m, c);
#pragma unroll
    for (int i = 0; i < W; ++i) {
        const float d = f[i] - m, e = tok_exp2(d * c.bin);
        a.s += e;
        if constexpr (EN) a.u = fmaf(e, fmaxf(d * c.nat, -1e30f), a.u);
    }
}
template <bool EN, int G>
__device__ __forceinline__ void tok_group(TokSum& a, const TokScale& c) {  // over the G lanes of a group (a power of two, <= 64)
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) {
        TokSum b;
        b.m = __shfl_xor(a.m, o, 64);
        b.s = __shfl_xor(a.s, o, 64);
        b.u = EN ? __shfl_xor(a.u, o, 64) : 0.0f;
        tok_merge<EN>(a, b, c);
    }
}
// over a workgroup of NW waves; `sh` holds NW entries and is free again when its next use has passed a barrier
template <bool EN, int NW>
__device__ __forceinline__ void tok_block(TokSum& a, const TokScale& c, TokSum* sh) {
    tok_group<EN, 64>(a, c);
    if constexpr (NW > 1) {
        if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = a;
        __syncthreads();
        a = sh[0];
#pragma unroll
        for (int w = 1; w < NW; ++w) tok_merge<EN>(a, sh[w], c);  // every thread in the same order: one result
    }
}

// ---------------------------------------------------------------- what a row's backward needs
// dx_j = a [j = token] - b p_j + h p_j (log p_j + H), all already divided by T; p_j = e^t / s
struct TokGrad { float m, rs, logs, H, a, b, h; int tok; };

template <class T, bool HE>
__device__ __forceinline__ void tok_grad(const float (&f)[T::W], int j, const TokGrad& g, const TokScale& c, float (&d)[T::W]) {
#pragma unroll
    for (int i = 0; i < T::W; ++i) {
        const float t = f[i] - g.m, p = tok_exp2(t * c.bin) * g.rs;
        float v = -g.b * p;
        if constexpr (HE) v = fmaf(g.h * p, fmaxf(t * c.nat, -1e30f) - g.logs + g.H, v);  // p = 0 where t is clamped
        d[i] = (j + i == g.tok) ? v + g.a : v;
    }
}
