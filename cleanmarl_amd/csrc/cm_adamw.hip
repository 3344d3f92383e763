// cm_adamw.hip -- AdamW over a list of tensors in one step, states in 32 or in 8 bits.
//
// The update rule is that of cm_optim.hip's CM_OPT_ADAMW (cleanmarl/mappo_multienvs.py:578-594 with optimizer = AdamW), for parameters that
// are the caller's own tensors (a model's matrices, vectors and odd ones) instead of one flat fp32 vector:
//   g' = g * grad_scale * min(1, max_norm / (|g| + 1e-6))
//   m = b1 m + (1 - b1) g'      v = b2 v + ((1 - b2) g') g'
//   p = p (1 - lr wd) - (lr / (1 - b1^t)) * (m / (sqrt v / sqrt(1 - b2^t) + eps))
// in fp32, every product and sum rounded by itself (no contraction: the same bits whatever surrounds the code), parameters rounded once to
// their type.  States live in two arenas of 256-element blocks; a tensor's states start at a block of their own, so a block never holds
// two tensors and an arena is one allocation to checkpoint.  With 8 bits a block keeps m and sqrt v as e4m3 codes times a scale that maps
// its largest magnitude to 448.  sqrt v and not v: the code's 2^-9 .. 448 then spans 11 decades of v.  A sqrt v above zero keeps at least
// the smallest code: rounded to zero it would leave eps alone under a moment m that was not.  The update itself uses the new moments
// before they are rounded.  An element whose moments have left fp32 has no part in its block's scales: sqrt v is a NaN code, read as infinity
// (its steps are 0 from then on, as with 32 bits, or NaN if m is none that is finite), m a zero or a NaN code.
#include "cm_common.h"
#include <float.h>
#include <math.h>

namespace {

constexpr int AW_BLOCK = 256, AW_TABLE = 88, AW_NT = 256, AW_CHUNK = 16;  // elements of a block; tensors of one launch; threads; blocks of one workgroup
constexpr int AW_NORM_GRID = 1024, AW_MOST = (1 << 24) - 1;  // the most workgroups of a launch: it ends at 2^32 threads

struct AwEntry { void* p; const void* g; void* copy; int64_t n; int first; int block; };  // first: the tensor's first workgroup; block: its first state block
struct AwTable { AwEntry e[AW_TABLE]; uint8_t kinds[AW_TABLE]; int count; };               // kinds: dtype of param | grad << 2 | copy << 4
struct AwArgs {
    void *m, *v; float* scale;
    float omb1, beta1, omb2, beta2, eps, wdf, step_size, inv_bc2, grad_scale;
    double lr, b1, b2;          // step_dev: the factors that depend on the step are made on the device
    const int32_t* step_dev;
    const float* coef;          // clip coefficient of this step; NULL: no clipping, or
    const double* parts; int nparts; float max_norm; float* norm;  // the few partial sums that it is made of (nparts > 0)
};
constexpr int AW_FEW = 256;     // partial sums that every wave adds up by itself: a launch less for short lists

typedef float aw_f4 __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned aw_u4 __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned aw_u2 __attribute__((ext_vector_type(2)));
typedef _Float16 aw_h2 __attribute__((ext_vector_type(2)));
typedef __bf16 aw_b2 __attribute__((ext_vector_type(2)));
typedef float aw_f2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float aw_coef(float norm, float max_norm) {
#pragma clang fp contract(off)
    const float c = max_norm / (norm + 1e-6f);
    return c < 1.0f || c != c ? c : 1.0f;  // a norm that is NaN reaches the parameters
}
__device__ __forceinline__ float aw_get(const void* p, int64_t i, int dt) {
    if (dt == CM_DTYPE_F32) return reinterpret_cast<const float*>(p)[i];
    if (dt == CM_DTYPE_F16) return (float)reinterpret_cast<const _Float16*>(p)[i];
    return (float)reinterpret_cast<const __bf16*>(p)[i];
}
__device__ __forceinline__ void aw_put(void* p, int64_t i, int dt, float v) {
    if (dt == CM_DTYPE_F32) reinterpret_cast<float*>(p)[i] = v;
    else if (dt == CM_DTYPE_F16) reinterpret_cast<_Float16*>(p)[i] = (_Float16)v;
    else reinterpret_cast<__bf16*>(p)[i] = (__bf16)v;
}
// eight elements from i on; k of them exist
__device__ __forceinline__ void aw_load(const void* p, int64_t i, int dt, int k, float (&f)[8]) {
    if (k >= 8) {
        if (dt == CM_DTYPE_F32) {
            const aw_f4* q = reinterpret_cast<const aw_f4*>(reinterpret_cast<const float*>(p) + i);
            const aw_f4 r0 = q[0], r1 = q[1];
#pragma unroll
            for (int j = 0; j < 4; ++j) { f[j] = r0[j]; f[4 + j] = r1[j]; }
        } else {
            const aw_u4 r = *reinterpret_cast<const aw_u4*>(reinterpret_cast<const uint16_t*>(p) + i);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if (dt == CM_DTYPE_F16) { const aw_h2 h = __builtin_bit_cast(aw_h2, (unsigned)r[q]); f[2 * q] = (float)h[0]; f[2 * q + 1] = (float)h[1]; }
                else { f[2 * q] = __uint_as_float(r[q] << 16); f[2 * q + 1] = __uint_as_float(r[q] & 0xffff0000u); }
            }
        }
    } else {
#pragma unroll
        for (int q = 0; q < 8; ++q) f[q] = q < k ? aw_get(p, i + q, dt) : 0.0f;
    }
}
__device__ __forceinline__ void aw_store(void* p, int64_t i, int dt, int k, const float (&f)[8]) {
    if (k >= 8) {
        if (dt == CM_DTYPE_F32) {
            aw_f4* q = reinterpret_cast<aw_f4*>(reinterpret_cast<float*>(p) + i);
            q[0] = aw_f4{f[0], f[1], f[2], f[3]}; q[1] = aw_f4{f[4], f[5], f[6], f[7]};
        } else {
            aw_u4 r;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if (dt == CM_DTYPE_F16) r[q] = __builtin_bit_cast(unsigned, aw_h2{(_Float16)f[2 * q], (_Float16)f[2 * q + 1]});
                else r[q] = __builtin_bit_cast(unsigned, __builtin_convertvector(aw_f2{f[2 * q], f[2 * q + 1]}, aw_b2));
            }
            *reinterpret_cast<aw_u4*>(reinterpret_cast<uint16_t*>(p) + i) = r;
        }
    } else {
#pragma unroll
        for (int q = 0; q < 8; ++q) if (q < k) aw_put(p, i + q, dt, f[q]);
    }
}

// the tensor that workgroup `wg` of a launch works on: the last one whose first workgroup is not behind it (uniform: scalar code)
__device__ __forceinline__ int aw_find(const AwTable& t, int wg) {
    int lo = 0, hi = t.count;
    while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (t.e[mid].first <= wg) lo = mid; else hi = mid; }
    return lo;
}

// maximum over the 32 lanes that hold one block: four rotations within the rows of 16 lanes, then the other row
template <int ROR> __device__ __forceinline__ float aw_max_ror(float v) {
    return fmaxf(v, __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), 0x120 + ROR, 0xf, 0xf, true)));
}
__device__ __forceinline__ float aw_block_max(float v) {
    v = aw_max_ror<8>(v); v = aw_max_ror<4>(v); v = aw_max_ror<2>(v); v = aw_max_ror<1>(v);
    return fmaxf(v, __uint_as_float(__builtin_amdgcn_ds_swizzle(__float_as_uint(v), 0x401f)));
}

// Half a wave per block of 256 elements, eight to a lane: 16-byte accesses of 16-bit tensors, one 8-byte access of a block's codes.  537 M bf16
// parameters with 8-bit states: 1.14 ms a pass among others, 4.7 TB/s (1.17 to 1.24 behind an idle GPU; a wave per block, four elements to a lane:
// 1.45 ms); 268 M fp32 masters, bf16 gradients and copies, 32-bit states and clipping: 1.65 ms, 4.9 TB/s of the bytes that both sweeps read and write.
// What is left to a large copy's 5.0 TB/s is the correctly rounded square root and division, some 25 instructions each for an element.
template <int BITS>
__global__ __launch_bounds__(AW_NT) void k_adamw(const AwTable t, const AwArgs a) {
#pragma clang fp contract(off)
    const int ti = aw_find(t, blockIdx.x);
    const AwEntry e = t.e[ti];
    const int pd = t.kinds[ti] & 3, gd = (t.kinds[ti] >> 2) & 3, cd = (t.kinds[ti] >> 4) & 3;
    float step_size = a.step_size, inv_bc2 = a.inv_bc2;
    if (a.step_dev) {
        const double s = (double)a.step_dev[0];
        step_size = (float)(a.lr / (1.0 - pow(a.b1, s)));
        inv_bc2 = (float)(1.0 / sqrt(1.0 - pow(a.b2, s)));
    }
    float coef = a.coef ? a.coef[0] : 1.0f;
    if (a.nparts) {
        double s = 0.0;
        for (int q = threadIdx.x & 63; q < a.nparts; q += 64) s += a.parts[q];
        const float norm = (float)sqrt(cm_wave_sum_d(s));
        coef = aw_coef(norm, a.max_norm);
        if (blockIdx.x == 0 && threadIdx.x == 0) { a.norm[0] = norm; a.norm[1] = coef; }
    }
    const int half = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t blocks = (e.n + AW_BLOCK - 1) / AW_BLOCK, b0 = (int64_t)(blockIdx.x - e.first) * AW_CHUNK;
    const int64_t b1 = min(b0 + AW_CHUNK, blocks);
    for (int64_t b = b0 + half; b < b1; b += AW_NT / 32) {
        const int64_t i = b * AW_BLOCK + 8 * lane, at = (e.block + b) * AW_BLOCK + 8 * lane;
        const int64_t left = e.n - i;
        const int k = left >= 8 ? 8 : (left > 0 ? (int)left : 0);
        float p[8], g[8], m[8], r[8];
        aw_u2 cm = {}, cr = {};
        float sm = 0.0f, sr = 0.0f;
        if (BITS == 8) {
            cm = reinterpret_cast<const aw_u2*>(a.m)[at / 8]; cr = reinterpret_cast<const aw_u2*>(a.v)[at / 8];
            sm = a.scale[2 * (e.block + b)]; sr = a.scale[2 * (e.block + b) + 1];
        }
        aw_load(e.p, i, pd, k, p);
        aw_load(e.g, i, gd, k, g);
        if (BITS == 32) {
            aw_load(a.m, at, CM_DTYPE_F32, 8, m);
            aw_load(a.v, at, CM_DTYPE_F32, 8, r);
        } else {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const aw_f2 m0 = __builtin_amdgcn_cvt_pk_f32_fp8(cm[q], false), m1 = __builtin_amdgcn_cvt_pk_f32_fp8(cm[q], true);
                const aw_f2 r0 = __builtin_amdgcn_cvt_pk_f32_fp8(cr[q], false), r1 = __builtin_amdgcn_cvt_pk_f32_fp8(cr[q], true);
                m[4 * q] = m0[0] * sm; m[4 * q + 1] = m0[1] * sm; m[4 * q + 2] = m1[0] * sm; m[4 * q + 3] = m1[1] * sm;
                r[4 * q] = r0[0] * sr; r[4 * q + 1] = r0[1] * sr; r[4 * q + 2] = r1[0] * sr; r[4 * q + 3] = r1[1] * sr;
            }
#pragma unroll
            for (int q = 0; q < 8; ++q) r[q] = fminf(r[q], INFINITY);  // NaN is infinity, numbers stay
        }
        float tm = 0.0f, tr = 0.0f;
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            const float gi = (g[q] * a.grad_scale) * coef;
            m[q] = a.beta1 * m[q] + a.omb1 * gi;
            const float v = a.beta2 * (BITS == 32 ? r[q] : r[q] * r[q]) + (a.omb2 * gi) * gi;
            const float root = sqrtf(v);
            p[q] = p[q] * a.wdf - step_size * (m[q] / (root * inv_bc2 + a.eps));
            if (BITS == 32) r[q] = v;
            else { r[q] = root; tm = fmaxf(tm, fabsf(m[q])); tr = fmaxf(tr, root); }
        }
        aw_store(e.p, i, pd, k, p);
        if (e.copy) aw_store(e.copy, i, cd, k, p);
        if (BITS == 32) {
            aw_store(a.m, at, CM_DTYPE_F32, k, m);
            aw_store(a.v, at, CM_DTYPE_F32, k, r);
        } else {
            const float f = 1.0f / 448.0f, least = 7.888609052210118e-31f;  // 2^-100: below it a scale would lose bits, and what it scales is nothing
            tm = aw_block_max(tm); tr = aw_block_max(tr);
            if (!(tm < INFINITY && tr < INFINITY)) {  // rare, and the same for all lanes of the block
                tm = tr = 0.0f;
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    const bool finite = fabsf(m[q]) < INFINITY;
                    if (!(finite && r[q] < INFINITY)) { m[q] = finite ? 0.0f : NAN; r[q] = NAN; }
                    tm = fmaxf(tm, fabsf(m[q])); tr = fmaxf(tr, r[q]);
                }
                tm = aw_block_max(tm); tr = aw_block_max(tr);
            }
            sm = tm < least ? 0.0f : tm * f; sr = tr < least ? 0.0f : tr * f;
            const float bm = sm > 0.0f ? 1.0f / sm : 0.0f, br = sr > 0.0f ? 1.0f / sr : 0.0f;
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                m[q] = m[q] * bm;
                r[q] = r[q] * br;
                r[q] = (r[q] > 0.0f && r[q] < 0.001953125f) ? 0.001953125f : r[q];
            }
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                int x = __builtin_amdgcn_cvt_pk_fp8_f32(m[4 * q], m[4 * q + 1], 0, false), y = __builtin_amdgcn_cvt_pk_fp8_f32(r[4 * q], r[4 * q + 1], 0, false);
                cm[q] = __builtin_amdgcn_cvt_pk_fp8_f32(m[4 * q + 2], m[4 * q + 3], x, true); cr[q] = __builtin_amdgcn_cvt_pk_fp8_f32(r[4 * q + 2], r[4 * q + 3], y, true);
            }
            // the places behind the tensor hold zeros and stay zero: m = v = g = 0 there
            reinterpret_cast<aw_u2*>(a.m)[at / 8] = cm; reinterpret_cast<aw_u2*>(a.v)[at / 8] = cr;
            if (lane == 0) { a.scale[2 * (e.block + b)] = sm; a.scale[2 * (e.block + b) + 1] = sr; }
        }
    }
}

// sums of squares of the scaled gradients in 64 bits: one partial per workgroup, which takes a fixed set of chunks of the launch's tensors
__global__ __launch_bounds__(AW_NT) void k_adamw_norm(const AwTable t, int chunks, float grad_scale, double* __restrict__ part) {
    __shared__ double sh[AW_NT / 64];
    double s = 0.0;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
        const int ti = aw_find(t, c);
        const AwEntry e = t.e[ti];
        const int gd = (t.kinds[ti] >> 2) & 3;
        const int64_t i0 = (int64_t)(c - e.first) * AW_CHUNK * AW_BLOCK;
        for (int b = threadIdx.x >> 5; b < AW_CHUNK; b += AW_NT / 32) {
            const int64_t i = i0 + b * AW_BLOCK + 8 * (lane & 31), left = e.n - i;
            if (left <= 0) continue;
            float g[8];
            aw_load(e.g, i, gd, left >= 8 ? 8 : (int)left, g);
#pragma unroll
            for (int q = 0; q < 8; ++q) { const double d = (double)(g[q] * grad_scale); s = fma(d, d, s); }
        }
    }
    s = cm_wave_sum_d(s);
    if (lane == 0) sh[wave] = s;
    __syncthreads();
    if (threadIdx.x == 0) { for (int w = 1; w < AW_NT / 64; ++w) s += sh[w]; part[blockIdx.x] = s; }
}
__global__ __launch_bounds__(1024) void k_adamw_coef(const double* __restrict__ part, int n, float max_norm, float* __restrict__ norm) {
    __shared__ double sh[16];
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += 1024) s += part[i];
    s = cm_wave_sum_d(s);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int w = 1; w < 16; ++w) s += sh[w];
    const float x = (float)sqrt(s);
    norm[0] = x;
    norm[1] = aw_coef(x, max_norm);
}

inline size_t aw_elem(int dtype) { return dtype == CM_DTYPE_F32 ? 4 : 2; }
inline bool aw_dtype(int d) { return d == CM_DTYPE_F32 || d == CM_DTYPE_F16 || d == CM_DTYPE_BF16; }

}  // namespace

extern "C" int64_t cm_adamw_state_blocks(int64_t n) { return n > 0 ? (n + AW_BLOCK - 1) / AW_BLOCK : 0; }
extern "C" size_t cm_adamw_workspace_bytes(int n_tensors) {
    if (n_tensors < 1) return 0;
    return (size_t)((n_tensors + AW_TABLE - 1) / AW_TABLE) * AW_NORM_GRID * sizeof(double);
}

extern "C" int cm_adamw_multi_step(const cm_adamw_tensor_t* tensors, int n_tensors, const cm_adamw_t* o, cm_stream_t stream) {
    CM_REQUIRE(o && n_tensors >= 0 && (tensors || n_tensors == 0), "cm_adamw_multi_step: NULL arguments");
    CM_REQUIRE(o->state_bits == 32 || o->state_bits == 8, "cm_adamw_multi_step: state_bits=%d (8 or 32)", (int)o->state_bits);
    CM_REQUIRE(o->step_dev || o->step >= 1, "cm_adamw_multi_step: step=%d", (int)o->step);
    CM_REQUIRE(o->exp_avg && o->exp_avg_sq && (o->state_bits == 32 || o->scale), "cm_adamw_multi_step: NULL state arena");
    CM_REQUIRE(((reinterpret_cast<uintptr_t>(o->exp_avg) | reinterpret_cast<uintptr_t>(o->exp_avg_sq) | reinterpret_cast<uintptr_t>(o->scale)) & 15) == 0,
               "cm_adamw_multi_step: state arenas must be 16-byte aligned");
    CM_REQUIRE(o->beta1 >= 0.0 && o->beta1 < 1.0 && o->beta2 >= 0.0 && o->beta2 < 1.0 && o->eps >= 0.0, "cm_adamw_multi_step: bad beta1 / beta2 / eps");
    const size_t need = cm_adamw_workspace_bytes(n_tensors);
    CM_REQUIRE(!(o->max_norm > 0.0) || (o->out_norm && o->ws && o->ws_bytes >= need && reinterpret_cast<uintptr_t>(o->ws) % 8 == 0),
               "cm_adamw_multi_step: clipping needs out_norm[2] and a workspace of %zu bytes", need);
    int64_t next = 0;
    for (int i = 0; i < n_tensors; ++i) {
        const cm_adamw_tensor_t& t = tensors[i];
        CM_REQUIRE(t.n >= 0, "cm_adamw_multi_step: tensor %d has n=%ld", i, (long)t.n);
        CM_REQUIRE(t.n <= (int64_t)AW_MOST * AW_CHUNK * AW_BLOCK, "cm_adamw_multi_step: %ld elements of one tensor (%d) are more than a launch takes", (long)t.n, i);
        CM_REQUIRE(aw_dtype(t.param_dtype) && aw_dtype(t.grad_dtype) && (!t.copy || aw_dtype(t.copy_dtype)), "cm_adamw_multi_step: tensor %d has an unknown dtype", i);
        CM_REQUIRE(t.n == 0 || (t.param && t.grad), "cm_adamw_multi_step: tensor %d has a NULL pointer", i);
        CM_REQUIRE(reinterpret_cast<uintptr_t>(t.param) % aw_elem(t.param_dtype) == 0 && reinterpret_cast<uintptr_t>(t.grad) % aw_elem(t.grad_dtype) == 0 &&
                   (!t.copy || reinterpret_cast<uintptr_t>(t.copy) % aw_elem(t.copy_dtype) == 0), "cm_adamw_multi_step: tensor %d is not aligned to its element", i);
        CM_REQUIRE(t.block >= next, "cm_adamw_multi_step: the states of tensor %d begin inside those of the one before it", i);
        next = t.block + cm_adamw_state_blocks(t.n);
        CM_REQUIRE(next <= o->n_blocks && next < ((int64_t)1 << 31), "cm_adamw_multi_step: the states of tensor %d end behind the arena", i);
    }
    hipStream_t s = (hipStream_t)stream;
    AwArgs a = {};
    a.m = o->exp_avg; a.v = o->exp_avg_sq; a.scale = o->scale;
    a.beta1 = (float)o->beta1; a.omb1 = (float)(1.0 - o->beta1); a.beta2 = (float)o->beta2; a.omb2 = (float)(1.0 - o->beta2); a.eps = (float)o->eps;
    a.wdf = (float)(1.0 - o->lr * o->weight_decay); a.grad_scale = (float)o->grad_scale;
    a.lr = o->lr; a.b1 = o->beta1; a.b2 = o->beta2; a.step_dev = o->step_dev;
    if (!o->step_dev) {
        a.step_size = (float)(o->lr / (1.0 - pow(o->beta1, (double)o->step)));
        a.inv_bc2 = (float)(1.0 / sqrt(1.0 - pow(o->beta2, (double)o->step)));
    }
    // two rounds over the list where the clip coefficient is needed first: all norms, then all updates.  The table travels in the launch's arguments: nothing is
    // copied to the device, nothing has to be kept alive, and a captured launch replays the addresses it was captured with.
    AwTable t;
    int parts = 0;
    for (int round = o->max_norm > 0.0 ? 0 : 1; round < 2; ++round) {
        int i = 0;
        while (i < n_tensors) {
            t.count = 0;
            int64_t chunks = 0;
            for (; i < n_tensors && t.count < AW_TABLE; ++i) {
                const cm_adamw_tensor_t& x = tensors[i];
                if (x.n == 0) continue;
                const int64_t c = (cm_adamw_state_blocks(x.n) + AW_CHUNK - 1) / AW_CHUNK;
                // the next launch's first: a tensor alone always fits (norms have a grid of their own, and room for its sums per AW_TABLE tensors)
                if (round == 1 && chunks + c > AW_MOST) break;
                t.e[t.count] = {x.param, x.grad, x.copy, x.n, (int)chunks, (int)x.block};
                t.kinds[t.count++] = (uint8_t)(x.param_dtype | x.grad_dtype << 2 | x.copy_dtype << 4);
                chunks += c;  // < 2^31: the blocks of all tensors together are
            }
            if (t.count == 0) break;
            if (round == 0) {
                const int grid = (int)(chunks < AW_NORM_GRID ? chunks : AW_NORM_GRID);
                hipLaunchKernelGGL(k_adamw_norm, dim3(grid), dim3(AW_NT), 0, s, t, (int)chunks, a.grad_scale, (double*)o->ws + parts);
                parts += grid;
            } else if (o->state_bits == 32) {
                hipLaunchKernelGGL(k_adamw<32>, dim3((unsigned)chunks), dim3(AW_NT), 0, s, t, a);
            } else {
                hipLaunchKernelGGL(k_adamw<8>, dim3((unsigned)chunks), dim3(AW_NT), 0, s, t, a);
            }
            CM_CHECK_LAUNCH("cm_adamw_multi_step");
        }
        if (round == 0 && parts > 0 && parts <= AW_FEW) {
            a.parts = (const double*)o->ws; a.nparts = parts; a.max_norm = (float)o->max_norm; a.norm = o->out_norm;
        } else if (round == 0) {
            hipLaunchKernelGGL(k_adamw_coef, dim3(1), dim3(1024), 0, s, (const double*)o->ws, parts, (float)o->max_norm, o->out_norm);
            CM_CHECK_LAUNCH("cm_adamw_multi_step/norm");
            a.coef = o->out_norm + 1;
        }
    }
    return 0;
}
