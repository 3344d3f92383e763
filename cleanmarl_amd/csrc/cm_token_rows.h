// cm_token_rows.h -- the kernels of cm_token.hip for one type of logits (instantiated by cm_token_{f32,f16,bf16}.hip).
#pragma once
#include "cm_token.h"

namespace {

__device__ __forceinline__ int64_t tok_token(const TokArgs& a, int64_t r) {
    return a.token_bytes == 8 ? reinterpret_cast<const int64_t*>(a.token)[r] : (int64_t) reinterpret_cast<const int32_t*>(a.token)[r];
}
// an input that no kernel of the launch writes, at an index that is the same for the whole wave: a scalar load.  As a vector load it would be
// the youngest in the queue, and using it would wait for every piece of a row that was asked for before it.
template <class X> __device__ __forceinline__ X tok_scalar(const X* p, int64_t i) { return ((const __attribute__((address_space(4))) X*)p)[i]; }
// preference: whether row r belongs to a sequence at all
__device__ __forceinline__ bool tok_in_range(const TokArgs& a, int64_t r) { return !a.range_lo || (r >= *a.range_lo && r < *a.range_hi); }

// the token's logit as the sums see it: -inf where it is not available; NaN behind the vocabulary -- an error that must be seen
template <class T, bool AV>
__device__ __forceinline__ float tok_logit(const typename T::elem* row, const uint8_t* av, int64_t tok, int V) {
    if (tok >= V) return NAN;
    return !AV || av[tok] ? T::get(row[tok]) : -INFINITY;
}

// the same in 64 bits, for sums over many rows; s = 0: a row that is left out
__device__ __forceinline__ double run_logp64(float x, float M, float s, const TokScale& c) { return ((double)x * c.full - (double)M) * 0.6931471805599453 - log((double)s); }
__device__ __forceinline__ double tok_logp64(float x, float m, float s, const TokScale& c) { return s == 0.0f ? 0.0 : ((double)x - (double)m) * c.full * 0.6931471805599453 - log((double)s); }

// scalars of the clipped policy loss of one row: adds its statistics to st (where `add`), returns g = dloss / dlogp and h = the entropy's factor
struct TokPolicyRow { float old, adv, ref, w; };
__device__ __forceinline__ TokPolicyRow tok_policy_load(const TokArgs& a, int64_t r) {
    return {a.logp_old[r], a.adv[r], a.logp_ref ? a.logp_ref[r] : 0.0f, a.weight ? a.weight[r] : 1.0f};
}
__device__ __forceinline__ void tok_policy_row(const TokArgs& a, const TokPolicyRow& q, float logp, float H, bool add, double (&st)[TOK_STATS], float& g, float& h) {
    const float delta = logp - q.old, rho = expf(delta), w = q.w;
    const float whole = q.adv * rho, cut = q.adv * fminf(fmaxf(rho, a.lo), a.hi);
    const bool number = whole == whole;
    const float pg = number ? fminf(whole, cut) : NAN;
    g = number ? (whole <= cut ? -whole : 0.0f) : NAN;  // torch.min's gradient: a tie inside the borders is the unclipped branch, one outside has adv = 0
    float loss = -pg - a.ent_coef * H, kl = 0.0f;
    if (a.logp_ref) {
        const float d = q.ref - logp, e = expm1f(d);
        kl = d < INFINITY ? e - d : d;  // a token that has become impossible: infinitely far, and no inf - inf
        if (a.kl_coef != 0.0f) {        // without it the divergence is only measured: 0 * inf would reach loss and gradient
            g -= a.kl_coef * e;
            loss += a.kl_coef * kl;
        }
    }
    g *= w;
    h = w * a.ent_coef;
    if (add) {
        st[CM_STAT_PG] += (double)(w * pg);
        st[CM_STAT_ENT] += (double)(w * H);
        st[CM_STAT_KL] += (double)(w * ((rho - 1.0f) - delta));
        st[CM_STAT_CLIP] += (rho < a.lo || rho > a.hi) ? (double)w : 0.0;
        st[CM_STAT_LOSS] += (double)(w * loss);
        st[CM_STAT_COUNT] += 1.0;
        st[CM_STAT_KL_REF] += (double)(w * kl);
        st[CM_STAT_WEIGHT] += (double)w;
    }
}

// The sums of a row that TokRun cannot form, by the whole workgroup (`sh` is not in use by anyone when this begins)
template <class T, bool AV, bool EN, int NT>
__device__ __forceinline__ TokSum tok_careful_sum(const typename T::elem* row, const uint8_t* av, const TokArgs& a, TokSum* sh) {
    TokSum z = {-FLT_MAX, 0.0f, 0.0f};
    for (int j = threadIdx.x * T::W; j < a.V; j += NT * T::W) {
        float f[T::W];
        tok_load<T, AV>(row, av, j, a.V, f);
        tok_add<EN>(z, f, a.c.bin, a.c.lo);
    }
    tok_block<EN, NT / 64>(z, a.c.bin, sh);
    return z;
}
// ... and its gradient, or zeros (not live)
template <class T, bool AV, bool EN, int NT>
__device__ __forceinline__ void tok_careful_grad(const typename T::elem* row, const uint8_t* av, typename T::elem* drow, const TokArgs& a, const TokGrad& g, bool live) {
    for (int j = threadIdx.x * T::W; j < a.V; j += NT * T::W) {
        float f[T::W], d[T::W] = {};
        if (live) {
            tok_load<T, AV>(row, av, j, a.V, f);
            tok_grad<EN>(f, j, g, a.c.bin, d);
        }
        tok_store<T>(drow, j, a.V, d);
    }
}

// Forward only, rows too long for a wave: a workgroup per row, several to a CU, two batches of U pieces to a thread in flight (U = 4 holds more in
// flight and fewer workgroups: 98 us against 90 for 4096 x 50001 fp16 with entropies).  TOK_POLICY: rows that no workgroup can hold; what k_tok_back needs
// of each goes to memory.
template <class T, int MODE, bool AV, bool EN, int NT, int U>
__global__ __launch_bounds__(NT) void k_tok_sum(const TokArgs a) {
    typedef typename T::elem elem;
    constexpr int W = T::W, NW = NT / 64;
    __shared__ TokRun sh[2][NW];
    __shared__ TokSum careful[NW];
    __shared__ double st[TOK_STATS];
    if (MODE == TOK_POLICY && threadIdx.x == 0) for (int i = 0; i < TOK_STATS; ++i) st[i] = 0.0;
    int turn = 0;
    const int tid = threadIdx.x;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        if (!tok_in_range(a, r)) continue;
        const int64_t tok = tok_token(a, r);
        const elem* row = reinterpret_cast<const elem*>(a.logits) + r * a.ld;
        const uint8_t* av = AV ? a.avail + r * a.avail_ld : nullptr;
        float x = 0.0f, logp = 0.0f, H = 0.0f;
        float2 keep = {0.0f, 0.0f};
        TokPolicyRow q = {};
        if (MODE == TOK_POLICY) q = tok_policy_load(a, r);
        if (tok >= 0 && (MODE != TOK_POLICY || q.w != 0.0f)) {
            x = tok_logit<T, AV>(row, av, tok, a.V);
            const TokShape shape = tok_shape<T>(row, a.V, a.peel);
            const elem* body = row + shape.head;
            const uint8_t* body_av = AV ? av + shape.head : nullptr;
            const int nfull = shape.full;
            TokRun z = {TOK_START, 0.0f, 0.0f};
            tok_u4 raw[U];
            TokAvail<W> ok[AV ? U : 1];
            auto load = [&](int i0) {  // no load depends on a condition: behind the end the row's last piece is read again
#pragma unroll
                for (int k = 0; k < U; ++k) {
                    const int i = min(i0 + k * NT + tid, nfull - 1);
                    raw[k] = reinterpret_cast<const typename T::vec*>(body)[i];
                    if (AV) ok[k] = tok_avail<W>(body_av, i * W);
                }
            };
            load(0);
            for (int i0 = 0; i0 < nfull; i0 += NT * U) {
                tok_u4 cur[U];
#pragma unroll
                for (int k = 0; k < U; ++k) { if (AV) tok_mask_raw<T>(ok[k], raw[k]); cur[k] = raw[k]; }
                load(i0 + NT * U);
#pragma unroll
                for (int k = 0; k < U; ++k) {
                    if (i0 + k * NT >= nfull) break;
                    float f[W];
                    T::unpack(cur[k], f);
                    if (i0 + k * NT + NT > nfull) {
                        const bool here = i0 + k * NT + tid < nfull;
#pragma unroll
                        for (int i = 0; i < W; ++i) f[i] = here ? f[i] : -INFINITY;
                    }
                    run_add<EN, true>(z, f, a.c.bin, a.c.lo);
                }
            }
            const int je = shape.edge(tid, W);
            if (tid < shape.edges && (!AV || av[je])) { const float one[1] = {T::get(row[je])}; run_add<EN, true>(z, one, a.c.bin, a.c.lo); }
            run_block<EN, NW>(z, sh[turn]);
            turn ^= 1;
            if (run_ordinary<EN>(z)) {
                const float logs = logf(z.s);
                logp = run_logp(x, z.M, logs, a.c);
                H = logs - z.u / z.s * TOK_LN2;
                keep = make_float2(z.M, -run_sum(z, a.c));
                if (a.logp64 && tid == 0) a.logp64[r] = run_logp64(x, z.M, z.s, a.c);
            } else {
                const TokSum y = tok_careful_sum<T, AV, EN, NT>(row, av, a, careful);
                const float logs = logf(y.s);
                if (y.s != 0.0f) { logp = tok_logp(x, y.m, logs, a.c); H = logs - y.u / y.s * TOK_LN2; }
                keep = make_float2(y.m, y.s);
                if (a.logp64 && tid == 0) a.logp64[r] = tok_logp64(x, y.m, y.s, a.c);
                __syncthreads();  // `careful` is free again
            }
        }
        if (tid == 0) {
            if (a.logp) a.logp[r] = logp;
            if (a.logp64 && tok < 0) a.logp64[r] = 0.0;
            if (EN && a.entropy) a.entropy[r] = H;
            if (a.keep) a.keep[r] = keep;
            if (MODE == TOK_POLICY && keep.y != 0.0f) {
                float g, h;
                tok_policy_row(a, q, logp, H, true, st, g, h);
                a.g_out[r] = g; a.h_out[r] = -h;
            }
        }
    }
    if (MODE == TOK_POLICY && tid == 0)
        for (int i = 0; i < TOK_STATS; ++i) { if (gridDim.x == 1) a.stats[i] = (float)st[i]; else a.part[(int64_t)blockIdx.x * TOK_STATS + i] = st[i]; }
}

// Few long rows: a row is cut into segments, a workgroup sums one, k_tok_join puts them together (figures: tok_launch4, where it is chosen).
template <class T, bool AV, bool EN, int NT>
__global__ __launch_bounds__(NT) void k_tok_part(const TokArgs a) {
    typedef typename T::elem elem;
    constexpr int W = T::W, NW = NT / 64;
    __shared__ TokRun sh[NW];
    const int tid = threadIdx.x, seg = blockIdx.x;
    const int64_t r = blockIdx.y;
    const int64_t tok = tok_in_range(a, r) ? tok_token(a, r) : -1;
    if (tok < 0) return;  // k_tok_join does not look at it either
    const elem* row = reinterpret_cast<const elem*>(a.logits) + r * a.ld;
    const uint8_t* av = AV ? a.avail + r * a.avail_ld : nullptr;
    const TokShape shape = tok_shape<T>(row, a.V, a.peel);
    const elem* body = row + shape.head;
    const int len = (shape.full + a.segs - 1) / a.segs, b = seg * len, e = min(b + len, shape.full);
    TokRun z = {TOK_START, 0.0f, 0.0f};
    for (int i = b + tid; i < e; i += NT) {
        tok_u4 raw = reinterpret_cast<const typename T::vec*>(body)[i];
        if (AV) tok_mask_raw<T>(tok_avail<W>(av + shape.head, i * W), raw);
        float f[W];
        T::unpack(raw, f);
        run_add<EN, true>(z, f, a.c.bin, a.c.lo);
    }
    const int je = shape.edge(tid, W);
    if (seg == 0 && tid < shape.edges && (!AV || av[je])) { const float one[1] = {T::get(row[je])}; run_add<EN, true>(z, one, a.c.bin, a.c.lo); }
    run_block<EN, NW>(z, sh);
    if (tid == 0) a.split[r * a.segs + seg] = make_float4(z.M, z.s, z.u, seg == 0 ? tok_logit<T, AV>(row, av, tok, a.V) : 0.0f);
}

// Half a wave per row.
template <class T, bool AV, bool EN, int NT>
__global__ __launch_bounds__(NT) void k_tok_join(const TokArgs a) {
    typedef typename T::elem elem;
    constexpr int PER = NT / 32;
    __shared__ TokSum careful[NT / 64], sums[PER];
    __shared__ int odd[PER];
    const int lane = threadIdx.x & 31, slot = threadIdx.x >> 5;
    const int64_t r0 = (int64_t)blockIdx.x * PER, r = r0 + slot;
    const bool here = r < a.rows && tok_in_range(a, r);
    const bool counts = here && tok_token(a, r) >= 0;
    TokRun z = {TOK_START, 0.0f, 0.0f};
    float x = 0.0f;
    if (counts) {
        const float4 v = lane < a.segs ? a.split[r * a.segs + lane] : make_float4(TOK_START, 0.0f, 0.0f, 0.0f);
        z = {v.x, v.y, v.z};
        x = __shfl(v.w, threadIdx.x & 32, 64);
        run_group<EN, 32>(z);
    }
    const bool ordinary = run_ordinary<EN>(z);
    if (lane == 0) odd[slot] = counts && !ordinary;
    __syncthreads();
    for (int p = 0; p < PER; ++p) {  // rows that have to be done over, by all
        if (!odd[p]) continue;
        const TokSum y = tok_careful_sum<T, AV, EN, NT>(reinterpret_cast<const elem*>(a.logits) + (r0 + p) * a.ld, AV ? a.avail + (r0 + p) * a.avail_ld : nullptr, a, careful);
        if (threadIdx.x == 0) sums[p] = y;
        __syncthreads();
    }
    if (!here || lane != 0) return;
    float logp = 0.0f, H = 0.0f;
    double logp64 = 0.0;
    float2 keep = {0.0f, 0.0f};
    if (counts) {
        const TokSum y = ordinary ? TokSum{0.0f, z.s, z.u} : sums[slot];
        const float logs = logf(y.s);
        if (y.s != 0.0f) {
            logp = ordinary ? run_logp(x, z.M, logs, a.c) : tok_logp(x, y.m, logs, a.c);
            if (EN) H = logs - y.u / y.s * TOK_LN2;
        }
        keep = ordinary ? make_float2(z.M, -run_sum(z, a.c)) : make_float2(y.m, y.s);
        logp64 = ordinary ? run_logp64(x, z.M, z.s, a.c) : tok_logp64(x, y.m, y.s, a.c);
    }
    if (a.logp) a.logp[r] = logp;
    if (a.logp64) a.logp64[r] = logp64;
    if (a.keep) a.keep[r] = keep;
    if (EN && a.entropy) a.entropy[r] = H;
}

// Backward only, rows too long for a wave: nothing is summed, so a workgroup takes NT * U pieces of one row, whichever.  The rows come in
// descending order: the last ones that a forward sweep has read are the ones still in a cache.  Stores are streaming ones, they would push the logits
// out of it (2048 x 32000 fp32, both sweeps: 160 us with ordinary ones, 129 with these).  8192 x 131072 bf16, a pass among others: 0.74 ms, 5.8 TB/s.
template <class T, bool AV, bool EN, int NT, int U>
__global__ __launch_bounds__(NT) void k_tok_back(const TokArgs a, int parts, int64_t tiles) {
    typedef typename T::elem elem;
    constexpr int W = T::W;
    const int tid = threadIdx.x;
    if (a.pair_part && blockIdx.x == 0) tok_sum_stats<NT>(a.pair_part, a.pairs, a.stats);
    for (int64_t t = tiles - 1 - blockIdx.x; t >= 0; t -= gridDim.x) {
        const int64_t r = t / parts;
        const int part = (int)(t - r * parts);
        if (!tok_in_range(a, r)) continue;
        const elem* row = reinterpret_cast<const elem*>(a.logits) + r * a.ld;
        elem* drow = reinterpret_cast<elem*>(a.dlogits) + r * a.dld;
        const uint8_t* av = AV ? a.avail + r * a.avail_ld : nullptr;
        const int64_t tok = tok_token(a, r);
        const float2 keep = a.keep_in[r];
        const bool live = tok >= 0 && keep.y != 0.0f;
        const TokShape shape = tok_shape<T>(drow, a.V, a.peel);
        const int nfull = shape.full, i0 = part * NT * U, je = shape.edge(tid, W);
        const bool edge = part == 0 && tid < shape.edges;
        typename T::vec* dbody = reinterpret_cast<typename T::vec*>(drow + shape.head);
        if (i0 >= nfull && part != 0) continue;
        if (!live) {
#pragma unroll
            for (int k = 0; k < U; ++k) if (i0 + k * NT + tid < nfull) dbody[i0 + k * NT + tid] = tok_u4{0u, 0u, 0u, 0u};
            if (edge) drow[je] = T::put(0.0f);
            continue;
        }
        TokGrad g = {};
        const bool run = keep.y < 0.0f;  // the form of TokRun (a sum that is NaN is none)
        const float s = fabsf(keep.y);
        g.m = keep.x; g.rs = 1.0f / s;
        g.a = g.b = (tok >= a.V ? NAN : a.d_logp[r]) * a.c.nat;
        if (EN) { g.K = a.entropy_in[r] - logf(s); g.h = -a.d_entropy[r] * a.c.nat; }
        g.tok = (int)(tok < a.V && (!AV || av[tok]) ? tok : -1);
        const RunGrad gr = run_grad_row<T, EN>(g.m, s, g.K, g.b, g.h);
        tok_u4 raw[U];
        TokAvail<W> ok[AV ? U : 1];
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int i = min(i0 + k * NT + tid, nfull - 1);
            raw[k] = reinterpret_cast<const typename T::vec*>(row + shape.head)[i];
            if (AV) ok[k] = tok_avail<W>(av + shape.head, i * W);
        }
        float last[1] = {-INFINITY};
        if (edge && (!AV || av[je])) last[0] = T::get(row[je]);
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int i = i0 + k * NT + tid;
            if (AV) tok_mask_raw<T>(ok[k], raw[k]);
            tok_u4 d;
            if (run) {
                d = run_grad<T, EN>(raw[k], gr, a.c.bin);
            } else {
                float f[W], v[W];
                T::unpack(raw[k], f);
                tok_grad_rest<EN>(f, g, a.c.bin, v);
                d = T::pack(v);
            }
            if (shape.piece(g.tok, W) == i && g.tok >= 0) {  // the token's own place: from its logit, rounded once
                float f[W], v[W];
                T::unpack(raw[k], f);
                T::unpack(d, v);
#pragma unroll
                for (int q = 0; q < W; ++q) {
                    const float one[1] = {f[q]};
                    float w[1];
                    if (run) w[0] = run_grad_one<EN>(f[q], gr, a.c.bin); else tok_grad_rest<EN>(one, g, a.c.bin, w);
                    if (shape.head + i * W + q == g.tok) v[q] = w[0] + g.a;
                }
                d = T::pack(v);  // the others are what they were
            }
            if (i < nfull) __builtin_nontemporal_store((typename T::vec)d, dbody + i);
        }
        if (edge) {
            float d[1];
            if (run) d[0] = run_grad_one<EN>(last[0], gr, a.c.bin); else tok_grad_rest<EN>(last, g, a.c.bin, d);
            drow[je] = T::put(je == g.tok ? d[0] + g.a : d[0]);
        }
    }
}

// Short rows: G lanes of a wave hold one row in registers (NV pieces of 16 bytes to a lane), 64 / G rows to a wave.  The row is read once.
// Bound by issue and latency rather than bytes for the smallest: 4.2 M rows of 5 fp32 actions with avail took 108 us at five waves to a SIMD and with the row
// waiting for its token, 70 us (4.6 TB/s) at eight and without.  65536 rows of 1032 bf16 columns: 101 us; a workgroup per row: 261.
template <class T, int MODE, bool AV, bool EN, int G, int NV>
__global__ __launch_bounds__(256, NV * G < 256 ? 8 : NV == 4 ? 5 : 4) void k_tok_short(const TokArgs a) {
    typedef typename T::elem elem;
    constexpr int W = T::W, PER = 256 / G;
    constexpr bool ENT = EN || MODE == TOK_POLICY;
    const int gl = threadIdx.x & (G - 1);  // lane in the group
    if (MODE == TOK_BWD && a.pair_part && blockIdx.x == 0) tok_sum_stats<256>(a.pair_part, a.pairs, a.stats);
    double st[TOK_STATS] = {};
    for (int64_t r = (int64_t)blockIdx.x * PER + threadIdx.x / G; r < a.rows; r += (int64_t)gridDim.x * PER) {
        if (!tok_in_range(a, r)) continue;
        const elem* row = reinterpret_cast<const elem*>(a.logits) + r * a.ld;
        const uint8_t* av = AV ? a.avail + r * a.avail_ld : nullptr;
        elem* drow = reinterpret_cast<elem*>(a.dlogits) + r * a.dld;
        const int64_t tok = tok_token(a, r);
        TokPolicyRow q = {};
        if (MODE == TOK_POLICY) q = tok_policy_load(a, r);
        bool live = tok >= 0 && (MODE != TOK_POLICY || q.w != 0.0f);
        float f[NV][W];
        float x = 0.0f;
        {  // of a row that is left out, too: waiting for its token first would cost more than the row
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int j = (k * G + gl) * W;
                if (j < a.V) tok_load<T, AV>(row, av, j, a.V, f[k]);
                else {
#pragma unroll
                    for (int i = 0; i < W; ++i) f[k][i] = -INFINITY;
                }
            }
            if (MODE != TOK_BWD) x = tok_logit<T, AV>(row, av, tok < 0 ? 0 : tok, a.V);
        }
        TokGrad g = {};
        if (MODE == TOK_BWD) {
            const float2 k = a.keep_in[r];
            live = live && k.y != 0.0f;
            g.m = k.x; g.rs = 1.0f / k.y;
            g.a = g.b = (tok >= a.V ? NAN : a.d_logp[r]) * a.c.nat;
            if (EN) { g.K = a.entropy_in[r] - logf(k.y); g.h = -a.d_entropy[r] * a.c.nat; }
        } else {
            float m = -FLT_MAX, s = 0.0f, u = 0.0f;
            if (live) {
#pragma unroll
                for (int k = 0; k < NV; ++k)
#pragma unroll
                    for (int i = 0; i < W; ++i) m = fmaxf(m, f[k][i]);
#pragma unroll
                for (int o = G / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
#pragma unroll
                for (int k = 0; k < NV; ++k)
#pragma unroll
                    for (int i = 0; i < W; ++i) {
                        const float d = f[k][i] - m, t = fmaf(d, a.c.lo, d * a.c.bin), e = tok_exp2(t);
                        s += e;
                        if (ENT) u = fmaf(e, fmaxf(t, TOK_FAR), u);
                    }
#pragma unroll
                for (int o = G / 2; o > 0; o >>= 1) { s += __shfl_xor(s, o, 64); if (ENT) u += __shfl_xor(u, o, 64); }
                live = s != 0.0f;
            }
            float logp = 0.0f, H = 0.0f;
            if (live) {
                const float logs = logf(s);
                g.m = m; g.rs = 1.0f / s;
                logp = tok_logp(x, m, logs, a.c);
                if (ENT) { g.K = -u * g.rs * TOK_LN2; H = logs + g.K; }
            }
            if (MODE == TOK_POLICY && live) {
                float gg, hh;
                tok_policy_row(a, q, logp, H, gl == 0, st, gg, hh);
                g.a = g.b = gg * a.c.nat; g.h = hh * a.c.nat;
            }
            if (gl == 0) {
                if (a.logp) a.logp[r] = logp;
                if (MODE == TOK_LOGP && a.logp64) a.logp64[r] = tok_logp64(x, m, live ? s : 0.0f, a.c);
                if (EN && a.entropy) a.entropy[r] = H;
                if (a.keep) a.keep[r] = make_float2(m, live ? s : 0.0f);
            }
        }
        if (MODE != TOK_LOGP) {
            g.tok = (int)(live && tok < a.V && (!AV || av[tok]) ? tok : -1);
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int j = (k * G + gl) * W;
                float d[W] = {};
                if (live) tok_grad<EN>(f[k], j, g, a.c.bin, d);
                if (j < a.V) tok_store<T>(drow, j, a.V, d);
            }
        }
    }
    if (MODE == TOK_POLICY) {  // lanes with gl != 0 hold zeros
        __shared__ double sh[4][TOK_STATS];
#pragma unroll
        for (int i = 0; i < TOK_STATS; ++i) {
            const double v = cm_wave_sum_d(st[i]);
            if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6][i] = v;
        }
        __syncthreads();
        if (threadIdx.x < TOK_STATS) {
            const double v = sh[0][threadIdx.x] + sh[1][threadIdx.x] + sh[2][threadIdx.x] + sh[3][threadIdx.x];
            if (gridDim.x == 1) a.stats[threadIdx.x] = (float)v; else a.part[(int64_t)blockIdx.x * TOK_STATS + threadIdx.x] = v;
        }
    }
}

// Long rows: a workgroup holds a row in registers, NV pieces of 16 bytes to a thread, so that the logits leave memory once
// (8192 x 131072 bf16: 0.81 ms, 5.3 TB/s, where a large copy gets 5.0; reading each row twice took 1.38 ms).  Workgroups are persistent; a piece's register is refilled with the NEXT row as soon as its gradient is stored, so loads are in flight during all of the arithmetic and no second workgroup is needed to hide them.
// That only works in straight-line code -- behind a branch the compiler waits for every load there is -- so no load depends on a condition:
// threads without a piece read the row's last one, and where the next row is left out the current one is read again (from a cache).
// The first FULL pieces of every thread exist (the choice of the kernel sees to that).
// avail: its bytes for the next row pass through a ring of R pieces in registers into LDS, where each thread finds its own again (kept in
// registers they would be half as much again as the logits: spills at 1024 threads).
template <class T, bool AV, bool EN, int NT, int NV, int FULL>
__global__ __launch_bounds__(NT) void k_tok_regs(const TokArgs a) {
    typedef typename T::elem elem;
    constexpr int W = T::W, NW = NT / 64;
    __shared__ TokRun sh[2][NW];
    __shared__ TokSum careful[NW];
    __shared__ double st[TOK_STATS];  // the first thread's: in registers they would be sixteen of every thread's
    if (threadIdx.x == 0) for (int i = 0; i < TOK_STATS; ++i) st[i] = 0.0;
    int turn = 0;
    const int tid = threadIdx.x;
    struct Row { int64_t tok; TokPolicyRow q; bool live; };
    auto scalars = [&](int64_t r) {
        Row s = {-1, {}, false};
        if (r < a.rows) {
            s.tok = a.token_bytes == 8 ? tok_scalar((const int64_t*)a.token, r) : (int64_t)tok_scalar((const int32_t*)a.token, r);
            s.q = {tok_scalar(a.logp_old, r), tok_scalar(a.adv, r), a.logp_ref ? tok_scalar(a.logp_ref, r) : 0.0f, a.weight ? tok_scalar(a.weight, r) : 1.0f};
            s.live = s.tok >= 0 && s.q.w != 0.0f;
        }
        return s;
    };
    auto row_at = [&](int64_t r) { return reinterpret_cast<const elem*>(a.logits) + r * a.ld; };
    auto drow_at = [&](int64_t r) { return reinterpret_cast<elem*>(a.dlogits) + r * a.dld; };
    auto av_at = [&](int64_t r) { return AV ? a.avail + r * a.avail_ld : nullptr; };
    // a scalar base per piece and a small vector offset: left to itself the compiler keeps an address per piece in registers
    auto base = [&](const void* p, unsigned off) {
        asm volatile("" : "+s"(off));
        return reinterpret_cast<const char*>(p) + off;
    };
    auto at = [&](const elem* row, int k) { return const_cast<typename T::vec*>(reinterpret_cast<const typename T::vec*>(base(row, k * NT * 16u) + (unsigned)tid * 16u)); };
    auto piece = [&](const elem* row, int nfull, int k) -> tok_u4 {  // row: where its body begins
        if (k < FULL) return *at(row, k);
        const int slot = min(tid, nfull - 1 - k * NT);  // below zero for a piece that no thread has: the row's last one then
        return *reinterpret_cast<const typename T::vec*>(base(row, k * NT * 16u) + slot * 16);
    };
    auto piece_av = [&](const uint8_t* av, int nfull, int k) {
        if (k < FULL) return tok_avail<W>(reinterpret_cast<const uint8_t*>(base(av, k * NT * W) + (unsigned)(tid * W)), 0);
        const int slot = min(tid, nfull - 1 - k * NT);
        return tok_avail<W>(reinterpret_cast<const uint8_t*>(base(av, k * NT * W) + slot * W), 0);
    };
    constexpr int R = NT == 1024 ? 4 : (NV < 8 ? NV : 8);
    __shared__ TokAvail<W> ok[AV ? NV : 1][AV ? NT : 1];
    tok_u4 raw[NV];
    TokAvail<W> ring[AV ? R : 1];
    elem last;
    uint8_t last_ok = 1;
    auto edges = [&](const elem* row, const uint8_t* av, const TokShape& s) {
        const int j = tid < s.edges ? s.edge(tid, W) : 0;
        last = row[j];
        if (AV) last_ok = av[j];
    };
    auto fill = [&](const elem* row, const uint8_t* av, const TokShape& s) {  // a whole row at once
        edges(row, av, s);
#pragma unroll
        for (int k = 0; k < NV; ++k) raw[k] = piece(row + s.head, s.full, k);
        if (AV) {
#pragma unroll
            for (int k = 0; k < NV + R; ++k) {
                if (k >= R) ok[k - R][tid] = ring[k % R];
                if (k < NV) ring[k % R] = piece_av(av + s.head, s.full, k);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
    int64_t r = blockIdx.x;
    Row now = scalars(r);
    TokShape shape = tok_shape<T>(drow_at(r), a.V, a.peel);
    fill(row_at(r), av_at(r), shape);
    for (; r < a.rows; r += gridDim.x) {
        const int64_t rn = r + gridDim.x;
        const Row next = scalars(rn);
        const elem *row = row_at(r), *nrow = next.live ? row_at(rn) : row;
        const uint8_t *av = av_at(r), *nav = next.live ? av_at(rn) : av;
        const TokShape nshape = tok_shape<T>(drow_at(rn), a.V, a.peel);
        const elem* nbody = nrow + nshape.head;
        const uint8_t* nbody_av = AV ? nav + nshape.head : nullptr;
        const int nfull = shape.full, je = tid < shape.edges ? shape.edge(tid, W) : 0;
        const bool edge = tid < shape.edges;
        const int64_t tok = now.tok;
        const int toki = (int)(tok < 0 ? 0 : (tok < a.V ? tok : a.V - 1));
        float x = T::get(row[toki]);
        bool tok_ok = true;
        if (AV) tok_ok = av[toki] != 0;
        x = tok < a.V ? (tok_ok ? x : -INFINITY) : NAN;
        TokRun z = {TOK_START, 0.0f, 0.0f};
        float lastf = -INFINITY;
        if (now.live) {
            lastf = edge && last_ok ? T::get(last) : -INFINITY;
            const float one[1] = {lastf};
            run_add<true, true>(z, one, a.c.bin, a.c.lo);
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                if (k >= FULL && k * NT >= nfull) break;
                if (AV) tok_mask_raw<T>(ok[k][tid], raw[k]);
                float f[W];
                T::unpack(raw[k], f);
                if (k < FULL) {
                    run_add<true, AV>(z, f, a.c.bin, a.c.lo);
                } else {
                    const bool here = tid + k * NT < nfull;
#pragma unroll
                    for (int i = 0; i < W; ++i) f[i] = here ? f[i] : -INFINITY;
                    run_add<true, true>(z, f, a.c.bin, a.c.lo);
                }
                asm volatile("" : "+v"(z.M), "+v"(z.s), "+v"(z.u));  // one piece after the other: interleaved, the floats of all of them would be live at once
                __builtin_amdgcn_sched_barrier(0);
            }
            if (AV) {
#pragma unroll
                for (int k = 0; k < R; ++k) ring[k] = piece_av(nbody_av, nshape.full, k);
            }
            run_block<true, NW>(z, sh[turn]);  // its barrier: all have read the token's logit before a gradient is written over it
            turn ^= 1;
        }
        const bool ordinary = run_ordinary<true>(z);
        TokSum y = {0.0f, 0.0f, 0.0f};
        if (now.live && !ordinary) { y = tok_careful_sum<T, AV, true, NT>(row, av, a, careful); __syncthreads(); }
        const float s = ordinary ? z.s : y.s;
        const bool live = now.live && s != 0.0f;
        TokGrad g = {};  // all zero: a row that is left out gets zeros
        RunGrad gr = {};
        float logp = 0.0f, H = 0.0f;
        if (live) {
            const float logs = logf(s);
            g.m = y.m; g.rs = 1.0f / s;
            logp = ordinary ? run_logp(x, z.M, logs, a.c) : tok_logp(x, y.m, logs, a.c);
            g.K = -(ordinary ? z.u : y.u) * g.rs * TOK_LN2; H = logs + g.K;
            float gg, hh;
            tok_policy_row(a, now.q, logp, H, tid == 0, st, gg, hh);
            g.a = g.b = gg * a.c.nat; g.h = hh * a.c.nat;
            if (ordinary) { const float sg = run_sum(z, a.c); gr = run_grad_row<T, EN>(z.M, sg, H - logf(sg), g.b, g.h); }
        }
        if (tid == 0 && a.logp) a.logp[r] = logp;
        {
            g.tok = live && tok < a.V && tok_ok ? toki : -1;
            elem *drow = drow_at(r), *dbody = drow + shape.head;
            if (now.live && ordinary) {
                if (edge) drow[je] = T::put(run_grad_one<EN>(lastf, gr, a.c.bin));
                edges(nrow, nav, nshape);
#pragma unroll
                for (int k = 0; k < NV; ++k) {
                    asm volatile("" : "+v"(raw[k]));  // unpacked again: the floats of the first sweep would be kept, at two registers for one
                    if (k < FULL || tid + k * NT < nfull) {
                        __builtin_nontemporal_store((typename T::vec)run_grad<T, EN>(raw[k], gr, a.c.bin), at(dbody, k));
                    }
                    if (AV) {
                        ok[k][tid] = ring[k % R];
                        if (k + R < NV) ring[k % R] = piece_av(nbody_av, nshape.full, k + R);
                    }
                    raw[k] = piece(nbody, nshape.full, k);
                    __builtin_amdgcn_sched_barrier(0);
                }
                // the token's place once more, by the thread that has just written it: a comparison in every piece would be a branch in every piece
                const int tp = shape.piece(g.tok, W);
                if (g.tok >= 0 && tid == (tp >= 0 ? tp & (NT - 1) : shape.edge_of(g.tok, W))) {
                    drow[g.tok] = T::put(run_grad_one<EN>(x, gr, a.c.bin) + g.a);
                }
            } else {  // zeros, or the careful form from memory; the next row replaces what the registers hold
                if (live) {
                    tok_careful_grad<T, AV, EN, NT>(row, av, drow, a, g, true);
                } else {
                    if (edge) drow[je] = T::put(0.0f);
                    for (int k = tid; k < nfull; k += NT) __builtin_nontemporal_store((typename T::vec)tok_u4{0u, 0u, 0u, 0u}, reinterpret_cast<typename T::vec*>(dbody) + k);
                }
                fill(nrow, nav, nshape);
            }
        }
        now = next; shape = nshape;
    }
    if (tid == 0)
        for (int i = 0; i < TOK_STATS; ++i) { if (gridDim.x == 1) a.stats[i] = (float)st[i]; else a.part[(int64_t)blockIdx.x * TOK_STATS + i] = st[i]; }
}

// ---------------------------------------------------------------- choice of a kernel
inline int tok_grid(int64_t items) { return (int)(items < TOK_MAX_GRID ? (items < 1 ? 1 : items) : TOK_MAX_GRID); }

template <class T, int MODE, bool AV, bool EN>
int tok_launch4(TokArgs& a, void* scratch, hipStream_t s) {
    const int64_t nvec = ((int64_t)a.V + T::W - 1) / T::W;
    // a policy loss of few rows in one workgroup, up to four rounds of short ones (2 us each): less than a second launch that adds up statistics (4 us); four
    // rounds of 4096 columns took 23 us
#define TOK_SHORT(G, NV) do { const int grid = MODE == TOK_POLICY && a.rows <= (G < 64 ? 4 : 1) * (256 / G) ? 1 : tok_grid((a.rows + 256 / G - 1) / (256 / G)); \
        hipLaunchKernelGGL((k_tok_short<T, MODE, AV, EN, G, NV>), dim3(grid), dim3(256), 0, s, a); return grid; } while (0)
    // the fewest lanes that hold the row, so that most of a wave works: up to 512 pieces (measured at 130 and 512: the wave is faster than a workgroup)
    if (nvec <= 2) TOK_SHORT(1, 2);
    if (nvec <= 8) TOK_SHORT(4, 2);
    if (nvec <= 32) TOK_SHORT(16, 2);
    if (nvec <= 128) TOK_SHORT(64, 2);
    if (nvec <= 256) TOK_SHORT(64, 4);
    if (nvec <= 512) TOK_SHORT(64, 8);
#undef TOK_SHORT
    const int64_t nfull = a.V / T::W;
    a.peel = 127u;
    auto back = [&](const TokArgs& b) {
        constexpr int NT = 256, U = 4;
        const int parts = (int)((nfull + NT * U - 1) / (NT * U));
        const int64_t tiles = b.rows * parts;
        hipLaunchKernelGGL((k_tok_back<T, AV, EN, NT, U>), dim3((unsigned)(tiles < (1 << 20) ? tiles : (1 << 20))), dim3(NT), 0, s, b, parts, tiles);
    };
    if constexpr (MODE == TOK_BWD) {
        back(a);
        return 0;
    }
    if constexpr (MODE == TOK_LOGP) {
        // Few long rows in segments of at least 512 pieces (8 KB).  GPU time among other launches, bf16: 16 rows of 131072 columns 14.2 -> 7.7 us, 64 rows 14.8 -> 11.1; but
        // 128 rows of 65536 9.3 -> 11.0, 64 rows of 16384 4.5 -> 7.5: below 8192 pieces a row is done before a second launch has begun.
        if (a.rows <= TOK_SPLIT_ROWS && nfull >= 8192) {
            const int64_t most = 1024 / a.rows < nfull / 512 ? 1024 / a.rows : nfull / 512;
            a.segs = (int)(most < TOK_SPLIT_SEGS ? most : TOK_SPLIT_SEGS);
            a.split = reinterpret_cast<float4*>(scratch);
            hipLaunchKernelGGL((k_tok_part<T, AV, EN, 256>), dim3(a.segs, (unsigned)a.rows), dim3(256), 0, s, a);
            hipLaunchKernelGGL((k_tok_join<T, AV, EN, 256>), dim3((unsigned)(a.rows + 7) / 8), dim3(256), 0, s, a);
            return 0;
        }
        const int grid = (int)(a.rows < (1 << 20) ? a.rows : (1 << 20));
        hipLaunchKernelGGL((k_tok_sum<T, MODE, AV, EN, 256, 2>), dim3(grid), dim3(256), 0, s, a);
        return grid;
    }
    if constexpr (MODE == TOK_POLICY) {
        constexpr int HEAD = (128 / (int)sizeof(typename T::elem) + T::W - 1) / T::W;  // the most pieces that a head takes from the body
        // The smallest workgroup whose registers hold the row, four pieces to a thread at a time: threads without a piece still load and mask.  FULL pieces of
        // every thread exist: nfull > NT * FULL; a head is only peeled off where they still do.
#define TOK_REGS(NT, NV, FULL, PER_CU) do { if (nfull <= NT * NV) { const int grid = (int)(a.rows < 256 * PER_CU ? a.rows : 256 * PER_CU); \
        a.peel = nfull - HEAD >= NT * FULL ? 127u : 0u; \
        hipLaunchKernelGGL((k_tok_regs<T, AV, EN, NT, NV, FULL>), dim3(grid), dim3(NT), 0, s, a); return grid; } } while (0)
        TOK_REGS(256, 4, 0, 8);
        TOK_REGS(256, 8, 4, 4);
        TOK_REGS(256, 12, 8, 4);
        TOK_REGS(256, 16, 12, 4);
        TOK_REGS(512, 12, 8, 2);
        TOK_REGS(512, 16, 12, 2);
        TOK_REGS(1024, 12, 8, 1);
        TOK_REGS(1024, 16, 12, 1);
        if constexpr (!AV) TOK_REGS(1024, 20, 16, 1);  // (with avail their LDS would not do.)  4096 x 151936 bf16: 0.50 ms, in two launches 0.62
#undef TOK_REGS
    }
    if constexpr (MODE == TOK_POLICY) {  // three sweeps of memory at 5 TB/s and more instead of two that a workgroup could overlap only by half (3.0 TB/s)
        const int grid = tok_grid(a.rows);
        a.peel = 127u;
        a.keep = reinterpret_cast<float2*>(scratch);
        a.g_out = reinterpret_cast<float*>(a.keep + a.rows); a.h_out = a.g_out + a.rows; a.entropy = a.h_out + a.rows;
        hipLaunchKernelGGL((k_tok_sum<T, MODE, AV, true, 256, 2>), dim3(grid), dim3(256), 0, s, a);
        TokArgs b = a;
        b.keep_in = a.keep; b.d_logp = a.g_out; b.d_entropy = a.h_out; b.entropy_in = a.entropy;
        back(b);
        return grid;
    }
    return 0;
}
template <class T, int MODE>
int tok_launch2(TokArgs& a, bool en, void* scratch, hipStream_t s) {
    if (a.avail) return en ? tok_launch4<T, MODE, true, true>(a, scratch, s) : tok_launch4<T, MODE, true, false>(a, scratch, s);
    return en ? tok_launch4<T, MODE, false, true>(a, scratch, s) : tok_launch4<T, MODE, false, false>(a, scratch, s);
}
template <class T>
int tok_launch_type(TokArgs& a, int mode, bool en, void* scratch, hipStream_t s) {
    if (mode == TOK_LOGP) return tok_launch2<T, TOK_LOGP>(a, en, scratch, s);
    if (mode == TOK_BWD) return tok_launch2<T, TOK_BWD>(a, en, scratch, s);
    return tok_launch2<T, TOK_POLICY>(a, en, scratch, s);
}

}  // namespace
