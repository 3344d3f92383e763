// cm_token.hip -- losses of policies whose action is a token: log-probability and entropy of rows of logits, the clipped policy loss with
// a KL term, the preference loss on paired log ratios; forward and backward.
//
// The counterpart, for logits that come out of the caller's own model, of what cm_ppo_actor_fwd_bwd does behind its fused MLP
// (cleanmarl/mappo_multienvs.py:172-183, 536-570: Categorical over masked logits, ratio, clipped surrogate, entropy bonus).  With
// x = logits / T and unavailable columns at -inf, a row needs  m = max x,  s = sum e^(x - m),  log p_j = x_j - m - log s,
// H = log s - sum p_j (x_j - m)  and every gradient below is  dx_j = (g ([j = token] - p_j) + h p_j (log p_j + H)) / T  with two
// scalars g and h per row.  All sums, statistics and scalars are fp32 or wider; the gradient is rounded once, to the logits' type.
#include "cm_token.h"

namespace {

enum { TOK_LOGP = 0, TOK_BWD = 1, TOK_POLICY = 2 };
constexpr int TOK_STATS = CM_NUM_STATS, TOK_MAX_GRID = 2048;

struct TokArgs {
    const void* logits; int64_t ld; const uint8_t* avail; int64_t avail_ld; const void* token; int token_bytes;
    int64_t rows; int V; TokScale c;
    float *logp, *entropy; float2* keep;                                     // forward
    const float2* keep_in; const float *entropy_in, *d_logp, *d_entropy;     // backward
    void* dlogits; int64_t dld;
    const float *logp_old, *adv, *logp_ref, *weight; float lo, hi, kl_coef, ent_coef; double* part;  // policy
    const int32_t* seq_start; int n_seq; const float* coef;                  // preference: rows of sequence q are [seq_start[q], seq_start[q + 1])
};

__device__ __forceinline__ int64_t tok_token(const TokArgs& a, int64_t r) {
    return a.token_bytes == 8 ? reinterpret_cast<const int64_t*>(a.token)[r] : (int64_t) reinterpret_cast<const int32_t*>(a.token)[r];
}
// the sequence that row r belongs to; -1: in front of the first or behind the last
__device__ __forceinline__ int tok_sequence(const TokArgs& a, int64_t r) {
    if (r < a.seq_start[0] || r >= a.seq_start[a.n_seq]) return -1;
    int lo = 0, hi = a.n_seq;
    while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (a.seq_start[mid] <= r) lo = mid; else hi = mid; }
    return lo;
}
// (x_token - m) / T - log s; a token behind the vocabulary is an error that must be seen: NaN
template <class T, bool AV>
__device__ __forceinline__ float tok_taken(const typename T::elem* row, const uint8_t* av, int64_t tok, int V, const TokSum& q, float logs, const TokScale& c) {
    if (tok >= V) return NAN;
    const bool ok = !AV || av[tok];
    return (ok ? T::get(row[tok]) - q.m : -INFINITY) * c.nat - logs;
}

// scalars of the clipped policy loss of one row: adds its statistics to st, returns g = dloss / dlogp and h = the entropy's factor
__device__ __forceinline__ void tok_policy_row(const TokArgs& a, int64_t r, float w, float logp, float H, double (&st)[TOK_STATS], float& g, float& h) {
    const float delta = logp - a.logp_old[r], rho = expf(delta), adv = a.adv[r];
    const float whole = adv * rho, cut = adv * fminf(fmaxf(rho, a.lo), a.hi);
    const float pg = fminf(whole, cut);
    g = whole <= cut ? -whole : 0.0f;  // torch.min's gradient: a tie inside the borders is the unclipped branch, one outside has adv = 0
    if (!(whole == whole) || !(cut == cut)) g = NAN;
    float loss = -pg - a.ent_coef * H, kl = 0.0f;
    if (a.logp_ref) {
        const float d = a.logp_ref[r] - logp, e = expm1f(d);
        kl = e - d;
        g -= a.kl_coef * e;
        loss += a.kl_coef * kl;
    }
    g *= w;
    h = w * a.ent_coef;
    st[CM_STAT_PG] += (double)(w * ((whole == whole && cut == cut) ? pg : NAN));
    st[CM_STAT_ENT] += (double)(w * H);
    st[CM_STAT_KL] += (double)(w * ((rho - 1.0f) - delta));
    st[CM_STAT_CLIP] += (rho < a.lo || rho > a.hi) ? (double)w : 0.0;
    st[CM_STAT_LOSS] += (double)(w * loss);
    st[CM_STAT_COUNT] += 1.0;
    st[CM_STAT_KL_REF] += (double)(w * kl);
    st[CM_STAT_WEIGHT] += (double)w;
}

// One workgroup walks whole rows: a first sweep for (m, s, u), a second one that reads the row again (it is still in a cache) and writes
// the gradient.
template <class T, int MODE, bool AV, bool EN, int NT>
__global__ __launch_bounds__(NT) void k_tok_stream(const TokArgs a) {
    typedef typename T::elem elem;
    constexpr int W = T::W, NW = NT / 64;
    __shared__ TokSum sh[2][NW];
    double st[TOK_STATS] = {};
    int turn = 0;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const elem* row = reinterpret_cast<const elem*>(a.logits) + r * a.ld;
        const uint8_t* av = AV ? a.avail + r * a.avail_ld : nullptr;
        int seq = 0;
        if (a.seq_start && (seq = tok_sequence(a, r)) < 0) continue;
        const int64_t tok = tok_token(a, r);
        float w = 1.0f;
        if (MODE == TOK_POLICY && a.weight) w = a.weight[r];
        bool live = tok >= 0 && w != 0.0f;
        TokGrad g = {};
        if (MODE == TOK_BWD) {
            const float2 k = a.keep_in[r];
            live = live && k.y != 0.0f;
            const float dl = a.coef ? a.coef[seq] : a.d_logp[r];
            g.m = k.x; g.rs = 1.0f / k.y; g.logs = logf(k.y); g.a = g.b = dl * a.c.nat;
            if (tok >= a.V) g.a = g.b = NAN;
            if (EN) { g.H = a.entropy_in[r]; g.h = -a.d_entropy[r] * a.c.nat; }
        } else {
            TokSum q = {-FLT_MAX, 0.0f, 0.0f};
            if (live) {
                for (int j = threadIdx.x * W; j < a.V; j += NT * W) {
                    float f[W];
                    tok_load<T, AV>(row, av, j, a.V, f);
                    tok_add<EN>(q, f, a.c);
                }
                tok_block<EN, NW>(q, a.c, sh[turn]);
                turn ^= 1;
                live = q.s != 0.0f;
            }
            float logp = 0.0f, H = 0.0f;
            if (live) {
                g.m = q.m; g.rs = 1.0f / q.s; g.logs = logf(q.s);
                logp = tok_taken<T, AV>(row, av, tok, a.V, q, g.logs, a.c);
                if (EN) H = g.H = g.logs - q.u * g.rs;
            }
            if (MODE == TOK_POLICY) {
                if (live) {
                    double s1[TOK_STATS] = {};
                    float gg, hh;
                    tok_policy_row(a, r, w, logp, H, s1, gg, hh);
                    g.a = g.b = gg * a.c.nat; g.h = hh * a.c.nat;
                    if (threadIdx.x == 0) for (int i = 0; i < TOK_STATS; ++i) st[i] += s1[i];
                }
            }
            if (threadIdx.x == 0) {
                if (a.logp) a.logp[r] = logp;
                if (EN && a.entropy) a.entropy[r] = H;
                if (a.keep) a.keep[r] = make_float2(q.m, live ? q.s : 0.0f);
            }
        }
        if (MODE == TOK_POLICY) __syncthreads();  // in place: the token's logit has been read by all before its gradient is written
        if (MODE != TOK_LOGP) {
            g.tok = (int)(live && tok < a.V && (!AV || av[tok]) ? tok : -1);  // an unavailable place has no gradient
            elem* drow = reinterpret_cast<elem*>(a.dlogits) + r * a.dld;
            for (int j = threadIdx.x * W; j < a.V; j += NT * W) {
                float f[W], d[W];
                if (live) {
                    tok_load<T, AV>(row, av, j, a.V, f);
                    tok_grad<T, EN>(f, j, g, a.c, d);
                } else {
#pragma unroll
                    for (int i = 0; i < W; ++i) d[i] = 0.0f;
                }
                tok_store<T>(drow, j, a.V, d);
            }
        }
    }
    if (MODE == TOK_POLICY && threadIdx.x == 0)
        for (int i = 0; i < TOK_STATS; ++i) a.part[(int64_t)blockIdx.x * TOK_STATS + i] = st[i];
}

// sums of n partial rows of statistics, in a fixed order
__global__ __launch_bounds__(256) void k_tok_stats(const double* __restrict__ part, int n, float* __restrict__ stats) {
    __shared__ double sh[256 / TOK_STATS][TOK_STATS];
    const int c = threadIdx.x % TOK_STATS, g = threadIdx.x / TOK_STATS;
    double s = 0.0;
    for (int i = g; i < n; i += 256 / TOK_STATS) s += part[(int64_t)i * TOK_STATS + c];
    sh[g][c] = s;
    __syncthreads();
    if (g == 0) {
        double t = 0.0;
        for (int i = 0; i < 256 / TOK_STATS; ++i) t += sh[i][c];
        stats[c] = (float)t;
    }
}

// One workgroup per pair: log-probabilities of its two sequences (64-bit sums: thousands of terms, and only their difference counts),
// the margin, the loss and the factor that every row of the two sequences gets.
struct PrefArgs {
    const float* logp; const int32_t* seq_start; int pairs; int64_t rows; const float* ref;
    double beta, smooth, scale; int kind;
    float *coef, *margin, *seq_logp; double* part;
};
__global__ __launch_bounds__(256) void k_pref_pair(const PrefArgs a) {
    __shared__ double sh[2][4];
    const int i = blockIdx.x;
    double L[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int q = i + k * a.pairs;
        const int64_t b = max((int64_t)a.seq_start[q], (int64_t)0), e = min((int64_t)a.seq_start[q + 1], a.rows);
        double s = 0.0;
        for (int64_t r = b + threadIdx.x; r < e; r += 256) s += (double)a.logp[r];
        s = cm_wave_sum_d(s);
        if ((threadIdx.x & 63) == 0) sh[k][threadIdx.x >> 6] = s;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; ++k) L[k] = sh[k][0] + sh[k][1] + sh[k][2] + sh[k][3];
    if (threadIdx.x != 0) return;
    const double margin = (L[0] - (double)a.ref[i]) - (L[1] - (double)a.ref[i + a.pairs]);
    double loss, d;
    if (a.kind == CM_PREFERENCE_SIGMOID) {
        const double z = a.beta * margin, en = exp(-fabs(z)), tail = log1p(en);  // log(1 + e^-|z|): neither exponential overflows
        const double down = z >= 0.0 ? en / (1.0 + en) : 1.0 / (1.0 + en);       // sigmoid(-z)
        loss = (1.0 - a.smooth) * (fmax(-z, 0.0) + tail) + a.smooth * (fmax(z, 0.0) + tail);
        if (z != z) loss = z;
        d = a.beta * (a.smooth * (1.0 - down) - (1.0 - a.smooth) * down);
    } else {
        const double off = margin - 0.5 / a.beta;
        loss = off * off;
        d = 2.0 * off;
    }
    a.coef[i] = (float)(a.scale * d);
    a.coef[i + a.pairs] = (float)(-a.scale * d);
    if (a.margin) a.margin[i] = (float)margin;
    if (a.seq_logp) { a.seq_logp[i] = (float)L[0]; a.seq_logp[i + a.pairs] = (float)L[1]; }
    double* p = a.part + (int64_t)i * TOK_STATS;
    p[CM_PREF_LOSS] = loss; p[CM_PREF_CORRECT] = margin > 0.0 ? 1.0 : 0.0; p[CM_PREF_MARGIN] = margin;
    p[CM_PREF_CHOSEN] = L[0]; p[CM_PREF_REJECTED] = L[1]; p[CM_PREF_COUNT] = 1.0; p[6] = p[7] = 0.0;
}

// ---------------------------------------------------------------- host side
template <class T, int MODE, bool AV, bool EN>
int tok_launch4(const TokArgs& a, int grid, hipStream_t s) {
    hipLaunchKernelGGL((k_tok_stream<T, MODE, AV, EN, 256>), dim3(grid), dim3(256), 0, s, a);
    return 0;
}
template <class T, int MODE>
int tok_launch2(const TokArgs& a, bool en, int grid, hipStream_t s) {
    if (a.avail) return en ? tok_launch4<T, MODE, true, true>(a, grid, s) : tok_launch4<T, MODE, true, false>(a, grid, s);
    return en ? tok_launch4<T, MODE, false, true>(a, grid, s) : tok_launch4<T, MODE, false, false>(a, grid, s);
}
template <int MODE>
int tok_launch(const TokArgs& a, int dtype, bool en, int grid, hipStream_t s, const char* who) {
    if (a.rows == 0) return 0;
    if (dtype == CM_DTYPE_F32) tok_launch2<TokF32, MODE>(a, en, grid, s);
    else if (dtype == CM_DTYPE_F16) tok_launch2<TokF16, MODE>(a, en, grid, s);
    else tok_launch2<TokBF16, MODE>(a, en, grid, s);
    CM_CHECK_LAUNCH(who);
    return 0;
}
int tok_grid(int64_t rows) { return (int)(rows < TOK_MAX_GRID ? (rows < 1 ? 1 : rows) : TOK_MAX_GRID); }

inline size_t tok_elem(int dtype) { return dtype == CM_DTYPE_F32 ? 4 : 2; }
inline size_t tok_up(size_t n) { return (n + 255) & ~(size_t)255; }

int tok_check(const char* who, const cm_token_rows_t* t) {
    CM_REQUIRE(t, "%s: NULL cm_token_rows_t", who);
    CM_REQUIRE(t->dtype == CM_DTYPE_F32 || t->dtype == CM_DTYPE_F16 || t->dtype == CM_DTYPE_BF16, "%s: unknown dtype %d", who, (int)t->dtype);
    CM_REQUIRE(t->rows >= 0 && t->vocab >= 1 && t->vocab <= (1 << 30), "%s: bad rows=%ld vocab=%d", who, (long)t->rows, (int)t->vocab);
    CM_REQUIRE(t->rows < ((int64_t)1 << 40), "%s: rows=%ld out of range", who, (long)t->rows);
    CM_REQUIRE(t->rows == 0 || (t->logits && t->token), "%s: NULL logits / token", who);
    CM_REQUIRE(t->rows <= 1 || t->ld >= t->vocab, "%s: row stride %ld of the logits is below the vocabulary %d", who, (long)t->ld, (int)t->vocab);
    CM_REQUIRE(!t->avail || t->rows <= 1 || t->avail_ld >= t->vocab, "%s: row stride %ld of avail is below the vocabulary %d", who, (long)t->avail_ld, (int)t->vocab);
    CM_REQUIRE(t->token_bytes == 4 || t->token_bytes == 8, "%s: token_bytes=%d (4 or 8)", who, (int)t->token_bytes);
    CM_REQUIRE(reinterpret_cast<uintptr_t>(t->logits) % tok_elem(t->dtype) == 0 && reinterpret_cast<uintptr_t>(t->token) % t->token_bytes == 0,
               "%s: logits / token not aligned to their element", who);
    CM_REQUIRE(t->temperature > 0.0 && t->temperature < 1e30 && 1.0 / t->temperature < 1e30, "%s: temperature must be positive and finite", who);
    return 0;
}
// the gradient's rows: either exactly the logits' (in place) or apart from them
int tok_check_grad(const char* who, const cm_token_rows_t* t, const void* dlogits, int64_t dld) {
    CM_REQUIRE(t->rows == 0 || dlogits, "%s: NULL dlogits", who);
    CM_REQUIRE(t->rows <= 1 || dld >= t->vocab, "%s: row stride %ld of dlogits is below the vocabulary %d", who, (long)dld, (int)t->vocab);
    const size_t e = tok_elem(t->dtype);
    CM_REQUIRE(reinterpret_cast<uintptr_t>(dlogits) % e == 0, "%s: dlogits not aligned to its element", who);
    if (t->rows == 0) return 0;
    const char *x = (const char*)t->logits, *d = (const char*)dlogits;
    const size_t nx = ((size_t)(t->rows - 1) * t->ld + t->vocab) * e, nd = ((size_t)(t->rows - 1) * dld + t->vocab) * e;
    const bool same = x == d && (t->rows == 1 || t->ld == dld);
    CM_REQUIRE(same || x + nx <= d || d + nd <= x, "%s: dlogits overlaps the logits without being the same rows", who);
    return 0;
}
TokArgs tok_args(const cm_token_rows_t* t) {
    TokArgs a = {};
    a.logits = t->logits; a.ld = t->ld; a.avail = t->avail; a.avail_ld = t->avail_ld; a.token = t->token; a.token_bytes = t->token_bytes;
    a.rows = t->rows; a.V = t->vocab;
    a.c.nat = (float)(1.0 / t->temperature); a.c.bin = (float)(1.4426950408889634074 / t->temperature);
    return a;
}

}  // namespace

extern "C" size_t cm_token_workspace_bytes(int64_t rows, int vocab) {
    if (rows < 0 || vocab < 1) return 0;
    return tok_up((size_t)TOK_MAX_GRID * TOK_STATS * sizeof(double));
}

extern "C" int cm_token_logprob(const cm_token_rows_t* t, float* logp, float* entropy, float* keep, void* ws, size_t ws_bytes, cm_stream_t stream) {
    if (int rc = tok_check("cm_token_logprob", t)) return rc;
    CM_REQUIRE(t->rows == 0 || logp, "cm_token_logprob: NULL logp");
    CM_REQUIRE(reinterpret_cast<uintptr_t>(keep) % 8 == 0, "cm_token_logprob: keep must be 8-byte aligned");
    const size_t need = cm_token_workspace_bytes(t->rows, t->vocab);
    CM_REQUIRE(ws && ws_bytes >= need, "cm_token_logprob: workspace too small (%zu < %zu)", ws_bytes, need);
    TokArgs a = tok_args(t);
    a.logp = logp; a.entropy = entropy; a.keep = (float2*)keep;
    return tok_launch<TOK_LOGP>(a, t->dtype, entropy != nullptr, tok_grid(t->rows), (hipStream_t)stream, "cm_token_logprob");
}

extern "C" int cm_token_logprob_bwd(const cm_token_rows_t* t, const float* keep, const float* entropy, const float* d_logp, const float* d_entropy,
                                    void* dlogits, int64_t dlogits_ld, cm_stream_t stream) {
    if (int rc = tok_check("cm_token_logprob_bwd", t)) return rc;
    if (int rc = tok_check_grad("cm_token_logprob_bwd", t, dlogits, dlogits_ld)) return rc;
    CM_REQUIRE(t->rows == 0 || (keep && d_logp), "cm_token_logprob_bwd: NULL keep / d_logp");
    CM_REQUIRE(!d_entropy || entropy, "cm_token_logprob_bwd: d_entropy needs the entropy of the forward call");
    CM_REQUIRE(reinterpret_cast<uintptr_t>(keep) % 8 == 0, "cm_token_logprob_bwd: keep must be 8-byte aligned");
    TokArgs a = tok_args(t);
    a.keep_in = (const float2*)keep; a.entropy_in = entropy; a.d_logp = d_logp; a.d_entropy = d_entropy; a.dlogits = dlogits; a.dld = dlogits_ld;
    return tok_launch<TOK_BWD>(a, t->dtype, d_entropy != nullptr, tok_grid(t->rows), (hipStream_t)stream, "cm_token_logprob_bwd");
}

extern "C" int cm_token_policy_fwd_bwd(const cm_token_rows_t* t, const float* logp_old, const float* adv, const float* logp_ref, const float* weight,
                                       double clip_low, double clip_high, double kl_coef, double entropy_coef, void* dlogits, int64_t dlogits_ld,
                                       float* logp, float* stats, void* ws, size_t ws_bytes, cm_stream_t stream) {
    if (int rc = tok_check("cm_token_policy_fwd_bwd", t)) return rc;
    if (int rc = tok_check_grad("cm_token_policy_fwd_bwd", t, dlogits, dlogits_ld)) return rc;
    CM_REQUIRE(t->rows == 0 || (logp_old && adv), "cm_token_policy_fwd_bwd: NULL logp_old / adv");
    CM_REQUIRE(stats, "cm_token_policy_fwd_bwd: NULL stats");
    CM_REQUIRE(clip_low >= 0.0 && clip_low <= 1.0 && clip_high >= 0.0, "cm_token_policy_fwd_bwd: clip_low must lie in [0, 1], clip_high must not be negative");
    CM_REQUIRE(kl_coef == 0.0 || logp_ref, "cm_token_policy_fwd_bwd: kl_coef without logp_ref");
    const size_t need = cm_token_workspace_bytes(t->rows, t->vocab);
    CM_REQUIRE(ws && ws_bytes >= need && reinterpret_cast<uintptr_t>(ws) % 16 == 0, "cm_token_policy_fwd_bwd: workspace too small (%zu < %zu) or not 16-byte aligned", ws_bytes, need);
    TokArgs a = tok_args(t);
    a.logp_old = logp_old; a.adv = adv; a.logp_ref = logp_ref; a.weight = weight;
    a.lo = (float)(1.0 - clip_low); a.hi = (float)(1.0 + clip_high); a.kl_coef = (float)kl_coef; a.ent_coef = (float)entropy_coef;
    a.dlogits = dlogits; a.dld = dlogits_ld; a.logp = logp; a.part = (double*)ws;
    const int grid = tok_grid(t->rows);
    if (int rc = tok_launch<TOK_POLICY>(a, t->dtype, true, grid, (hipStream_t)stream, "cm_token_policy_fwd_bwd")) return rc;
    hipLaunchKernelGGL(k_tok_stats, dim3(1), dim3(256), 0, (hipStream_t)stream, a.part, t->rows ? grid : 0, stats);
    CM_CHECK_LAUNCH("cm_token_policy_fwd_bwd/stats");
    return 0;
}

extern "C" size_t cm_preference_workspace_bytes(int64_t rows, int vocab, int pairs) {
    if (rows < 0 || vocab < 1 || pairs < 1) return 0;
    return tok_up((size_t)rows * sizeof(float2)) + tok_up((size_t)rows * sizeof(float)) + tok_up((size_t)pairs * 2 * sizeof(float)) +
           tok_up((size_t)pairs * TOK_STATS * sizeof(double));
}

extern "C" int cm_preference_fwd_bwd(const cm_token_rows_t* t, const int32_t* seq_start, int pairs, const float* logp_ref, double beta,
                                     double label_smoothing, int kind, double scale, void* dlogits, int64_t dlogits_ld, float* margin,
                                     float* seq_logp, float* stats, void* ws, size_t ws_bytes, cm_stream_t stream) {
    if (int rc = tok_check("cm_preference_fwd_bwd", t)) return rc;
    if (int rc = tok_check_grad("cm_preference_fwd_bwd", t, dlogits, dlogits_ld)) return rc;
    CM_REQUIRE(pairs >= 1 && pairs <= (1 << 24), "cm_preference_fwd_bwd: pairs=%d", pairs);
    CM_REQUIRE(t->rows < ((int64_t)1 << 31), "cm_preference_fwd_bwd: rows=%ld does not fit the int32 sequence starts", (long)t->rows);
    CM_REQUIRE(seq_start && logp_ref && stats, "cm_preference_fwd_bwd: NULL seq_start / logp_ref / stats");
    CM_REQUIRE(kind == CM_PREFERENCE_SIGMOID || kind == CM_PREFERENCE_SQUARED, "cm_preference_fwd_bwd: unknown kind %d", kind);
    CM_REQUIRE(beta > 0.0, "cm_preference_fwd_bwd: beta must be positive");
    CM_REQUIRE(label_smoothing >= 0.0 && label_smoothing < 0.5, "cm_preference_fwd_bwd: label_smoothing must lie in [0, 0.5)");
    CM_REQUIRE(kind == CM_PREFERENCE_SIGMOID || label_smoothing == 0.0, "cm_preference_fwd_bwd: the squared loss takes no label_smoothing");
    const size_t need = cm_preference_workspace_bytes(t->rows, t->vocab, pairs);
    CM_REQUIRE(ws && ws_bytes >= need && reinterpret_cast<uintptr_t>(ws) % 16 == 0, "cm_preference_fwd_bwd: workspace too small (%zu < %zu) or not 16-byte aligned", ws_bytes, need);
    char* w = (char*)ws;
    float2* keep = (float2*)w; w += tok_up((size_t)t->rows * sizeof(float2));
    float* logp = (float*)w; w += tok_up((size_t)t->rows * sizeof(float));
    float* coef = (float*)w; w += tok_up((size_t)pairs * 2 * sizeof(float));
    double* part = (double*)w;
    hipStream_t s = (hipStream_t)stream;
    TokArgs a = tok_args(t);
    a.seq_start = seq_start; a.n_seq = 2 * pairs; a.logp = logp; a.keep = keep;
    if (int rc = tok_launch<TOK_LOGP>(a, t->dtype, false, tok_grid(t->rows), s, "cm_preference_fwd_bwd/logp")) return rc;
    PrefArgs p = {logp, seq_start, pairs, t->rows, logp_ref, beta, label_smoothing, scale, kind, coef, margin, seq_logp, part};
    hipLaunchKernelGGL(k_pref_pair, dim3(pairs), dim3(256), 0, s, p);
    CM_CHECK_LAUNCH("cm_preference_fwd_bwd/pair");
    a.keep_in = keep; a.coef = coef; a.dlogits = dlogits; a.dld = dlogits_ld;
    if (int rc = tok_launch<TOK_BWD>(a, t->dtype, false, tok_grid(t->rows), s, "cm_preference_fwd_bwd/bwd")) return rc;
    hipLaunchKernelGGL(k_tok_stats, dim3(1), dim3(256), 0, s, part, pairs, stats);
    CM_CHECK_LAUNCH("cm_preference_fwd_bwd/stats");
    return 0;
}
