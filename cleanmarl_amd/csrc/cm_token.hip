// cm_token.hip -- losses of policies whose action is a token: log-probability and entropy of rows of logits, the clipped policy loss with
// a KL term, the preference loss on paired log ratios; forward and backward.
//
// The counterpart, for logits that come out of the caller's own model, of what cm_ppo_actor_fwd_bwd does behind its fused MLP
// (cleanmarl/mappo_multienvs.py:172-183, 536-570: Categorical over masked logits, ratio, clipped surrogate, entropy bonus).  With
// x = logits / T and unavailable columns at -inf, a row needs  m = max x,  s = sum e^(x - m),  log p_j = x_j - m - log s,
// H = log s - sum p_j (x_j - m)  and every gradient below is  dx_j = (g ([j = token] - p_j) + h p_j (log p_j + H)) / T  with two
// scalars g and h per row.  All sums, statistics and scalars are fp32 or wider; the gradient is rounded once, to the logits' type.
#include "cm_token.h"
#include <initializer_list>

namespace {

__global__ __launch_bounds__(1024) void k_tok_stats(const double* __restrict__ part, int n, float* __restrict__ stats) { tok_sum_stats<1024>(part, n, stats); }

// One workgroup per pair: log-probabilities of its two sequences (64-bit sums: thousands of terms, and only their difference counts),
// the margin, the loss and the factor that every row of the two sequences gets.
struct PrefArgs {
    const double* logp; const int32_t* seq_start; int pairs; int64_t rows; const float* ref;
    double beta, smooth, scale; int kind;
    float *coef, *margin, *seq_logp; double* part;  // coef: one factor per row
};
__global__ __launch_bounds__(256) void k_pref_pair(const PrefArgs a) {
    __shared__ double sh[2][4];
    const int i = blockIdx.x;
    int64_t b[2], e[2];
    double L[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int q = i + k * a.pairs;
        b[k] = max((int64_t)a.seq_start[q], (int64_t)0); e[k] = min((int64_t)a.seq_start[q + 1], a.rows);
        double s = 0.0;
        for (int64_t r = b[k] + threadIdx.x; r < e[k]; r += 256) s += a.logp[r];
        s = cm_wave_sum_d(s);
        if ((threadIdx.x & 63) == 0) sh[k][threadIdx.x >> 6] = s;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; ++k) L[k] = sh[k][0] + sh[k][1] + sh[k][2] + sh[k][3];
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
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const float c = (float)(k ? -a.scale * d : a.scale * d);
        for (int64_t r = b[k] + threadIdx.x; r < e[k]; r += 256) a.coef[r] = c;
    }
    if (threadIdx.x != 0) return;
    if (a.margin) a.margin[i] = (float)margin;
    if (a.seq_logp) { a.seq_logp[i] = (float)L[0]; a.seq_logp[i + a.pairs] = (float)L[1]; }
    double* p = a.part + (int64_t)i * TOK_STATS;
    p[CM_PREF_LOSS] = loss; p[CM_PREF_CORRECT] = margin > 0.0 ? 1.0 : 0.0; p[CM_PREF_MARGIN] = margin;
    p[CM_PREF_CHOSEN] = L[0]; p[CM_PREF_REJECTED] = L[1]; p[CM_PREF_COUNT] = 1.0; p[6] = p[7] = 0.0;
}

// ---------------------------------------------------------------- host side
int tok_launch(const TokArgs& a, int dtype, int mode, bool en, void* scratch, hipStream_t s) {  // the number of partial rows of statistics
    if (a.rows == 0) return 0;
    return dtype == CM_DTYPE_F32 ? tok_launch_f32(a, mode, en, scratch, s) : dtype == CM_DTYPE_F16 ? tok_launch_f16(a, mode, en, scratch, s) : tok_launch_bf16(a, mode, en, scratch, s);
}

inline size_t tok_elem(int dtype) { return dtype == CM_DTYPE_F32 ? 4 : 2; }
constexpr size_t tok_up(size_t n) { return (n + 255) & ~(size_t)255; }
constexpr size_t TOK_PART_BYTES = (size_t)TOK_MAX_GRID * TOK_STATS * sizeof(double);

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
// What a call writes lies over nothing it reads and over nothing else it writes: rows are read ahead of those that are written, per-row inputs through the scalar
// cache, which does not see this launch's stores.  (dlogits and logits: tok_check_grad.)  NULL: not there.
struct TokSpan { const char* name; const void* p; size_t n; };
int tok_check_apart(const char* who, std::initializer_list<TokSpan> out, std::initializer_list<TokSpan> in) {
    auto over = [](const TokSpan& a, const TokSpan& b) {
        const char *x = (const char*)a.p, *y = (const char*)b.p;
        return x && y && a.n && b.n && x < y + b.n && y < x + a.n;
    };
    for (const TokSpan* a = out.begin(); a != out.end(); ++a) {
        for (const TokSpan* b = out.begin(); b != a; ++b) CM_REQUIRE(!over(*a, *b), "%s: %s overlaps %s", who, a->name, b->name);
        for (const TokSpan& b : in) CM_REQUIRE(!over(*a, b), "%s: %s overlaps %s", who, a->name, b.name);
    }
    return 0;
}
size_t tok_bytes(int64_t rows, int64_t ld, int vocab, size_t elem) { return rows > 0 ? ((size_t)(rows - 1) * ld + vocab) * elem : 0; }
TokSpan tok_span_logits(const cm_token_rows_t* t) { return {"logits", t->logits, tok_bytes(t->rows, t->ld, t->vocab, tok_elem(t->dtype))}; }
TokSpan tok_span_avail(const cm_token_rows_t* t) { return {"avail", t->avail, tok_bytes(t->rows, t->avail_ld, t->vocab, 1)}; }
TokSpan tok_span_token(const cm_token_rows_t* t) { return {"token", t->token, (size_t)t->rows * t->token_bytes}; }
TokSpan tok_span_grad(const cm_token_rows_t* t, const void* d, int64_t ld) { return {"dlogits", d, tok_bytes(t->rows, ld, t->vocab, tok_elem(t->dtype))}; }
TokArgs tok_args(const cm_token_rows_t* t) {
    TokArgs a = {};
    a.logits = t->logits; a.ld = t->ld; a.avail = t->avail; a.avail_ld = t->avail_ld; a.token = t->token; a.token_bytes = t->token_bytes;
    a.rows = t->rows; a.V = t->vocab;
    a.c.full = 1.4426950408889634074 / t->temperature;
    a.c.nat = (float)(1.0 / t->temperature); a.c.bin = (float)a.c.full;
    if ((double)a.c.bin > a.c.full) a.c.bin = nextafterf(a.c.bin, 0.0f);
    a.c.lo = fmaxf((float)(a.c.full - (double)a.c.bin), FLT_MIN);
    return a;
}

}  // namespace

extern "C" size_t cm_token_workspace_bytes(int64_t rows, int vocab) {
    if (rows < 0 || vocab < 1) return 0;
    static_assert(TOK_PART_BYTES >= TOK_SPLIT_BYTES, "log-probabilities use the room of the statistics");
    return TOK_PART_BYTES + (vocab > TOK_HELD / 4 ? tok_up((size_t)rows * TOK_ROW_BYTES) : 0);
}

extern "C" int cm_token_logprob(const cm_token_rows_t* t, float* logp, float* entropy, float* keep, void* ws, size_t ws_bytes, cm_stream_t stream) {
    if (int rc = tok_check("cm_token_logprob", t)) return rc;
    CM_REQUIRE(t->rows == 0 || logp, "cm_token_logprob: NULL logp");
    CM_REQUIRE(reinterpret_cast<uintptr_t>(keep) % 8 == 0, "cm_token_logprob: keep must be 8-byte aligned");
    const size_t need = cm_token_workspace_bytes(t->rows, t->vocab);
    CM_REQUIRE(ws && ws_bytes >= need && reinterpret_cast<uintptr_t>(ws) % 16 == 0, "cm_token_logprob: workspace too small (%zu < %zu) or not 16-byte aligned", ws_bytes, need);
    const size_t row = (size_t)t->rows * sizeof(float);
    if (int rc = tok_check_apart("cm_token_logprob", {{"logp", logp, row}, {"entropy", entropy, row}, {"keep", keep, 2 * row}, {"the workspace", ws, need}},
                                 {tok_span_logits(t), tok_span_avail(t), tok_span_token(t)})) return rc;
    TokArgs a = tok_args(t);
    a.logp = logp; a.entropy = entropy; a.keep = (float2*)keep;
    tok_launch(a, t->dtype, TOK_LOGP, entropy != nullptr, ws, (hipStream_t)stream);
    CM_CHECK_LAUNCH("cm_token_logprob");
    return 0;
}

extern "C" int cm_token_logprob_bwd(const cm_token_rows_t* t, const float* keep, const float* entropy, const float* d_logp, const float* d_entropy,
                                    void* dlogits, int64_t dlogits_ld, cm_stream_t stream) {
    if (int rc = tok_check("cm_token_logprob_bwd", t)) return rc;
    if (int rc = tok_check_grad("cm_token_logprob_bwd", t, dlogits, dlogits_ld)) return rc;
    CM_REQUIRE(t->rows == 0 || (keep && d_logp), "cm_token_logprob_bwd: NULL keep / d_logp");
    CM_REQUIRE(!d_entropy || entropy, "cm_token_logprob_bwd: d_entropy needs the entropy of the forward call");
    CM_REQUIRE(reinterpret_cast<uintptr_t>(keep) % 8 == 0, "cm_token_logprob_bwd: keep must be 8-byte aligned");
    const size_t row = (size_t)t->rows * sizeof(float);
    if (int rc = tok_check_apart("cm_token_logprob_bwd", {tok_span_grad(t, dlogits, dlogits_ld)},
                                 {tok_span_avail(t), tok_span_token(t), {"keep", keep, 2 * row}, {"entropy", entropy, row}, {"d_logp", d_logp, row}, {"d_entropy", d_entropy, row}})) return rc;
    TokArgs a = tok_args(t);
    a.keep_in = (const float2*)keep; a.entropy_in = entropy; a.d_logp = d_logp; a.d_entropy = d_entropy; a.dlogits = dlogits; a.dld = dlogits_ld;
    tok_launch(a, t->dtype, TOK_BWD, d_entropy != nullptr, nullptr, (hipStream_t)stream);
    CM_CHECK_LAUNCH("cm_token_logprob_bwd");
    return 0;
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
    const size_t row = (size_t)t->rows * sizeof(float);
    const TokSpan sums[] = {{"logp", logp, row}, {"stats", stats, CM_NUM_STATS * sizeof(float)}, {"the workspace", ws, need}};
    if (int rc = tok_check_apart("cm_token_policy_fwd_bwd", {tok_span_grad(t, dlogits, dlogits_ld), sums[0], sums[1], sums[2]},
                                 {tok_span_avail(t), tok_span_token(t), {"logp_old", logp_old, row}, {"adv", adv, row}, {"logp_ref", logp_ref, row}, {"weight", weight, row}})) return rc;
    if (int rc = tok_check_apart("cm_token_policy_fwd_bwd", {sums[0], sums[1], sums[2]}, {tok_span_logits(t)})) return rc;
    TokArgs a = tok_args(t);
    a.logp_old = logp_old; a.adv = adv; a.logp_ref = logp_ref; a.weight = weight;
    a.lo = (float)(1.0 - clip_low); a.hi = (float)(1.0 + clip_high); a.kl_coef = (float)kl_coef; a.ent_coef = (float)entropy_coef;
    a.dlogits = dlogits; a.dld = dlogits_ld; a.logp = logp; a.part = (double*)ws; a.stats = stats;
    const int parts = tok_launch(a, t->dtype, TOK_POLICY, entropy_coef != 0.0, t->vocab > TOK_HELD / 4 ? (char*)ws + TOK_PART_BYTES : nullptr, (hipStream_t)stream);
    CM_CHECK_LAUNCH("cm_token_policy_fwd_bwd");
    if (parts != 1) {  // one workgroup has written the sums itself
        hipLaunchKernelGGL(k_tok_stats, dim3(1), dim3(1024), 0, (hipStream_t)stream, a.part, parts, stats);
        CM_CHECK_LAUNCH("cm_token_policy_fwd_bwd/stats");
    }
    return 0;
}

extern "C" size_t cm_preference_workspace_bytes(int64_t rows, int vocab, int pairs) {
    if (rows < 0 || vocab < 1 || pairs < 1) return 0;
    return tok_up((size_t)rows * sizeof(float2)) + tok_up((size_t)rows * sizeof(double)) + tok_up((size_t)rows * sizeof(float)) +
           tok_up((size_t)pairs * TOK_STATS * sizeof(double)) +
           tok_up(TOK_SPLIT_BYTES);
}

extern "C" int cm_preference_fwd_bwd(const cm_token_rows_t* t, const int32_t* seq_start, int pairs, const float* logp_ref, double beta,
                                     double label_smoothing, int kind, double scale, void* dlogits, int64_t dlogits_ld, float* margin,
                                     float* seq_logp, float* stats, void* ws, size_t ws_bytes, cm_stream_t stream) {
    if (int rc = tok_check("cm_preference_fwd_bwd", t)) return rc;
    if (int rc = tok_check_grad("cm_preference_fwd_bwd", t, dlogits, dlogits_ld)) return rc;
    CM_REQUIRE(pairs >= 1 && pairs < (1 << 24), "cm_preference_fwd_bwd: pairs=%d (a launch has fewer than 2^24 workgroups of 256 threads)", pairs);
    CM_REQUIRE(t->rows < ((int64_t)1 << 31), "cm_preference_fwd_bwd: rows=%ld does not fit the int32 sequence starts", (long)t->rows);
    CM_REQUIRE(seq_start && logp_ref && stats, "cm_preference_fwd_bwd: NULL seq_start / logp_ref / stats");
    CM_REQUIRE(kind == CM_PREFERENCE_SIGMOID || kind == CM_PREFERENCE_SQUARED, "cm_preference_fwd_bwd: unknown kind %d", kind);
    CM_REQUIRE(beta > 0.0, "cm_preference_fwd_bwd: beta must be positive");
    CM_REQUIRE(label_smoothing >= 0.0 && label_smoothing < 0.5, "cm_preference_fwd_bwd: label_smoothing must lie in [0, 0.5)");
    CM_REQUIRE(kind == CM_PREFERENCE_SIGMOID || label_smoothing == 0.0, "cm_preference_fwd_bwd: the squared loss takes no label_smoothing");
    const size_t need = cm_preference_workspace_bytes(t->rows, t->vocab, pairs);
    CM_REQUIRE(ws && ws_bytes >= need && reinterpret_cast<uintptr_t>(ws) % 16 == 0, "cm_preference_fwd_bwd: workspace too small (%zu < %zu) or not 16-byte aligned", ws_bytes, need);
    const size_t per_pair = (size_t)pairs * sizeof(float);
    const TokSpan sums[] = {{"margin", margin, per_pair}, {"seq_logp", seq_logp, 2 * per_pair}, {"stats", stats, CM_NUM_STATS * sizeof(float)}, {"the workspace", ws, need}};
    if (int rc = tok_check_apart("cm_preference_fwd_bwd", {tok_span_grad(t, dlogits, dlogits_ld), sums[0], sums[1], sums[2], sums[3]},
                                 {tok_span_avail(t), tok_span_token(t), {"seq_start", seq_start, (2 * (size_t)pairs + 1) * sizeof(int32_t)}, {"logp_ref", logp_ref, 2 * per_pair}})) return rc;
    if (int rc = tok_check_apart("cm_preference_fwd_bwd", {sums[0], sums[1], sums[2], sums[3]}, {tok_span_logits(t)})) return rc;
    char* w = (char*)ws;
    float2* keep = (float2*)w; w += tok_up((size_t)t->rows * sizeof(float2));
    double* logp = (double*)w; w += tok_up((size_t)t->rows * sizeof(double));
    float* coef = (float*)w; w += tok_up((size_t)t->rows * sizeof(float));
    double* part = (double*)w; w += tok_up((size_t)pairs * TOK_STATS * sizeof(double));
    hipStream_t s = (hipStream_t)stream;
    TokArgs a = tok_args(t);
    a.range_lo = seq_start; a.range_hi = seq_start + 2 * pairs; a.logp64 = logp; a.keep = keep;
    tok_launch(a, t->dtype, TOK_LOGP, false, w, s);
    CM_CHECK_LAUNCH("cm_preference_fwd_bwd/logp");
    PrefArgs p = {logp, seq_start, pairs, t->rows, logp_ref, beta, label_smoothing, scale, kind, coef, margin, seq_logp, part};
    hipLaunchKernelGGL(k_pref_pair, dim3(pairs), dim3(256), 0, s, p);
    CM_CHECK_LAUNCH("cm_preference_fwd_bwd/pair");
    a.keep_in = keep; a.d_logp = coef; a.dlogits = dlogits; a.dld = dlogits_ld;
    a.pair_part = part; a.pairs = pairs; a.stats = stats;
    tok_launch(a, t->dtype, TOK_BWD, false, nullptr, s);
    CM_CHECK_LAUNCH("cm_preference_fwd_bwd/bwd");
    if (t->rows == 0) {
        hipLaunchKernelGGL(k_tok_stats, dim3(1), dim3(1024), 0, s, part, pairs, stats);
        CM_CHECK_LAUNCH("cm_preference_fwd_bwd/stats");
    }
    return 0;
}
