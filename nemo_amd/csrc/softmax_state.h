// Softmax statistics of a row gathered in one pass, and the best entries of a row: what log_probs.hip and bank_log_probs.hip share.
//
// Scores z = scale * logit - weight (each operation rounded, so that the order of two scores is that of elementary 32-bit
// operations); a weight of +inf leaves the place out whatever the logit is (z = -inf).  A state is
//     m = max(-FLT_MAX, z...)      s = sum exp(z - m)      t = sum exp(z - m) (z - m)
// with m finite from the start, so that no difference of infinities arises: a row with nothing left has s = 0, any other at least 1
// (its largest entry); a NaN or +inf among the scores makes s NaN.  Then
//     lse = m + log s,   log p_j = (z_j - m) - log s,   entropy = log s - t / s.
// All of it is kept in 32 bits.
#pragma once
#include <float.h>

#include "dense.h"

namespace nemo {

constexpr int kMaxTop = 16;

struct SoftmaxState { float m, s, t; };

__device__ inline SoftmaxState empty_state() { return {-FLT_MAX, 0.0f, 0.0f}; }

__device__ inline float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }

// exp(d) d: 0 where exp(d) is 0, also where d has overflowed to -inf.
__device__ inline float weighted(float e, float d) { return e * fmaxf(d, -200.0f); }

__device__ inline SoftmaxState join_states(const SoftmaxState& a, const SoftmaxState& b) {
    SoftmaxState r;
    r.m = fmaxf(a.m, b.m);
    const float da = a.m - r.m, db = b.m - r.m;
    const float ea = expf(da), eb = expf(db);
    r.s = a.s * ea + b.s * eb;
    r.t = ea * (a.t + fmaxf(da, -200.0f) * a.s) + eb * (b.t + fmaxf(db, -200.0f) * b.s);
    return r;
}

__device__ inline SoftmaxState wave_join(SoftmaxState a) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const SoftmaxState b = {__shfl_xor(a.m, o), __shfl_xor(a.s, o), __shfl_xor(a.t, o)};
        a = join_states(a, b);
    }
    return a;
}

__device__ inline float score(float logit, float scale) { return __fmul_rn(logit, scale); }
__device__ inline float score(float logit, float scale, float w) {
    return w == __builtin_inff() ? neg_inf() : __fsub_rn(__fmul_rn(logit, scale), w);
}

// An entry of a row: larger values first, lower places first among equal ones.  place < 0: nothing.
struct Entry { float z; int place; };
__device__ inline bool ahead(const Entry& a, const Entry& b) { return a.z > b.z || (a.z == b.z && a.place < b.place); }

__device__ inline Entry wave_best(Entry a) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const Entry b = {__shfl_xor(a.z, o), __shfl_xor(a.place, o)};
        if (ahead(b, a)) a = b;
    }
    return a;
}

constexpr int kNoPlace = 0x7FFFFFFF;               // sorts behind every place of the same score
__device__ inline Entry no_entry() { return {neg_inf(), kNoPlace}; }

// What a call returns for a row, from its joined state.  z_target is read only where 0 <= target < cols.
struct RowOut {
    float* logp;          // any of these may be null
    float* entropy;
    float* lse;
    float* stats;         // [rows][4]: m, log s, entropy, 0 - what the gradient needs
    float* top_logp;      // [rows][top]
    long long* top_index;
    int top;
};

__device__ inline float row_logp(const SoftmaxState& a, float z) { return z == neg_inf() ? z : (z - a.m) - logf(a.s); }

__device__ inline void write_row(const RowOut& o, long row, const SoftmaxState& a, long long target, long long cols, float z_target) {
    const float log_s = logf(a.s);                                     // -inf for a row with nothing left, NaN for a broken one
    const bool nothing = a.s == 0.0f;
    const float h = nothing ? 0.0f : log_s - a.t / a.s;
    float lp = 0.0f;
    if (target >= 0 && target < cols) lp = a.s != a.s ? a.s : row_logp(a, z_target);
    else if (target != -1) lp = __builtin_nanf("");
    if (o.logp) o.logp[row] = lp;
    if (o.entropy) o.entropy[row] = h;
    if (o.lse) o.lse[row] = nothing ? neg_inf() : a.m + log_s;
    if (o.stats) *(f32x4*)(o.stats + 4 * row) = (f32x4){a.m, log_s, h, 0.0f};
}

__device__ inline void write_top(const RowOut& o, long row, int i, const SoftmaxState& a, const Entry& e) {
    const bool broken = a.s != a.s, none = e.z == neg_inf();
    o.top_logp[row * o.top + i] = broken ? a.s : none ? neg_inf() : (e.z - a.m) - logf(a.s);
    o.top_index[row * o.top + i] = broken || none ? -1 : e.place;
}

// The gradient of one score: log p = (z - m) - log s, p = exp(log p),
//     dz = p (g_lse - g_logp - g_entropy (log p + entropy)) + [j = target] g_logp = p (c - g_entropy log p) + [j = target] g_logp.
// Places that are left out get none.
struct RowCoef { float m, log_s, c, g_entropy, g_logp; int target; };
__device__ inline RowCoef row_coef(const float* stats, const float* g_logp, const float* g_entropy, const float* g_lse, const long long* targets,
                                   long row, long long cols) {
    const f32x4 st = *(const f32x4*)(stats + 4 * row);
    const long long t = targets[row];
    RowCoef k;
    k.m = st[0];
    k.log_s = st[1];
    k.g_entropy = g_entropy ? g_entropy[row] : 0.0f;
    k.g_logp = g_logp && t >= 0 && t < cols ? g_logp[row] : 0.0f;
    k.c = (g_lse ? g_lse[row] : 0.0f) - k.g_logp - k.g_entropy * st[2];
    if (t < -1 || t >= cols) k.c = __builtin_nanf("");                 // a target outside the row: the gradient is as undefined as logp
    k.target = t >= 0 && t < cols ? (int)t : -1;
    return k;
}
__device__ inline float score_gradient(const RowCoef& k, float z, int j) {
    if (z == neg_inf()) return 0.0f;
    const float lp = (z - k.m) - k.log_s, p = expf(lp);
    const float d = p == 0.0f ? 0.0f : p * (k.c - k.g_entropy * lp);
    return j == k.target ? d + k.g_logp : d;
}

}  // namespace nemo
