// Softmax statistics of a row gathered in one pass, and the best entries of a row: what log_probs.hip and bank_log_probs.hip share.
//
// Scores z = scale * logit - weight (each operation rounded, so that the order of two scores is that of elementary 32-bit
// operations); a weight of +inf leaves the place out whatever the logit is (z = -inf).  With x = (z - max z) log2 e a state is
//     m = the largest score so far,  s = sum exp2(x),  t = sum exp2(x) x,
// m finite from the start (-FLT_MAX), so that no difference of infinities arises: a row with nothing left has s = 0, any other at least 1
// (its largest entry); a NaN or +inf among the scores makes s NaN.  Then
//     lse = m + log s,   log2 p_j = x_j - log2 s,   entropy = log 2 (log2 s - t / s).
// The bank kernels without weights keep m in units of log 2 (m = k v for the product v, k = |scale| log2 e) and take x = fma(k, v, -m), one
// operation instead of three; the rounding of k is then the same in m and in every x and drops out of log p.  All of it is kept in 32 bits.
#pragma once
#include <float.h>

#include "dense.h"

namespace nemo {

constexpr int kMaxTop = 16;

struct SoftmaxState { float m, s, t; };

__device__ inline SoftmaxState empty_state() { return {-FLT_MAX, 0.0f, 0.0f}; }

constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;

__device__ inline float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }      // within one step; 0 below 2^-126

// unit: log2 e where m is a score, 1 where it is in units of log 2.
__device__ inline SoftmaxState join_states(const SoftmaxState& a, const SoftmaxState& b, float unit) {
    SoftmaxState r;
    r.m = fmaxf(a.m, b.m);
    const float da = (a.m - r.m) * unit, db = (b.m - r.m) * unit;
    const float ea = exp2_fast(da), eb = exp2_fast(db);
    r.s = a.s * ea + b.s * eb;
    r.t = ea * (a.t + fmaxf(da, -1.0e4f) * a.s) + eb * (b.t + fmaxf(db, -1.0e4f) * b.s);
    return r;
}

// Makes room for scores up to `m`: the old sums in the new units.
__device__ inline void raise(SoftmaxState& a, float m, float unit) {
    const float d = (a.m - m) * unit, f = exp2_fast(d);
    a.t = f * (a.t + fmaxf(d, -1.0e4f) * a.s);
    a.s *= f;
    a.m = m;
}

// The states of a wave's lanes as one, the same in every lane.
__device__ inline SoftmaxState wave_join(SoftmaxState a, float unit) {
    raise(a, wave_max(a.m), unit);
    a.s = wave_sum(a.s);
    a.t = wave_sum(a.t);
    return a;
}

__device__ inline float score(float logit, float scale) { return __fmul_rn(logit, scale); }
__device__ inline float score(float logit, float scale, float w) {
    return w == __builtin_inff() ? neg_inf() : __fsub_rn(__fmul_rn(logit, scale), w);
}

// An entry of a row: larger values first, lower places first among equal ones.  place < 0: nothing.
struct Entry { float z; int place; };
__device__ inline bool ahead(const Entry& a, const Entry& b) { return a.z > b.z || (a.z == b.z && a.place < b.place); }

constexpr int kNoPlace = 0x7FFFFFFF;               // sorts behind every place of the same score
__device__ inline Entry no_entry() { return {neg_inf(), kNoPlace}; }
// The first of a wave's entries, the same in every lane.
__device__ inline Entry wave_best(const Entry& a) {
    const float z = wave_max(a.z);
    return {z, wave_min(a.z == z ? a.place : kNoPlace)};
}

// What a call returns for a row, from its joined state.
struct RowOut {
    float* logp;          // any of these may be null
    float* entropy;
    float* lse;
    float* stats;         // [rows][4]: m, log2 s, entropy, 0 - what the gradient needs
    float* top_logp;      // [rows][top]
    long long* top_index;
    int top;
    float k;              // 0: m is a score; else m is in units of log 2 and entries are products, x = k v - m
};

__device__ inline float state_unit(const RowOut& o) { return o.k == 0.0f ? kLog2e : 1.0f; }
// log p of a score (product).
__device__ inline float entry_logp(const RowOut& o, const SoftmaxState& a, float v) {
    if (v == neg_inf()) return v;
    return o.k == 0.0f ? (v - a.m) - kLn2 * log2f(a.s) : kLn2 * (__builtin_fmaf(o.k, v, -a.m) - log2f(a.s));
}

// v_target is read only where 0 <= target < cols.
__device__ inline void write_row(const RowOut& o, long row, const SoftmaxState& a, long long target, long long cols, float v_target) {
    const float log2_s = log2f(a.s);                                   // -inf for a row with nothing left, NaN for a broken one
    const bool nothing = a.s == 0.0f;
    const float h = nothing ? 0.0f : kLn2 * (log2_s - a.t / a.s);
    float lp = 0.0f;
    if (target >= 0 && target < cols) lp = a.s != a.s ? a.s : entry_logp(o, a, v_target);
    else if (target != -1) lp = __builtin_nanf("");
    if (o.logp) o.logp[row] = lp;
    if (o.entropy) o.entropy[row] = h;
    if (o.lse) o.lse[row] = nothing ? neg_inf() : o.k == 0.0f ? a.m + kLn2 * log2_s : kLn2 * (a.m + log2_s);
    if (o.stats) *(f32x4*)(o.stats + 4 * row) = (f32x4){a.m, log2_s, h, 0.0f};
}

__device__ inline void write_top(const RowOut& o, long row, int i, const SoftmaxState& a, const Entry& e) {
    const bool broken = a.s != a.s, none = e.z == neg_inf();
    o.top_logp[row * o.top + i] = broken ? a.s : none ? neg_inf() : entry_logp(o, a, e.z);
    o.top_index[row * o.top + i] = broken || none ? -1 : e.place;
}

// The gradient of one score: with log2 p = x - log2 s,
//     dz = p (g_lse - g_logp - g_entropy (log p + entropy)) + [j = target] g_logp = p (c - g2 log2 p) + [j = target] g_logp,
// c = g_lse - g_logp - g_entropy entropy and g2 = g_entropy log 2.  Places that are left out get none.
constexpr float kNoProbability = 1.0e30f;              // exp2(x - this) is 0, and 0 times it as well
struct RowCoef { float m, log2_s, c, g2, g_logp; int target; };
__device__ inline RowCoef row_coef(const float* stats, const float* g_logp, const float* g_entropy, const float* g_lse, const long long* targets,
                                   long row, long long cols) {
    const f32x4 st = *(const f32x4*)(stats + 4 * row);
    const long long t = targets[row];
    const float ge = g_entropy ? g_entropy[row] : 0.0f;
    RowCoef k;
    k.m = st[0];
    k.log2_s = st[1] == neg_inf() ? kNoProbability : st[1];            // a row with nothing left: p = 0 everywhere
    k.g2 = ge * kLn2;
    k.g_logp = g_logp && t >= 0 && t < cols ? g_logp[row] : 0.0f;
    k.c = (g_lse ? g_lse[row] : 0.0f) - k.g_logp - ge * st[2];
    if (t < -1 || t >= cols) k.c = __builtin_nanf("");                 // a target outside the row: the gradient is as undefined as logp
    k.target = t >= 0 && t < cols ? (int)t : -1;
    return k;
}
// dz without the target's share, of a place whose log2 p is lp2; -inf (p = 0) is clamped, so that 0 is not multiplied by an infinity.
__device__ inline float prob_gradient(float lp2, float c, float g2) { return exp2_fast(lp2) * (c - g2 * fmaxf(lp2, -200.0f)); }

}  // namespace nemo
