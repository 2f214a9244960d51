// The log probabilities of log_probs.hip straight from features and bank, z = scale <feature, bank row> - weight, without ever writing the
// [rows, bank rows] matrix, and the gradients of features and bank.
//
// All three kernels multiply 32 "owner" rows, whose fragments a wave keeps in registers, with tiles of "other" rows that the workgroup's
// four waves share in LDS (two buffers, copied from global memory without registers), on v_mfma_f32_32x32x{16 bf16, 2 f32} with the
// other rows as first operand.  Register 4 b + i of lane l then holds the product of owner row l % 32 with other row 8 b + 4 (l / 32) + i:
// a lane sees one owner row only.
//   forward   owners = features, others = bank: the softmax state of a row and its best entries live in the lane, no exchange until the end
//   features' gradient   the scores again, then dz (dense.h) in the registers of the first product is, as it stands, the second operand of
//             a second product  dx^T[c][row] += sum_j bank[j][c] dz[j][row]  (k runs in the order of the registers, and the first operand is
//             read from LDS in that order)
//   bank's gradient      the same with the roles changed: owners = bank rows, others = features; what dz needs of a feature row is staged
//             beside the tile
// In 16 bits dz is split into two pieces, dz = hi + lo, each of them multiplied: a single bf16 piece would put an error of 2^-9 of the largest
// term into sums whose terms largely cancel (the target's against all others').
//
// Work is split over the other axis where there are too few owners to fill the device; states, lists and gradients of the parts are joined
// in their order by a second kernel.  Results of two calls are the same bits.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/nemo_hip.h"
#include "errors.h"
#include "softmax_state.h"

namespace nemo {

__device__ const u32x4 g_zero_row = {0, 0, 0, 0};

template <typename T> struct Wide;                                     // 32 x 32 products; a fragment is 16 bytes a lane
template <> struct Wide<float> {
    static constexpr int KF = 8;                                       // k of a fragment: group g holds 4 g .. 4 g + 3
    static __device__ inline void run(f32x16_t& acc, const u32x4& p, const u32x4& q) { Mma<float>::run(acc, p, q); }
};
template <> struct Wide<bf16> {
    static constexpr int KF = 16;                                      // group g holds 8 g .. 8 g + 7
    static __device__ inline void run(f32x16_t& acc, const u32x4& p, const u32x4& q) {
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, p), __builtin_bit_cast(bf16x8, q), acc, 0, 0, 0);
    }
};

struct BankArgs {
    const void* own;               // rows whose fragments stay in registers
    const void* other;
    long ld_own, ld_other;         // elements
    int n_own, n_other, channels;
    const float* weights;          // [features][ldw] or one row (ldw = 0) or null
    long ldw;
    const long long* targets;
    float scale;
    int parts, part_tiles;         // tiles of other rows a part
    // forward
    float* part_state;             // [3][2 parts][rows]
    float* part_z;                 // [2 parts][rows][top]
    int* part_place;
    float* z_target;               // [rows]
    RowOut out;
    // backward
    const float* coef;             // [6][features]: m, log s, c, g_entropy, g_logp, target (bits)
    float* partial;                // [parts][n_own][CP] when parts > 1
    void* grad;                    // [n_own][channels]
};

// Chunk c of row r of a tile with CPR chunks a row lies at c ^ spread(r): the rows that one LDS read touches differ in it.
template <int CPR> __device__ inline int spread(int r) { return CPR >= 16 ? r & 15 : CPR >= 8 ? r & 7 : (r >> 1) & (CPR - 1); }

template <typename T, int CP, int ROWS>
__device__ inline void stage_rows(char* lds, const T* base, long ld, int row0, int rows, int channels, int wave, int lane) {
    constexpr int EPC = 16 / (int)sizeof(T), CPR = CP / EPC, TOTAL = ROWS * CPR;
    static_assert(TOTAL % 256 == 0, "every wave copies the same number of kilobytes");
#pragma unroll
    for (int i = 0; i < TOTAL / 256; ++i) {
        const int j = i * 4 + wave, idx = j * 64 + lane;
        const int r = idx / CPR, c = (idx & (CPR - 1)) ^ spread<CPR>(r);
        const bool in = row0 + r < rows && c * EPC < channels;
        const T* src = base + (size_t)(row0 + r) * ld + c * EPC;
        copy_to_lds(in ? (const void*)src : (const void*)&g_zero_row, lds + j * 1024);
    }
}

template <typename T, int CP>
__device__ inline u32x4 row_fragment(const char* lds, int row, int kf, int lane) {
    constexpr int CPR = CP * (int)sizeof(T) / 16;
    const int r = row + (lane & 31), c = kf * 2 + (lane >> 5);
    return *(const u32x4*)(lds + r * (CP * (int)sizeof(T)) + ((c ^ spread<CPR>(r)) << 4));
}

// Fragment of owner rows straight from memory.
template <typename T, int CP>
__device__ inline void own_fragments(u32x4 (&q)[CP / Wide<T>::KF], const BankArgs& a, int own0, int lane) {
    constexpr int EPC = 16 / (int)sizeof(T);
    const int row = own0 + (lane & 31);
#pragma unroll
    for (int kf = 0; kf < CP / Wide<T>::KF; ++kf) {
        const int c = (kf * 2 + (lane >> 5)) * EPC;
        q[kf] = row < a.n_own && c < a.channels ? *(const u32x4*)((const T*)a.own + (size_t)row * a.ld_own + c) : u32x4{0, 0, 0, 0};
    }
}

template <typename T, int CP>
__device__ inline f32x16_t products(const char* lds, int row, const u32x4 (&q)[CP / Wide<T>::KF], int lane) {
    f32x16_t acc = {};
#pragma unroll
    for (int kf = 0; kf < CP / Wide<T>::KF; ++kf) Wide<T>::run(acc, row_fragment<T, CP>(lds, row, kf, lane), q[kf]);
    return acc;
}

// Scores of the lane's 16 other rows j0 + 8 b + 4 g + i; rows at or beyond `end` are -inf.  w: the weights of the lane's feature row (already
// offset to column 0) or null.
__device__ inline void scores(float z[16], const f32x16_t& acc, float scale, const float* w, int j0, int g, int end) {
    if (w) {
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int j = j0 + 8 * b + 4 * g + i;
                z[4 * b + i] = j < end ? score(acc[4 * b + i], scale, w[j]) : neg_inf();
            }
    } else if (j0 + 32 <= end) {
#pragma unroll
        for (int i = 0; i < 16; ++i) z[i] = score(acc[i], scale);
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) z[i] = j0 + 8 * (i >> 2) + 4 * g + (i & 3) < end ? score(acc[i], scale) : neg_inf();
    }
}

template <int TOP>
__device__ inline void insert(float (&tv)[TOP], int (&tp)[TOP], float z, int place) {
    // places arrive in rising order, so an equal score goes behind those already there
#pragma unroll
    for (int i = TOP - 1; i >= 0; --i) {
        const bool above = z > tv[i];
        const bool shift = i > 0 && z > tv[i > 0 ? i - 1 : 0];
        if (above) {
            tv[i] = shift ? tv[i > 0 ? i - 1 : 0] : z;
            tp[i] = shift ? tp[i > 0 ? i - 1 : 0] : place;
        }
    }
}

template <typename T, int CP, int TOP>
__global__ __launch_bounds__(256) void bank_forward_kernel(BankArgs a) {
    constexpr int BJ = CP * sizeof(T) >= 1024 ? 32 : 64;
    __shared__ __attribute__((aligned(16))) char lds0[BJ * CP * sizeof(T)];
    __shared__ __attribute__((aligned(16))) char lds1[BJ * CP * sizeof(T)];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 5;
    const int part = (int)(blockIdx.x % a.parts);
    const int own0 = (int)(blockIdx.x / a.parts) * 128 + wave * 32, row = own0 + (lane & 31);
    const bool live = row < a.n_own;
    u32x4 q[CP / Wide<T>::KF];
    own_fragments<T, CP>(q, a, own0, lane);
    const float* w = a.weights ? a.weights + (live ? row : 0) * a.ldw : nullptr;
    const long long tl = live ? a.targets[row] : -1;
    const int target = tl >= 0 && tl < a.n_other ? (int)tl : -1;
    SoftmaxState st = empty_state();
    float tv[TOP > 0 ? TOP : 1];
    int tp[TOP > 0 ? TOP : 1];
#pragma unroll
    for (int i = 0; i < TOP; ++i) { tv[i] = neg_inf(); tp[i] = kNoPlace; }

    auto consume = [&](const char* lds, int j_tile) {
#pragma unroll
        for (int s = 0; s < BJ / 32; ++s) {
            const int j0 = j_tile + s * 32;
            const f32x16_t acc = products<T, CP>(lds, s * 32, q, lane);
            float z[16];
            scores(z, acc, a.scale, w, j0, g, a.n_other);
            float m = st.m;
#pragma unroll
            for (int i = 0; i < 16; ++i) m = fmaxf(m, z[i]);
            const float d = st.m - m, f = fast_exp(d);
            st.t = f * (st.t + fmaxf(d, -200.0f) * st.s);
            st.s *= f;
            st.m = m;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float dz = z[i] - m, e = fast_exp(dz);
                st.s += e;
                st.t += weighted(e, dz);
            }
            const int at = target - j0 - 4 * g;                        // 8 b + i if the lane holds the target's score
            if (target >= j0 && target < j0 + 32 && (at & 4) == 0 && at >= 0) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (at == 8 * (i >> 2) + (i & 3)) a.z_target[row] = z[i];
            }
            if (TOP > 0) {
                float peak = z[0];
#pragma unroll
                for (int i = 1; i < 16; ++i) peak = fmaxf(peak, z[i]);
                if (peak > tv[TOP > 0 ? TOP - 1 : 0]) {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (z[i] > tv[TOP > 0 ? TOP - 1 : 0]) insert(tv, tp, z[i], j0 + 8 * (i >> 2) + 4 * g + (i & 3));
                }
            }
        }
    };
    const int tiles = (a.n_other + BJ - 1) / BJ;
    const int t0 = part * a.part_tiles, t1 = min(tiles, t0 + a.part_tiles);
    const T* other = (const T*)a.other;
    if (t0 < t1) stage_rows<T, CP, BJ>(lds0, other, a.ld_other, t0 * BJ, a.n_other, a.channels, wave, lane);
    for (int t = t0; t < t1; t += 2) {
        __syncthreads();
        if (t + 1 < t1) stage_rows<T, CP, BJ>(lds1, other, a.ld_other, (t + 1) * BJ, a.n_other, a.channels, wave, lane);
        consume(lds0, t * BJ);
        if (t + 1 >= t1) break;
        __syncthreads();
        if (t + 2 < t1) stage_rows<T, CP, BJ>(lds0, other, a.ld_other, (t + 2) * BJ, a.n_other, a.channels, wave, lane);
        consume(lds1, (t + 1) * BJ);
    }
    if (!live) return;
    const size_t rows = a.n_own, at = (size_t)(part * 2 + g) * rows + row, plane = (size_t)2 * a.parts * rows;
    a.part_state[at] = st.m;
    a.part_state[plane + at] = st.s;
    a.part_state[2 * plane + at] = st.t;
#pragma unroll
    for (int i = 0; i < TOP; ++i)
        if (i < a.out.top) {
            a.part_z[at * a.out.top + i] = tv[i];
            a.part_place[at * a.out.top + i] = tp[i];
        }
}

// Joins the 2 x parts (at most 64) states and lists of a row: a wave a row, a lane a state.
__global__ __launch_bounds__(256) void bank_join_kernel(BankArgs a) {
    const int lane = threadIdx.x & 63, n = 2 * a.parts, top = a.out.top;
    const int row = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= a.n_own) return;
    const size_t at = (size_t)lane * a.n_own + row, plane = (size_t)n * a.n_own;
    SoftmaxState st = empty_state();
    if (lane < n) st = {a.part_state[at], a.part_state[plane + at], a.part_state[2 * plane + at]};
    st = wave_join(st);
    if (lane == 0) {
        const long long t = a.targets[row];
        write_row(a.out, row, st, t, a.n_other, t >= 0 && t < a.n_other ? a.z_target[row] : 0.0f);
    }
    int walk = 0;
    for (int i = 0; i < top; ++i) {
        Entry mine = no_entry();
        if (lane < n && walk < top) mine = {a.part_z[at * top + walk], a.part_place[at * top + walk]};
        const Entry e = wave_best(mine);
        if (mine.place == e.place && mine.z == e.z) ++walk;
        if (lane == 0) write_top(a.out, row, i, st, e);
    }
}

// What the gradient kernels need of every feature row, in six arrays.
__global__ __launch_bounds__(256) void bank_coef_kernel(const float* stats, const float* g_logp, const float* g_entropy, const float* g_lse,
                                                        const long long* targets, int rows, int cols, float* coef) {
    const int row = blockIdx.x * 256 + threadIdx.x;
    if (row >= rows) return;
    const RowCoef k = row_coef(stats, g_logp, g_entropy, g_lse, targets, row, cols);
    const size_t n = rows;
    coef[row] = k.m;
    coef[n + row] = k.log_s;
    coef[2 * n + row] = k.c;
    coef[3 * n + row] = k.g_entropy;
    coef[4 * n + row] = k.g_logp;
    coef[5 * n + row] = __builtin_bit_cast(float, k.target);
}

__device__ inline float gradient_of(float z, float m, float log_s, float c, float ge, float gl, int target, int j) {
    const float lp = (z - m) - log_s, p = fast_exp(lp);
    const float d = p == 0.0f ? 0.0f : p * (c - ge * lp);
    return z == neg_inf() ? 0.0f : j == target ? d + gl : d;
}

// A value of the second product's first operand; `clean` turns infinities and NaN into 0 (see bank_gradient_kernel).
__device__ inline float clean_value(float v) { return __builtin_fabsf(v) <= FLT_MAX ? v : 0.0f; }

// First operand of the second product: columns cb .. cb + 31 of the tile's rows, in the order in which the first product's registers hold
// them.  f32: step b takes registers 4 b .. 4 b + 3, rows 8 b + 4 g + i.  bf16: step b takes registers 8 b .. 8 b + 7, rows
// 16 b + 8 (e / 4) + 4 g + e % 4, two transposing reads of four rows each.
template <typename T, int CP>
__device__ inline u32x4 column_fragment(const char* lds, int row0, int b, int cb, int lane, bool clean) {
    constexpr int RB = CP * (int)sizeof(T), CPR = RB / 16;
    const int g = lane >> 5;
    if constexpr (sizeof(T) == 4) {
        u32x4 v;
        const int c = cb + (lane & 31);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = row0 + 8 * b + 4 * g + i;
            float f = *(const float*)(lds + r * RB + (((c >> 2) ^ spread<CPR>(r)) << 4) + (c & 3) * 4);
            if (clean) f = clean_value(f);
            v[i] = __builtin_bit_cast(uint32_t, f);
        }
        return v;
    } else {
        const int i = lane & 15, c = cb + 16 * ((lane >> 4) & 1) + 4 * (i & 3);
        union { i16x4 h[2]; u32x4 v; bf16 t[8]; } u;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = row0 + 16 * b + 8 * e + 4 * g + (i >> 2);
            u.h[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (NEMO_LDS i16x4*)(lds + r * RB + (((c >> 3) ^ spread<CPR>(r)) << 4) + (c & 7) * 2));
        }
        if (clean)
#pragma unroll
            for (int e = 0; e < 8; ++e) u.t[e] = (bf16)clean_value((float)u.t[e]);
        return u.v;
    }
}

// OWN_BANK: owners are bank rows, others features.  The products of places that are left out must not count even where a feature or bank row
// holds infinities or NaN (0 x NaN): when a wave ends with a value that is not finite, it goes through its part again with such values of the
// second product's first operand taken as 0.  Where they are not left out the scores themselves, and with them dz, are NaN, and so stays
// the result.
template <typename T, int CP, bool OWN_BANK>
__global__ __launch_bounds__(256) void bank_gradient_kernel(BankArgs a) {
    constexpr int BJ = CP * sizeof(T) >= 1024 ? 32 : 64;
    __shared__ __attribute__((aligned(16))) char lds0[BJ * CP * sizeof(T)];
    __shared__ __attribute__((aligned(16))) char lds1[BJ * CP * sizeof(T)];
    __shared__ __attribute__((aligned(16))) float s_coef[2][OWN_BANK ? 6 : 1][OWN_BANK ? BJ : 4];
    __shared__ int s_again;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 5;
    const int part = (int)(blockIdx.x % a.parts);
    const int own0 = (int)(blockIdx.x / a.parts) * 128 + wave * 32, own = own0 + (lane & 31);
    const bool live = own < a.n_own;
    u32x4 q[CP / Wide<T>::KF];
    own_fragments<T, CP>(q, a, own0, lane);
    const size_t n_feat = OWN_BANK ? a.n_other : a.n_own;
    float m = 0.0f, log_s = __builtin_inff(), c = 0.0f, ge = 0.0f, gl = 0.0f;      // of an owner beyond the last: p = 0
    int target = -1;
    const float* w = nullptr;
    if (!OWN_BANK && live) {
        m = a.coef[own];
        log_s = a.coef[n_feat + own];
        c = a.coef[2 * n_feat + own];
        ge = a.coef[3 * n_feat + own];
        gl = a.coef[4 * n_feat + own];
        target = __builtin_bit_cast(int, a.coef[5 * n_feat + own]);
    }
    if (a.weights) w = OWN_BANK ? a.weights + (live ? own : 0) : a.weights + (live ? own : 0) * a.ldw;
    f32x16_t acc[CP / 32];

    auto stage = [&](char* lds, int buf, int tile) {
        stage_rows<T, CP, BJ>(lds, (const T*)a.other, a.ld_other, tile * BJ, a.n_other, a.channels, wave, lane);
        if (OWN_BANK) {
            for (int i = threadIdx.x; i < 6 * BJ; i += 256) {
                const int k = i / BJ, r = tile * BJ + i % BJ;
                // a feature row beyond the last: log s = inf, p = 0
                s_coef[buf][k][i % BJ] = r < a.n_other ? a.coef[k * n_feat + r] : k == 1 ? __builtin_inff() : k == 5 ? __builtin_bit_cast(float, -1) : 0.0f;
            }
        }
    };
    auto consume = [&](const char* lds, int buf, int tile, bool clean) {
#pragma unroll 1
        for (int s = 0; s < BJ / 32; ++s) {
            const int j0 = tile * BJ + s * 32;
            const f32x16_t pr = products<T, CP>(lds, s * 32, q, lane);
            float z[16];
            if (!OWN_BANK) {
                scores(z, pr, a.scale, w, j0, g, a.n_other);
#pragma unroll
                for (int i = 0; i < 16; ++i) z[i] = gradient_of(z[i], m, log_s, c, ge, gl, target, j0 + 8 * (i >> 2) + 4 * g + (i & 3));
            } else {
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    f32x4 k[6];
#pragma unroll
                    for (int x = 0; x < 6; ++x) k[x] = *(const f32x4*)&s_coef[buf][x][s * 32 + 8 * b + 4 * g];
                    const f32x4 tf = k[5];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int r = j0 + 8 * b + 4 * g + i;
                        float zz = w ? score(pr[4 * b + i], a.scale, w[(size_t)min(r, a.n_other - 1) * a.ldw]) : score(pr[4 * b + i], a.scale);
                        const float tb = tf[i];
                        z[4 * b + i] = gradient_of(zz, k[0][i], k[1][i], k[2][i], k[3][i], k[4][i], __builtin_bit_cast(int, tb), own);
                    }
                }
            }
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const f32x4 d = {z[4 * b], z[4 * b + 1], z[4 * b + 2], z[4 * b + 3]};
                    const u32x4 dq = __builtin_bit_cast(u32x4, d);
#pragma unroll
                    for (int x = 0; x < CP / 32; ++x) Wide<T>::run(acc[x], column_fragment<T, CP>(lds, s * 32, b, x * 32, lane, clean), dq);
                }
            } else {
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    bf16x8 hi, lo;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        hi[e] = (bf16)z[8 * b + e];
                        lo[e] = (bf16)(z[8 * b + e] - (float)hi[e]);
                    }
                    const u32x4 hq = __builtin_bit_cast(u32x4, hi), lq = __builtin_bit_cast(u32x4, lo);
#pragma unroll
                    for (int x = 0; x < CP / 32; ++x) {
                        const u32x4 p = column_fragment<T, CP>(lds, s * 32, b, x * 32, lane, clean);
                        Wide<T>::run(acc[x], p, hq);
                        Wide<T>::run(acc[x], p, lq);
                    }
                }
            }
        }
    };
    const int tiles = (a.n_other + BJ - 1) / BJ;
    const int t0 = part * a.part_tiles, t1 = min(tiles, t0 + a.part_tiles);
    for (int again = 0; again < 2; ++again) {
#pragma unroll
        for (int x = 0; x < CP / 32; ++x) acc[x] = {};
        if (t0 < t1) stage(lds0, 0, t0);
        for (int t = t0; t < t1; t += 2) {
            __syncthreads();
            if (t + 1 < t1) stage(lds1, 1, t + 1);
            consume(lds0, 0, t, again);
            if (t + 1 >= t1) break;
            __syncthreads();
            if (t + 2 < t1) stage(lds0, 0, t + 2);
            consume(lds1, 1, t + 1, again);
        }
        if (again) break;
        bool broken = false;
#pragma unroll
        for (int x = 0; x < CP / 32; ++x)
#pragma unroll
            for (int i = 0; i < 16; ++i) broken |= !(__builtin_fabsf(acc[x][i]) <= FLT_MAX);
        if (threadIdx.x == 0) s_again = 0;
        __syncthreads();                                               // also: nobody reads the tiles any more
        if (broken) s_again = 1;
        __syncthreads();
        if (!s_again) break;
    }
    if (!live) return;
#pragma unroll
    for (int x = 0; x < CP / 32; ++x)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int ch = x * 32 + 8 * b + 4 * g;
            if (a.parts > 1) {
                *(f32x4*)(a.partial + ((size_t)part * a.n_own + own) * CP + ch) =
                    (f32x4){acc[x][4 * b], acc[x][4 * b + 1], acc[x][4 * b + 2], acc[x][4 * b + 3]};
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (ch + i < a.channels) ((T*)a.grad)[(size_t)own * a.channels + ch + i] = from_f32<T>(a.scale * acc[x][4 * b + i]);
            }
        }
}

template <typename T>
__global__ __launch_bounds__(256) void bank_gradient_join_kernel(BankArgs a, int cp) {
    const long id = (long)blockIdx.x * 256 + threadIdx.x;
    if (id >= (long)a.n_own * a.channels) return;
    const int row = (int)(id / a.channels), ch = (int)(id % a.channels);
    float v = 0.0f;
    for (int s = 0; s < a.parts; ++s) v += a.partial[((size_t)s * a.n_own + row) * cp + ch];
    ((T*)a.grad)[id] = from_f32<T>(a.scale * v);
}

// rows x cols -> rows x ld_out with the columns beyond cols zero (rows that do not start on 16 bytes).
template <typename T>
__global__ __launch_bounds__(256) void pack_rows_kernel(const T* src, long ld, int rows, int cols, T* dst, int ld_out) {
    const long id = (long)blockIdx.x * 256 + threadIdx.x;
    if (id >= (long)rows * ld_out) return;
    const int r = (int)(id / ld_out), c = (int)(id % ld_out);
    dst[id] = c < cols ? src[r * ld + c] : (T)0.0f;
}

// ---- host ---------------------------------------------------------------------------------------------------------------------
static size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }
static int elem(int dtype) { return dtype == NEMO_F32 ? 4 : 2; }
static int padded_channels(int c) { return c <= 32 ? 32 : c <= 64 ? 64 : c <= 128 ? 128 : 256; }
static int tile_rows(int cp, int es) { return cp * es >= 1024 ? 32 : 64; }
static bool aligned_rows(const void* p, int64_t ld, int64_t cols, int es) {
    return ((uintptr_t)p & 15) == 0 && (ld * es) % 16 == 0 && (cols * es) % 16 == 0;
}
static size_t pack_bytes(const void* p, int64_t ld, int64_t rows, int64_t cols, int dtype) {
    return aligned_rows(p, ld, cols, elem(dtype)) ? 0 : align256((size_t)rows * padded_channels((int)cols) * elem(dtype));
}

// Parts of the other axis: two workgroups a compute unit, at least two tiles a part, at most 32.
struct Parts { int parts, tiles; };
static Parts parts_of_bank(int64_t owners, int64_t others, int cp, int es) {
    const int64_t groups = (owners + 127) / 128, tiles = (others + tile_rows(cp, es) - 1) / tile_rows(cp, es);
    int64_t p = groups > 0 ? 512 / groups : 1;
    if (p > tiles / 2) p = tiles / 2;
    if (p > 32) p = 32;
    if (p < 1) p = 1;
    const int64_t per = tiles > 0 ? (tiles + p - 1) / p : 1;
    return {(int)(tiles > 0 ? (tiles + per - 1) / per : 1), (int)per};
}

static int check_bank(const char* who, int64_t rows, int64_t cols, int64_t channels, int dtype, int top) {
    if (rows < 0 || cols < 0 || channels <= 0) return fail(NEMO_ERR_INVALID, "%s: bad size", who);
    if (dtype != NEMO_F32 && dtype != NEMO_BF16) return fail(NEMO_ERR_UNSUPPORTED, "%s: element type %d (takes f32 and bf16)", who, dtype);
    if (channels > 256) return fail(NEMO_ERR_UNSUPPORTED, "%s: %lld channels (takes up to 256)", who, (long long)channels);
    if (top < 0 || top > kMaxTop) return fail(NEMO_ERR_UNSUPPORTED, "%s: %d best entries (takes 0 to %d)", who, top, kMaxTop);
    if (rows >= (1LL << 24) || cols >= (1LL << 24)) return fail(NEMO_ERR_UNSUPPORTED, "%s: 2^24 rows or more", who);
    return NEMO_OK;
}

struct RowsIn { const void* p; int64_t ld; };
static RowsIn rows_in(int dtype, const void* p, int64_t ld, int64_t rows, int64_t cols, char*& ws, hipStream_t st) {
    if (aligned_rows(p, ld, cols, elem(dtype)) || rows == 0) return {p, ld};
    const int cp = padded_channels((int)cols);
    void* dst = ws;
    ws += pack_bytes(p, ld, rows, cols, dtype);
    const unsigned wgs = (unsigned)((rows * cp + 255) / 256);
    if (dtype == NEMO_F32)
        hipLaunchKernelGGL((pack_rows_kernel<float>), dim3(wgs), dim3(256), 0, st, (const float*)p, ld, (int)rows, (int)cols, (float*)dst, cp);
    else
        hipLaunchKernelGGL((pack_rows_kernel<bf16>), dim3(wgs), dim3(256), 0, st, (const bf16*)p, ld, (int)rows, (int)cols, (bf16*)dst, cp);
    return {dst, cp};
}

template <typename T, int CP>
static void launch_forward(const BankArgs& a, hipStream_t st) {
    const dim3 grid((unsigned)((a.n_own + 127) / 128 * a.parts));
    const int top = a.out.top;
    if (top == 0) hipLaunchKernelGGL((bank_forward_kernel<T, CP, 0>), grid, dim3(256), 0, st, a);
    else if (top == 1) hipLaunchKernelGGL((bank_forward_kernel<T, CP, 1>), grid, dim3(256), 0, st, a);
    else if (top <= 5) hipLaunchKernelGGL((bank_forward_kernel<T, CP, 5>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((bank_forward_kernel<T, CP, 16>), grid, dim3(256), 0, st, a);
}

template <typename T>
static void launch_forward(const BankArgs& a, hipStream_t st) {
    switch (padded_channels(a.channels)) {
        case 32: launch_forward<T, 32>(a, st); break;
        case 64: launch_forward<T, 64>(a, st); break;
        case 128: launch_forward<T, 128>(a, st); break;
        default: launch_forward<T, 256>(a, st);
    }
    hipLaunchKernelGGL(bank_join_kernel, dim3((a.n_own + 3) / 4), dim3(256), 0, st, a);
}

template <typename T, int CP>
static void launch_gradient(const BankArgs& a, bool own_bank, hipStream_t st) {
    const dim3 grid((unsigned)((a.n_own + 127) / 128 * a.parts));
    if (own_bank) hipLaunchKernelGGL((bank_gradient_kernel<T, CP, true>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((bank_gradient_kernel<T, CP, false>), grid, dim3(256), 0, st, a);
    if (a.parts > 1)
        hipLaunchKernelGGL((bank_gradient_join_kernel<T>), dim3((unsigned)(((long)a.n_own * a.channels + 255) / 256)), dim3(256), 0, st, a, CP);
}

template <typename T>
static void launch_gradient(const BankArgs& a, bool own_bank, hipStream_t st) {
    switch (padded_channels(a.channels)) {
        case 32: launch_gradient<T, 32>(a, own_bank, st); break;
        case 64: launch_gradient<T, 64>(a, own_bank, st); break;
        case 128: launch_gradient<T, 128>(a, own_bank, st); break;
        default: launch_gradient<T, 256>(a, own_bank, st);
    }
}

}  // namespace nemo

using namespace nemo;

extern "C" size_t nemo_bank_log_probs_workspace(const void* features, int64_t ldf, const void* bank, int64_t ldb, int64_t rows, int64_t cols,
                                                int64_t channels, int32_t dtype, int32_t top) {
    if (rows <= 0 || cols < 0 || channels <= 0 || channels > 256) return 0;
    const Parts p = parts_of_bank(rows, cols, padded_channels((int)channels), elem(dtype));
    return pack_bytes(features, ldf, rows, channels, dtype) + pack_bytes(bank, ldb, cols, channels, dtype) +
           align256((size_t)3 * 2 * p.parts * rows * 4) + 2 * align256((size_t)2 * p.parts * rows * top * 4) + align256((size_t)rows * 4);
}

extern "C" int nemo_bank_log_probs(const void* features, int64_t ldf, const void* bank, int64_t ldb, const float* weights, int64_t ldw,
                                   const int64_t* targets, int64_t rows, int64_t cols, int64_t channels, int32_t dtype, float scale,
                                   int32_t top, float* out_logp, float* out_entropy, float* out_lse, float* out_stats, float* out_top_logp,
                                   int64_t* out_top_index, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check_bank("nemo_bank_log_probs", rows, cols, channels, dtype, top);
    if (rc) return rc;
    if (rows == 0) return NEMO_OK;
    if (!features || !targets || (cols > 0 && !bank) || (top > 0 && (!out_top_logp || !out_top_index)))
        return fail(NEMO_ERR_INVALID, "nemo_bank_log_probs: null argument");
    if (ldf < channels || (cols > 0 && ldb < channels) || (weights && ldw != 0 && ldw < cols))
        return fail(NEMO_ERR_INVALID, "nemo_bank_log_probs: a row stride shorter than the row");
    if ((uintptr_t)out_stats & 15) return fail(NEMO_ERR_INVALID, "nemo_bank_log_probs: out_stats must start on 16 bytes");
    const size_t need = nemo_bank_log_probs_workspace(features, ldf, bank, ldb, rows, cols, channels, dtype, top);
    if (workspace_bytes < need || (need && !workspace))
        return fail(NEMO_ERR_INVALID, "nemo_bank_log_probs: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    hipStream_t st = (hipStream_t)stream;
    char* ws = (char*)workspace;
    const RowsIn f = rows_in(dtype, features, ldf, rows, channels, ws, st), b = rows_in(dtype, bank, ldb, cols, channels, ws, st);
    const Parts p = parts_of_bank(rows, cols, padded_channels((int)channels), elem(dtype));
    BankArgs a = {};
    a.own = f.p; a.ld_own = f.ld; a.n_own = (int)rows;
    a.other = b.p; a.ld_other = b.ld; a.n_other = (int)cols;
    a.channels = (int)channels;
    a.weights = weights; a.ldw = ldw; a.targets = (const long long*)targets; a.scale = scale;
    a.parts = p.parts; a.part_tiles = p.tiles;
    a.part_state = (float*)ws;
    ws += align256((size_t)3 * 2 * p.parts * rows * 4);
    a.part_z = (float*)ws;
    ws += align256((size_t)2 * p.parts * rows * top * 4);
    a.part_place = (int*)ws;
    ws += align256((size_t)2 * p.parts * rows * top * 4);
    a.z_target = (float*)ws;
    a.out = {out_logp, out_entropy, out_lse, out_stats, out_top_logp, (long long*)out_top_index, top};
    if (dtype == NEMO_F32) launch_forward<float>(a, st);
    else launch_forward<bf16>(a, st);
    HIP_TRY(hipGetLastError());
    return NEMO_OK;
}

extern "C" size_t nemo_bank_log_probs_backward_workspace(const void* features, int64_t ldf, const void* bank, int64_t ldb, int64_t rows,
                                                         int64_t cols, int64_t channels, int32_t dtype) {
    if (rows <= 0 || cols <= 0 || channels <= 0 || channels > 256) return 0;
    const int cp = padded_channels((int)channels);
    const Parts pf = parts_of_bank(rows, cols, cp, elem(dtype)), pb = parts_of_bank(cols, rows, cp, elem(dtype));
    const size_t bf = pf.parts > 1 ? (size_t)pf.parts * rows * cp * 4 : 0, bb = pb.parts > 1 ? (size_t)pb.parts * cols * cp * 4 : 0;
    return pack_bytes(features, ldf, rows, channels, dtype) + pack_bytes(bank, ldb, cols, channels, dtype) + align256((size_t)6 * rows * 4) +
           align256(bf > bb ? bf : bb);
}

extern "C" int nemo_bank_log_probs_backward(const void* features, int64_t ldf, const void* bank, int64_t ldb, const float* weights, int64_t ldw,
                                            const int64_t* targets, const float* stats, const float* g_logp, const float* g_entropy,
                                            const float* g_lse, int64_t rows, int64_t cols, int64_t channels, int32_t dtype, float scale,
                                            void* grad_features, void* grad_bank, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check_bank("nemo_bank_log_probs_backward", rows, cols, channels, dtype, 0);
    if (rc) return rc;
    if (rows == 0 || cols == 0) return NEMO_OK;
    if (!features || !bank || !targets || !stats) return fail(NEMO_ERR_INVALID, "nemo_bank_log_probs_backward: null argument");
    if (ldf < channels || ldb < channels || (weights && ldw != 0 && ldw < cols))
        return fail(NEMO_ERR_INVALID, "nemo_bank_log_probs_backward: a row stride shorter than the row");
    if ((uintptr_t)stats & 15) return fail(NEMO_ERR_INVALID, "nemo_bank_log_probs_backward: stats must start on 16 bytes");
    const size_t need = nemo_bank_log_probs_backward_workspace(features, ldf, bank, ldb, rows, cols, channels, dtype);
    if (workspace_bytes < need || (need && !workspace))
        return fail(NEMO_ERR_INVALID, "nemo_bank_log_probs_backward: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    hipStream_t st = (hipStream_t)stream;
    char* ws = (char*)workspace;
    const RowsIn f = rows_in(dtype, features, ldf, rows, channels, ws, st), b = rows_in(dtype, bank, ldb, cols, channels, ws, st);
    float* coef = (float*)ws;
    ws += align256((size_t)6 * rows * 4);
    hipLaunchKernelGGL(bank_coef_kernel, dim3((unsigned)((rows + 255) / 256)), dim3(256), 0, st, stats, g_logp, g_entropy, g_lse,
                       (const long long*)targets, (int)rows, (int)cols, coef);
    const int cp = padded_channels((int)channels);
    for (int own_bank = 0; own_bank < 2; ++own_bank) {
        void* grad = own_bank ? grad_bank : grad_features;
        if (!grad) continue;
        const RowsIn own = own_bank ? b : f, other = own_bank ? f : b;
        const int64_t n_own = own_bank ? cols : rows, n_other = own_bank ? rows : cols;
        const Parts p = parts_of_bank(n_own, n_other, cp, elem(dtype));
        BankArgs a = {};
        a.own = own.p; a.ld_own = own.ld; a.n_own = (int)n_own;
        a.other = other.p; a.ld_other = other.ld; a.n_other = (int)n_other;
        a.channels = (int)channels;
        a.weights = weights; a.ldw = ldw; a.targets = (const long long*)targets; a.scale = scale;
        a.parts = p.parts; a.part_tiles = p.tiles;
        a.coef = coef; a.partial = (float*)ws; a.grad = grad;
        if (dtype == NEMO_F32) launch_gradient<float>(a, own_bank, st);
        else launch_gradient<bf16>(a, own_bank, st);
    }
    HIP_TRY(hipGetLastError());
    return NEMO_OK;
}
