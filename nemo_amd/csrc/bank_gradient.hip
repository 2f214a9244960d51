// The gradients of bank_log_probs.hip.  The scores are computed again (first product, bank_tiles.h); dz (softmax_state.h) in its registers is, as
// it stands, the second operand of a second product
//     gradient^T[c][owner] += sum_j other[j][c] dz[j][owner],
// whose k runs in the order of those registers; the first operand is read from LDS in that order.
//     features' gradient   owners = features, others = bank
//     bank's gradient      owners = bank rows, others = features; what dz needs of a feature row is staged beside the tile
// In bf16 dz is split into two pieces, dz = hi + lo, each of them multiplied: a single piece would put an error of 2^-9 of the largest term into
// sums whose terms largely cancel (the target's against all others').  The other axis is split where there are too few owners to fill the
// device; the parts are joined in their order by a second kernel.  Results of two calls are the same bits.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/nemo_hip.h"
#include "bank_tiles.h"

namespace nemo {

__global__ __launch_bounds__(256) void bank_coef_kernel(const float* stats, const float* g_logp, const float* g_entropy, const float* g_lse,
                                                        const long long* targets, int rows, int cols, float* coef, bool join_m) {
    const int row = blockIdx.x * 256 + threadIdx.x, n = coef_rows(rows);
    if (row >= n) return;
    RowCoef k = {0.0f, __builtin_inff(), 0.0f, 0.0f, 0.0f, -1};
    if (row < rows) k = row_coef(stats, g_logp, g_entropy, g_lse, targets, row, cols);
    coef[K_M * n + row] = join_m ? k.m + k.log2_s : k.m;
    coef[K_LOG2_S * n + row] = k.log2_s;
    coef[K_C * n + row] = k.c;
    coef[K_G2 * n + row] = k.g2;
    coef[K_LOGP * n + row] = k.g_logp;
    coef[K_TARGET * n + row] = __builtin_bit_cast(float, k.target);
}

// dz of one score or product without the target's share.  In bf16 and without weights m holds m + log2 s, one operation less: off by u |lse|
// (1e-6 at 16), far below the rounding of dz's pieces.  SAFE: log2 p may be -inf.
template <typename T, bool GENERAL, bool SAFE>
__device__ inline float pair_gradient(float v, float k, float m, float log2_s, float c, float g2) {
    float lp2;
    if (GENERAL) lp2 = __builtin_fmaf(v - m, kLog2e, -log2_s);
    else if (sizeof(T) == 4) lp2 = __builtin_fmaf(k, v, -m) - log2_s;
    else lp2 = __builtin_fmaf(k, v, -m);
    return SAFE ? prob_gradient(lp2, c, g2) : exp2_fast(lp2) * (c - g2 * lp2);
}

// A value of the second product's first operand; `clean` turns infinities and NaN into 0 (see bank_gradient_kernel).
__device__ inline float clean_value(float v) { return __builtin_fabsf(v) <= FLT_MAX ? v : 0.0f; }

// First operand of the second product: columns cb .. cb + 31 (cb a multiple of 32) of the tile's rows, in the order in which the first product's
// registers hold them.  f32: step b takes registers 4 b .. 4 b + 3, rows 8 b + 4 g + i.  bf16: step b takes registers 8 b .. 8 b + 7, rows
// 16 b + 8 (e / 4) + 4 g + e % 4, two transposing reads of four rows each (lane i of a group of 16 supplies columns 4 (i % 4) .. + 3 of row
// i / 4 and receives column i of the four rows).
template <typename T, int CP>
__device__ inline u32x4 column_fragment(const char* lds, int row0, int b, int cb, int lane, bool clean) {
    typedef Tile<T, CP> L;
    const int g = lane >> 5;
    if constexpr (sizeof(T) == 4) {
        u32x4 v;
        const int low = (lane & 31) >> 2;                              // chunk within the 32 columns; flip reaches no further
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int f = L::RPI == 8 ? 4 * g + i : L::flip(i);        // flip of row 8 b + 4 g + i
            float x = *(const float*)(lds + L::row(row0) + L::row(8 * b + i) + cb * 4 + L::row(4) * g + ((low ^ f) << 4) + (lane & 3) * 4);
            if (clean) x = clean_value(x);
            v[i] = __builtin_bit_cast(uint32_t, x);
        }
        return v;
    } else {
        const int i = lane & 15, t = 2 * ((lane >> 4) & 1) + ((i & 3) >> 1), r = 4 * g + (i >> 2);
        const int low = (((cb >> 3) & L::MASK) + t) ^ L::flip(r);
        const char* at = lds + L::row(row0) + L::row(16 * b) + (((cb >> 3) & ~L::MASK) << 4) + L::row(4) * g + L::row(i >> 2) + (low << 4) + (i & 1) * 8;
        union { i16x4 h[2]; u32x4 v; bf16 t[8]; } u;
        u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((NEMO_LDS i16x4*)at);
        u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((NEMO_LDS i16x4*)(at + (L::RPI >= 16 ? 8 * L::RB : L::row(8))));
        if (clean)
#pragma unroll
            for (int e = 0; e < 8; ++e) u.t[e] = (bf16)clean_value((float)u.t[e]);
        return u.v;
    }
}

// OWN_BANK: owners are bank rows, others features.  The products of places that are left out must not count even where a feature or bank row
// holds infinities or NaN (0 x NaN): when a wave ends with a value that is not finite, its workgroup goes through its part again with such
// values of the second product's first operand taken as 0 (and with log2 p = -inf allowed for).  Where they are not left out the scores themselves, and with them dz, are NaN, and
// so stays the result.
// GENERAL as in the forward kernel.
template <typename T, int CP, bool OWN_BANK, bool GENERAL>
__global__ __launch_bounds__(256, CP == 256 ? 1 : 2) void bank_gradient_kernel(BankArgs a) {
    constexpr int BJ = Tile<T, CP>::ROWS;
    constexpr bool F32 = sizeof(T) == 4, SPLIT = GENERAL || F32;       // log2 s apart from m
    __shared__ __attribute__((aligned(16))) char lds0[Tile<T, CP>::BYTES];
    __shared__ __attribute__((aligned(16))) char lds1[Tile<T, CP>::BYTES];
    __shared__ __attribute__((aligned(16))) float s_coef0[OWN_BANK ? K_COUNT : 1][64];
    __shared__ __attribute__((aligned(16))) float s_coef1[OWN_BANK ? K_COUNT : 1][64];
    __shared__ int s_again;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 5;
    const int part = (int)(blockIdx.x % a.parts);
    const int own0 = (int)(blockIdx.x / a.parts) * 128 + wave * 32, own = own0 + (lane & 31);
    const bool live = own < a.n_own;
    u32x4 q[CP / Wide<T>::KF];
    own_fragments<T, CP>(q, a, own0, lane, !GENERAL && a.scale < 0.0f);
    const int n_coef = coef_rows(OWN_BANK ? a.n_other : a.n_own);
    const float k = a.out.k;
    float m = 0.0f, log2_s = __builtin_inff(), c = 0.0f, g2 = 0.0f, gl = 0.0f;     // of an owner beyond the last
    int target = -1;
    const float* w = nullptr;
    if (!OWN_BANK && live) {
        m = a.coef[K_M * n_coef + own];
        log2_s = a.coef[K_LOG2_S * n_coef + own];
        c = a.coef[K_C * n_coef + own];
        g2 = a.coef[K_G2 * n_coef + own];
        gl = a.coef[K_LOGP * n_coef + own];
        target = __builtin_bit_cast(int, a.coef[K_TARGET * n_coef + own]);
    }
    if (GENERAL && a.weights) w = OWN_BANK ? a.weights + (live ? own : 0) : a.weights + (live ? own : 0) * a.ldw;
    f32x16_t acc[CP / 32];

    auto stage = [&](char* lds, float (*coef)[64], int tile) __attribute__((always_inline)) {
        stage_rows<T, CP>(lds, (const T*)a.other, a.ld_other, tile * BJ, a.n_other, a.channels, wave, lane);
        if (OWN_BANK) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (wave + 4 * i < K_COUNT)
                    copy_words_to_lds(a.coef + (size_t)(wave + 4 * i) * n_coef + tile * BJ + lane, &coef[OWN_BANK ? wave + 4 * i : 0][0]);
        }
    };
    auto consume = [&](const char* lds, const float (*coef)[64], int tile, auto clean_tag) __attribute__((always_inline)) {
        constexpr bool CLEAN = decltype(clean_tag)::value, SAFE = GENERAL || CLEAN;
#pragma unroll 1
        for (int s = 0; s < BJ / 32; ++s) {
            const int j0 = tile * BJ + s * 32;
            float wv[16];
            if (GENERAL && w) {
                if (!OWN_BANK) {
                    row_weights(wv, w, j0, g, a.n_other);
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        wv[i] = w[(size_t)min(j0 + 8 * (i >> 2) + 4 * g + (i & 3), a.n_other - 1) * a.ldw];
                }
            }
            const f32x16_t pr = products<T, CP>(lds, s * 32, q, lane);
            float z[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) z[i] = !GENERAL ? pr[i] : w ? score(pr[i], a.scale, wv[i]) : score(pr[i], a.scale);
            // dz; the target's share only where the block holds some target
            if (!OWN_BANK) {
                const bool hit = __any(target >= j0 && target < j0 + 32);
                const int at = target - j0 - 4 * g, left = a.n_other - j0 - 4 * g;
                uint32_t gone = 0;
                if (GENERAL && hit) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) gone |= z[i] == neg_inf() ? 1u << i : 0u;
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) z[i] = pair_gradient<T, GENERAL, SAFE>(z[i], k, m, log2_s, c, g2);
                if (hit) {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (at == 8 * (i >> 2) + (i & 3) && !(gone >> i & 1)) z[i] += gl;
                }
                if (j0 + 32 > a.n_other) {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (8 * (i >> 2) + (i & 3) >= left) z[i] = 0.0f;
                }
            } else {
                const int t = __builtin_bit_cast(int, coef[K_TARGET][s * 32 + (lane & 31)]);
                const bool hit = __any(t >= own0 && t < own0 + 32);
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const int r = s * 32 + 8 * b + 4 * g;
                    const f32x4 km = *(const f32x4*)&coef[K_M][r], kc = *(const f32x4*)&coef[K_C][r], kg = *(const f32x4*)&coef[K_G2][r];
                    f32x4 ks = {};
                    if (SPLIT) ks = *(const f32x4*)&coef[K_LOG2_S][r];
                    if (!hit) {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            z[4 * b + i] = pair_gradient<T, GENERAL, SAFE>(z[4 * b + i], k, km[i], ks[i], kc[i], kg[i]);
                    } else {
                        const f32x4 kl = *(const f32x4*)&coef[K_LOGP][r], kt = *(const f32x4*)&coef[K_TARGET][r];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float v = z[4 * b + i], d = pair_gradient<T, GENERAL, SAFE>(v, k, km[i], ks[i], kc[i], kg[i]), tb = kt[i];
                            z[4 * b + i] = __builtin_bit_cast(int, tb) == own && !(GENERAL && v == neg_inf()) ? d + kl[i] : d;
                        }
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            // the second product; fragments are read one step ahead of the matrix cores, no further
            if constexpr (F32) {
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const f32x4 d = {z[4 * b], z[4 * b + 1], z[4 * b + 2], z[4 * b + 3]};
                    const u32x4 dq = __builtin_bit_cast(u32x4, d);
#pragma unroll
                    for (int x = 0; x < CP / 32; ++x) {
                        Wide<T>::run(acc[x], column_fragment<T, CP>(lds, s * 32, b, x * 32, lane, CLEAN), dq);
                        if (x % 4 == 3) __builtin_amdgcn_sched_barrier(0);
                    }
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
                        const u32x4 p = column_fragment<T, CP>(lds, s * 32, b, x * 32, lane, CLEAN);
                        Wide<T>::run(acc[x], p, hq);
                        Wide<T>::run(acc[x], p, lq);
                        if (x % 4 == 3) __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
        }
    };
    const int tiles = (a.n_other + BJ - 1) / BJ;
    const int t0 = part * a.part_tiles, t1 = min(tiles, t0 + a.part_tiles);
    auto pass = [&](auto clean_tag) __attribute__((always_inline)) {
#pragma unroll
        for (int x = 0; x < CP / 32; ++x) acc[x] = {};
        if (t0 < t1) stage(lds0, s_coef0, t0);
        for (int t = t0; t < t1; t += 2) {
            __syncthreads();
            if (t + 1 < t1) stage(lds1, s_coef1, t + 1);
            consume(lds0, s_coef0, t, clean_tag);
            if (t + 1 >= t1) break;
            __syncthreads();
            if (t + 2 < t1) stage(lds0, s_coef0, t + 2);
            consume(lds1, s_coef1, t + 1, clean_tag);
        }
    };
    pass(std::false_type{});
    bool broken = false;
#pragma unroll
    for (int x = 0; x < CP / 32; ++x)
#pragma unroll
        for (int i = 0; i < 16; ++i) broken |= !(__builtin_fabsf(acc[x][i]) <= FLT_MAX);
    if (threadIdx.x == 0) s_again = 0;
    __syncthreads();                                                   // also: nobody reads the tiles any more
    if (broken) s_again = 1;
    __syncthreads();
    if (s_again) pass(std::true_type{});
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


template <typename T, int CP>
static void launch_gradient(const BankArgs& a, bool own_bank, hipStream_t st) {
    const dim3 grid((unsigned)((a.n_own + 127) / 128 * a.parts));
    const bool general = a.out.k == 0.0f;
    if (own_bank) {
        if (general) hipLaunchKernelGGL((bank_gradient_kernel<T, CP, true, true>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((bank_gradient_kernel<T, CP, true, false>), grid, dim3(256), 0, st, a);
    } else {
        if (general) hipLaunchKernelGGL((bank_gradient_kernel<T, CP, false, true>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((bank_gradient_kernel<T, CP, false, false>), grid, dim3(256), 0, st, a);
    }
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


void launch_bank_gradient(const BankArgs& a, int dtype, bool own_bank, hipStream_t st) {
    if (dtype == NEMO_F32) launch_gradient<float>(a, own_bank, st);
    else launch_gradient<bf16>(a, own_bank, st);
}

void launch_bank_coef(const float* stats, const float* g_logp, const float* g_entropy, const float* g_lse, const long long* targets, int rows,
                      int cols, float* coef, bool join_m, hipStream_t st) {
    hipLaunchKernelGGL(bank_coef_kernel, dim3((unsigned)((coef_rows(rows) + 255) / 256)), dim3(256), 0, st, stats, g_logp, g_entropy, g_lse,
                       targets, rows, cols, coef, join_m);
}

}  // namespace nemo
