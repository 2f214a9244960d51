// The gradients of bank_log_probs.hip.  The scores are computed again (first product, bank_tiles.h); dz (softmax_state.h) in its registers is, as
// it stands, the second operand of a second product
//     gradient^T[c][owner] += sum_j other[j][c] dz[j][owner],
// whose k runs in the order of those registers; the first operand is read from LDS in that order.
//     features' gradient   owners = features, others = bank
//     bank's gradient      owners = bank rows, others = features; what dz needs of a feature row is staged beside the tile
// In bf16 dz is split into two pieces, dz = hi + lo, each of them multiplied: a single piece would put an error of 2^-9 of the largest term into
// sums whose terms largely cancel (the target's against all others').  The other axis is split where there are too few owners to fill the
// device; the parts are joined in their order by a second kernel.  Results of two calls are the same bits.  Compiled once for each element type
// (NEMO_ELEMENT).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/nemo_hip.h"
#include "bank_tiles.h"

namespace nemo {

// dz of one score or product without the target's share.  In bf16 and without weights m holds m + log2 s, one operation less: log2 p off by u |lse| /
// log 2 more, as much as the sums behind a score of that size are off themselves, and below the rounding of dz's pieces up to |lse| of
// about 100.  SAFE: log2 p may be -inf.
template <bool F32, bool GENERAL, bool SAFE>
__device__ inline float pair_gradient(float v, float k, float m, float log2_s, float c, float g2) {
    float lp2;
    if (GENERAL) lp2 = __builtin_fmaf(v - m, kLog2e, -log2_s);
    else if (F32) lp2 = __builtin_fmaf(k, v, -m) - log2_s;
    else lp2 = __builtin_fmaf(k, v, -m);
    return SAFE ? prob_gradient(lp2, c, g2) : exp2_fast(lp2) * (c - g2 * lp2);
}

// A value of the second product's first operand; `clean` turns infinities and NaN into 0 (see bank_gradient_kernel).
__device__ inline float clean_value(float v) { return __builtin_fabsf(v) <= FLT_MAX ? v : 0.0f; }

// First operand of the second product: columns cb .. cb + 31 (cb a multiple of 32) of the tile's rows, one piece, in the order in which the first
// product's registers hold them: step b takes registers 8 b .. 8 b + 7, rows 16 b + 8 (e / 4) + 4 g + e % 4, two transposing reads of four
// rows each (lane i of a group of 16 supplies columns 4 (i % 4) .. + 3 of row i / 4 and receives column i of the four rows).
template <int CP>
__device__ inline u32x4 column_fragment(const char* lds, int b, int cb, int lane, bool clean) {
    typedef Tile<CP> L;
    const int g = lane >> 5, i = lane & 15, t = 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
    union { i16x4 h[2]; u32x4 v; bf16 t[8]; } u;
#pragma unroll
    for (int e = 0; e < 2; ++e)
        u.h[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (NEMO_LDS i16x4*)(lds + L::row(16 * b + 8 * e) + L::row(4) * g + L::row(i >> 2) + L::chunk(cb >> 3, t, L::flip(8 * e + 4 * g + (i >> 2))) + (i & 1) * 8));
    if (clean)
#pragma unroll
        for (int e = 0; e < 8; ++e) u.t[e] = (bf16)clean_value((float)u.t[e]);
    return u.v;
}

// 16 dz of a lane as second operands of the second product, filled two values at a time.  Rows of one piece: dz = hi + lo, 16 bits, both multiplied.
// Rows of three pieces: dz of three pieces, paired as in the first product.
template <int NP> struct Pieces {
    static constexpr int STEPS = 2, N = NP == 1 ? 2 : 3, PAIRS = NP == 1 ? 2 : 6;
    static __device__ constexpr int first(int u) { return NP == 1 ? 0 : Pairs<3>::first(u); }       // piece of the rows
    static __device__ constexpr int second(int u) { return NP == 1 ? u : Pairs<3>::second(u); }     // piece of dz
    u32x4 p[STEPS][N];
    __device__ inline void pair(int i, float z0, float z1) {
        typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const bf16x2 hi = {(bf16)z0, (bf16)z1};
            const uint32_t h = __builtin_bit_cast(uint32_t, hi);
            p[i >> 2][n][i & 3] = h;
            z0 -= __builtin_bit_cast(float, h << 16);
            z1 -= __builtin_bit_cast(float, h & 0xFFFF0000u);
        }
    }
    __device__ inline void settle_pair(int i) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            uint32_t x = p[i >> 2][n][i & 3];
            asm volatile("" : "+v"(x));
            p[i >> 2][n][i & 3] = x;
        }
    }
};

template <int NP, int CP>
__device__ inline void second_product(f32x16_t (&acc)[CP / 32], const char* lds, const Pieces<NP>& dz, int lane, bool clean) {
    typedef Pieces<NP> P;
#pragma unroll
    for (int b = 0; b < P::STEPS; ++b)
#pragma unroll
        for (int x = 0; x < CP / 32; ++x) {
            u32x4 f[NP];
#pragma unroll
            for (int n = 0; n < NP; ++n) f[n] = column_fragment<CP>(lds + n * Tile<CP>::BYTES, b, x * 32, lane, clean);
#pragma unroll
            for (int u = 0; u < P::PAIRS; ++u) wide_mma(acc[x], f[P::first(u)], dz.p[b][P::second(u)]);
        }
}

// OWN_BANK: owners are bank rows, others features.  GENERAL as in the forward kernel.
//
// Tiles of 32 other rows.  Matrix cores and vector units work side by side only if a wave has something for both: in step n it multiplies
// tile n + 1 (first product), computes dz of tile n from the products of the step before, and multiplies the dz of tile n - 1 (second product),
// none of which waits for another; the instructions are interleaved in slices that the compiler may not mix.  That takes four tiles in LDS (n - 1, n,
// n + 1 and n + 2 on its way), one barrier a step, and straight code: the targets' share of dz is left out of it and added at the end.  In the
// features' gradient it is one bank row a feature row; in the bank's gradient the feature rows whose targets are among the owners are gathered
// and multiplied (a product of its own in every step that has one costs all four waves its time: 10007 rows
// of 3678 places, 128 channels: 163 us against 117 in f32, 110 against 78 in bf16 with weights).  At 256 channels there are not enough registers for two steps at once: one after the other.
//
// Measured (features' gradient / bank's gradient, us).  32768 x 15976 x 128 bf16: 335 / 380; the three products of a pair take 303; the bank's reads
// what dz needs of every feature row from LDS, with which LDS (2.0 k cycles a step of eight waves) is busier than the matrix cores (1.5 k).
// 10007 x 3678 x 128 f32: 109 / 117, with weights for every pair 125 / 147; the twelve products of a pair take 85.  Weights loaded a
// step ahead, in 16 more registers, changed nothing (128 / 152): the compiler waits for all loads under way at the first transposing read of a
// step, for those too.  It is also why four tiles hide no more of a copy than part of a step.
//
// Products of places that are left out must not count even where a feature or bank row holds infinities or NaN (0 x NaN): when a wave ends with
// a value that is not finite, its workgroup goes through its part again, step after step, with such values of the second product's first
// operand taken as 0 and with log2 p = -inf allowed for.  Where they are not left out the scores themselves, and with them dz, are NaN, and
// so stays the result.
template <typename T, int CP, bool OWN_BANK, bool GENERAL>
__global__ __launch_bounds__(256, CP == 256 || (CP == 128 && sizeof(T) == 4) ? 1 : 2) void bank_gradient_kernel(BankArgs a) {
    typedef Tile<CP> L;
    constexpr bool F32 = sizeof(T) == 4, SPLIT = GENERAL || F32;       // log2 s apart from m
    constexpr bool SIDE_BY_SIDE = CP <= 128;
    constexpr int NP = F32 ? 3 : 1, NX = CP / 32, NKF = CP / kFragK;
    typedef Pieces<NP> Dz;
    __shared__ __attribute__((aligned(16))) char lds0[NP * L::BYTES];
    __shared__ __attribute__((aligned(16))) char lds1[NP * L::BYTES];
    __shared__ __attribute__((aligned(16))) char lds2[SIDE_BY_SIDE ? NP * L::BYTES : 16];
    __shared__ __attribute__((aligned(16))) char lds3[SIDE_BY_SIDE ? NP * L::BYTES : 16];
    __shared__ __attribute__((aligned(16))) float s_coef0[OWN_BANK ? K_COUNT : 1][64];
    __shared__ __attribute__((aligned(16))) float s_coef1[OWN_BANK ? K_COUNT : 1][64];
    __shared__ __attribute__((aligned(16))) float s_coef2[OWN_BANK && SIDE_BY_SIDE ? K_COUNT : 1][64];
    __shared__ __attribute__((aligned(16))) float s_coef3[OWN_BANK && SIDE_BY_SIDE ? K_COUNT : 1][64];
    __shared__ int s_again;
    // of the targets' share: feature rows (fewer than 32 left over and those of one look), how many each wave found, what belongs to 32 of them
    __shared__ int s_list[OWN_BANK ? 32 + 1024 : 1], s_found[16], s_target[32];
    __shared__ float s_share[32];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 5;
    const int part = (int)(blockIdx.x % a.parts);
    const int own0 = (int)(blockIdx.x / a.parts) * 128 + wave * 32, own = own0 + (lane & 31);
    const bool live = own < a.n_own;
    u32x4 q[NP][NKF];
    own_fragments<NP, CP>(q, a, own0, lane, !GENERAL && a.scale < 0.0f);
    const int n_coef = coef_rows(OWN_BANK ? a.n_other : a.n_own);
    const float k = a.out.k;
    float m = 0.0f, log2_s = 0.0f, c = 0.0f, g2 = 0.0f;               // of an owner beyond the last: dz = 0
    const float* w = nullptr;
    if (!OWN_BANK && live) {
        m = a.coef[K_M * n_coef + own];
        log2_s = a.coef[K_LOG2_S * n_coef + own];
        c = a.coef[K_C * n_coef + own];
        g2 = a.coef[K_G2 * n_coef + own];
    }
    if (GENERAL && a.weights) w = OWN_BANK ? a.weights + (live ? own : 0) : a.weights + (live ? own : 0) * a.ldw;
    f32x16_t acc[NX];

    const Stager<NP, CP> stager(a, wave, lane);
    auto stage = [&](char* lds, float (*coef)[64], int tile) __attribute__((always_inline)) {
        stager.copy(lds, tile);
        if (OWN_BANK) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (wave + 4 * i < K_COUNT)
                    copy_words_to_lds(a.coef + (size_t)(wave + 4 * i) * n_coef + tile * 32 + lane, &coef[OWN_BANK ? wave + 4 * i : 0][0]);
        }
    };
    auto load_weights = [&](float (&wv)[16], int tile) __attribute__((always_inline)) {
        if (!GENERAL || !w) return;
        const int j0 = tile * 32;
        if (!OWN_BANK) {
            row_weights(wv, w, j0, g, a.n_other);
        } else if (j0 + 32 <= a.n_other) {
            // 32-bit offsets of a lane from addresses that all lanes share
            const uint32_t at = (uint32_t)((live ? own : 0) + 4 * g * (int)a.ldw);
#pragma unroll
            for (int i = 0; i < 16; ++i) wv[i] = (a.weights + (size_t)(j0 + 8 * (i >> 2) + (i & 3)) * a.ldw)[at];
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int j = j0 + 8 * (i >> 2) + 4 * g + (i & 3);
                wv[i] = j < a.n_other ? w[(size_t)j * a.ldw] : __builtin_inff();
            }
        }
    };
    // what dz needs of the four feature rows 8 b + 4 g + i, or of the owner
    struct Quad { f32x4 m, s, c, g2; };
    auto quad = [&](const float (*coef)[64], int b) __attribute__((always_inline)) {
        Quad k4 = {{m, m, m, m}, {log2_s, log2_s, log2_s, log2_s}, {c, c, c, c}, {g2, g2, g2, g2}};
        if (OWN_BANK) {
            const int r = 8 * b + 4 * g;
            k4.m = *(const f32x4*)&coef[K_M][r];
            k4.c = *(const f32x4*)&coef[OWN_BANK ? K_C : 0][r];
            k4.g2 = *(const f32x4*)&coef[OWN_BANK ? K_G2 : 0][r];
            if (SPLIT) k4.s = *(const f32x4*)&coef[OWN_BANK ? K_LOG2_S : 0][r];
        }
        return k4;
    };
    // product i of a tile -> dz without the targets' share
    auto differentiate = [&](const f32x16_t& pr, const float (&wv)[16], const Quad& k4, int i, int tile, auto safe_tag) __attribute__((always_inline)) {
        constexpr bool SAFE = decltype(safe_tag)::value || GENERAL;
        const float s = !GENERAL ? pr[i] : w ? score(pr[i], a.scale, wv[i]) : score(pr[i], a.scale);
        const float d = pair_gradient<F32, GENERAL, SAFE>(s, k, k4.m[i & 3], k4.s[i & 3], k4.c[i & 3], k4.g2[i & 3]);
        // rows beyond the last are zeros (with weights, left out), but where all scores are far below 0 the probability of a 0 is not even finite
        return decltype(safe_tag)::value && !OWN_BANK && !(GENERAL && w) && tile * 32 + 8 * (i >> 2) + 4 * g + (i & 3) >= a.n_other ? 0.0f : d;
    };
    const int tiles = (a.n_other + 31) / 32;
    const int t0 = part * a.part_tiles, t1 = min(tiles, t0 + a.part_tiles);

    // one step after the other
    auto plain_pass = [&](auto clean_tag) __attribute__((always_inline)) {
        constexpr bool CLEAN = decltype(clean_tag)::value;
#pragma unroll
        for (int x = 0; x < NX; ++x) acc[x] = {};
        auto one = [&](const char* lds, const float (*coef)[64], int tile) __attribute__((always_inline)) {
            float wv[16];
            load_weights(wv, tile);
            const f32x16_t pr = products<NP, CP>(lds, q, lane);
            Dz dz;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const Quad k4 = quad(coef, b);
                float z[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) z[i] = differentiate(pr, wv, k4, 4 * b + i, tile, clean_tag);
                dz.pair(2 * b, z[0], z[1]);
                dz.pair(2 * b + 1, z[2], z[3]);
            }
            __builtin_amdgcn_sched_barrier(0);
            second_product<NP, CP>(acc, lds, dz, lane, CLEAN);
        };
        if (t0 < t1) stage(lds0, s_coef0, t0);
        for (int t = t0; t < t1; t += 2) {
            publish_lds();
            if (t + 1 < t1) stage(lds1, s_coef1, t + 1);
            one(lds0, s_coef0, t);
            if (t + 1 >= t1) break;
            publish_lds();
            if (t + 2 < t1) stage(lds0, s_coef0, t + 2);
            one(lds1, s_coef1, t + 1);
        }
    };
    // two products and dz side by side
    auto pass = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int x = 0; x < NX; ++x) acc[x] = {};
        if (t0 >= t1) return;
        Dz dz = {};                                             // of the tile before, whose rows are in lds3 at the start
        for (int i = threadIdx.x * 16; i < NP * L::BYTES; i += 4096) *(u32x4*)(lds3 + i) = u32x4{0, 0, 0, 0};
        stage(lds0, s_coef0, t0);
        if (t0 + 1 < t1) stage(lds1, s_coef1, t0 + 1);
        publish_lds();
        f32x16_t pr = products<NP, CP>(lds0, q, lane);
        auto step = [&](int t, const char* before, const char* next, char* after, const float (*coef)[64],
                        float (*coef_after)[64]) __attribute__((always_inline)) {
            publish_lds();                                             // tile t + 1 is there; nobody reads tile t - 2 any more
            stage(after, coef_after, t + 2);                           // also behind the part's last tile, to no effect: no branch
            float wv[16];
            load_weights(wv, t);
            f32x16_t nxt = {};
            Dz mine;
            float z[16];
            Quad k4 = quad(coef, 0), ahead_k4 = k4;
            // One slice: one matrix instruction and a share of dz: 16 values, then, in pairs, their pieces.  Fragments are read two ahead.  Weights may
            // arrive during the first half of the slices.
            constexpr int G1 = Pairs<NP>::N, G2 = Dz::PAIRS, S1 = NKF * G1, SLICES = S1 + NX * Dz::STEPS * G2, UNITS = 24;
            constexpr int F1 = NKF * NP, FRAGS = F1 + NX * Dz::STEPS * NP;
            u32x4 f[3];
            auto read = [&](int n) __attribute__((always_inline)) {
                const int piece = n % NP * L::BYTES, group = (n - F1) / NP;
                if (n < F1) f[n % 3] = row_fragment<CP>(next + piece, n / NP, lane);
                else if (n < FRAGS) f[n % 3] = column_fragment<CP>(before + piece, group / NX, group % NX * 32, lane, false);
            };
            read(0);
            read(1);
#pragma unroll
            for (int i = 0; i < SLICES; ++i) {
                const bool one = i < S1;
                const int group = one ? i / G1 : (i - S1) / G2, pair = one ? i % G1 : (i - S1) % G2;
                const int n = one ? group * NP + Pairs<NP>::first(pair) : F1 + group * NP + Dz::first(pair);
                const int second = one ? Pairs<NP>::second(pair) : Dz::second(pair);
                if (second == 0) {
                    read(n + 2);
                    settle(f[n % 3]);
                }
                if (one) wide_mma(nxt, f[n % 3], q[one ? second : 0][one ? group : 0]);
                else wide_mma(acc[one ? 0 : group % NX], f[n % 3], dz.p[one ? 0 : group / NX][second]);
                const int from = GENERAL ? (2 * i < SLICES ? 0 : (2 * i - SLICES) * UNITS / SLICES) : i * UNITS / SLICES;
                const int to = GENERAL ? (2 * i + 2 < SLICES ? 0 : (2 * i + 2 - SLICES) * UNITS / SLICES) : (i + 1) * UNITS / SLICES;
#pragma unroll
                for (int u = from; u < to; ++u) {
                    if (u < 16) {
                        if (u % 4 == 0 && u > 0) k4 = ahead_k4;
                        if (OWN_BANK && u % 4 == 0 && u < 12) ahead_k4 = quad(coef, u / 4 + 1);
                        z[u] = differentiate(pr, wv, k4, u, t, std::false_type{});
                        settle(z[u]);
                    } else {
                        mine.pair(u - 16, z[2 * (u - 16)], z[2 * (u - 16) + 1]);
                        mine.settle_pair(u - 16);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            pr = nxt;
            dz = mine;
        };
        int t = t0;                                                    // no way out of the loop's middle: it would cost copies of the sums
        for (; t + 4 <= t1; t += 4) {
            step(t, lds3, lds1, lds2, s_coef0, s_coef2);
            step(t + 1, lds0, lds2, lds3, s_coef1, s_coef3);
            step(t + 2, lds1, lds3, lds0, s_coef2, s_coef0);
            step(t + 3, lds2, lds0, lds1, s_coef3, s_coef1);
        }
        if (t < t1) step(t, lds3, lds1, lds2, s_coef0, s_coef2);
        if (t + 1 < t1) step(t + 1, lds0, lds2, lds3, s_coef1, s_coef3);
        if (t + 2 < t1) step(t + 2, lds1, lds3, lds0, s_coef2, s_coef0);
        const int last = (t1 - 1 - t0) & 3;
        second_product<NP, CP>(acc, last == 0 ? lds0 : last == 1 ? lds1 : last == 2 ? lds2 : lds3, dz, lane, false);
    };
    // The targets' share in the bank's gradient: the feature rows of this part whose target is one of the workgroup's owners are listed, in
    // rising order, and multiplied 32 at a time like a tile of their own.
    auto add_targets = [&](bool clean) __attribute__((always_inline)) {
        if (!OWN_BANK) return;
        constexpr int SCAN = 4;                                        // rows a thread looks at in one go
        int listed = 0;
        auto multiply = [&](int n) __attribute__((always_inline)) {    // the first n (at most 32) of the list
            publish_lds();
            if (threadIdx.x < 32) {
                const int r = (int)threadIdx.x < n ? s_list[threadIdx.x] : 0;
                s_target[threadIdx.x] = (int)threadIdx.x < n ? __builtin_bit_cast(int, a.coef[K_TARGET * n_coef + r]) : -1;
                s_share[threadIdx.x] = a.coef[K_LOGP * n_coef + r];
            }
            stager.gather(lds0, a, s_list, n, lane);
            publish_lds();
            const int t = s_target[lane & 31];
            if (__any(t >= own0 && t < own0 + 32)) {
                float z[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int r = 8 * (i >> 2) + 4 * g + (i & 3);
                    const bool mine = s_target[r] == own;
                    z[i] = mine ? s_share[r] : 0.0f;
                    if (GENERAL && w && mine && w[(size_t)s_list[r] * a.ldw] == __builtin_inff()) z[i] = 0.0f;     // left out for that row
                }
                Dz dz;
#pragma unroll
                for (int i = 0; i < 8; ++i) dz.pair(i, z[2 * i], z[2 * i + 1]);
                second_product<NP, CP>(acc, lds0, dz, lane, clean);
            }
        };
        const int first_owner = (int)(blockIdx.x / a.parts) * 128, end = t1 * 32;
#pragma unroll 1
        for (int base = t0 * 32; base < end; base += SCAN * 256) {
            uint64_t found[SCAN];
#pragma unroll
            for (int i = 0; i < SCAN; ++i) {
                const int r = base + i * 256 + (int)threadIdx.x;
                const int t = r < end ? __builtin_bit_cast(int, a.coef[K_TARGET * n_coef + r]) : -1;
                found[i] = __ballot(t >= first_owner && t < first_owner + 128);
            }
            publish_lds();                                             // nobody reads the list or the counts any more
            if (lane == 0)
#pragma unroll
                for (int i = 0; i < SCAN; ++i) s_found[i * 4 + wave] = __builtin_popcountll(found[i]);
            __syncthreads();
            int at[SCAN], total = listed;
#pragma unroll
            for (int i = 0; i < SCAN * 4; ++i) {
                if (i % 4 == wave) at[i / 4] = total;
                total += s_found[i];
            }
#pragma unroll
            for (int i = 0; i < SCAN; ++i)
                if (found[i] >> lane & 1) s_list[at[i] + __builtin_popcountll(found[i] & ((1ull << lane) - 1))] = base + i * 256 + (int)threadIdx.x;
            listed = total;
            const bool last = base + SCAN * 256 >= end;
#pragma unroll 1
            while (listed >= 32 || (last && listed > 0)) {
                multiply(min(listed, 32));
                publish_lds();
                int keep[SCAN];                                        // the rest moves to the front
#pragma unroll
                for (int i = 0; i < SCAN; ++i) keep[i] = s_list[32 + i * 256 + threadIdx.x];
                __syncthreads();
#pragma unroll
                for (int i = 0; i < SCAN; ++i) s_list[i * 256 + threadIdx.x] = keep[i];
                listed = max(listed - 32, 0);
            }
        }
    };
    if constexpr (SIDE_BY_SIDE) pass();
    else plain_pass(std::false_type{});
    add_targets(false);
    bool broken = false;
#pragma unroll
    for (int x = 0; x < NX; ++x)
#pragma unroll
        for (int i = 0; i < 16; ++i) broken |= live && !(__builtin_fabsf(acc[x][i]) <= FLT_MAX);
    if (threadIdx.x == 0) s_again = 0;
    publish_lds();                                                     // also: nobody reads the tiles any more, and no copy is under way
    if (broken) s_again = 1;
    __syncthreads();
    if (s_again) {
        // read again: they need not stay in registers in between (at 256 channels of f32 that made it slower)
        if (NP * CP < 768) own_fragments<NP, CP>(q, a, own0, lane, !GENERAL && a.scale < 0.0f);
        plain_pass(std::true_type{});
        add_targets(true);
    }
    if (!live) return;
    if (!OWN_BANK && part == 0) {
        const int target = __builtin_bit_cast(int, a.coef[K_TARGET * n_coef + own]);
        const float gl = a.coef[K_LOGP * n_coef + own];
        if (target >= 0 && !(GENERAL && w && w[target] == __builtin_inff())) {
            const bf16* row = a.other + (size_t)target * a.ld_other + 4 * g;
            typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
#pragma unroll
            for (int x = 0; x < NX; ++x)
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const int ch = x * 32 + 8 * b;
                    if (ch >= a.channels) continue;
                    bf16x4 v[NP];                                      // rows start on 16 bytes
#pragma unroll
                    for (int n = 0; n < NP; ++n) v[n] = *(const bf16x4*)(row + n * CP + ch);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float sum = 0.0f;
#pragma unroll
                        for (int n = NP - 1; n >= 0; --n) sum += to_f32(v[n][i]);
                        acc[x][4 * b + i] += gl * sum;
                    }
                }
        }
    }
#pragma unroll
    for (int x = 0; x < NX; ++x)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int ch = x * 32 + 8 * b + 4 * g;
            if (a.parts > 1) {
                *(f32x4*)(a.partial + ((size_t)part * a.n_own + own) * CP + ch) =
                    (f32x4){acc[x][4 * b], acc[x][4 * b + 1], acc[x][4 * b + 2], acc[x][4 * b + 3]};
            } else {
                T* at = (T*)a.grad + (size_t)own * a.grad_channels + ch;
                typename Loose<T, 4>::V v;
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = from_f32<T>(a.scale * acc[x][4 * b + i]);
                if (ch + 4 <= a.grad_channels) store_loose<4>(at, v);
                else
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (ch + i < a.grad_channels) at[i] = v[i];
            }
        }
}

template <typename T>
__global__ __launch_bounds__(256) void bank_gradient_join_kernel(BankArgs a, int cp) {
    const uint32_t id = blockIdx.x * 256u + threadIdx.x;               // fewer than 2^24 rows of at most 256 channels
    if (id >= (uint32_t)a.n_own * (uint32_t)a.grad_channels) return;
    const uint32_t row = id / (uint32_t)a.grad_channels, ch = id - row * (uint32_t)a.grad_channels;
    float v = 0.0f;
    for (int s = 0; s < a.parts; ++s) v += a.partial[((size_t)s * a.n_own + row) * cp + ch];
    ((T*)a.grad)[id] = from_f32<T>(a.scale * v);
}


template <typename T, int CP>
static void launch(const BankArgs& a, bool own_bank, hipStream_t st) {
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
        hipLaunchKernelGGL((bank_gradient_join_kernel<T>), dim3((unsigned)(((long)a.n_own * a.grad_channels + 255) / 256)), dim3(256), 0, st, a, CP);
}

template <> void launch_bank_gradient<NEMO_ELEMENT>(const BankArgs& a, bool own_bank, hipStream_t st) {
    switch (padded_channels(a.channels)) {
        case 64: launch<NEMO_ELEMENT, 64>(a, own_bank, st); break;
        case 128: launch<NEMO_ELEMENT, 128>(a, own_bank, st); break;
        default: launch<NEMO_ELEMENT, 256>(a, own_bank, st);
    }
}

}  // namespace nemo
