// The log probabilities of log_probs.hip straight from features and bank, z = scale <feature, bank row> - weight, without ever writing the
// [rows, bank rows] matrix: owners (bank_tiles.h) are the feature rows, others the bank; the softmax state of a row and its best entries live
// in the lane, no exchange until the end.  The bank is split where there are too few feature rows to fill the device; states and lists of the
// parts, and of the two lanes of a row, are joined by a second kernel in a fixed order.  Compiled once for each element type (NEMO_ELEMENT).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/nemo_hip.h"
#include "bank_tiles.h"

namespace nemo {

// Puts z into the list.  Places arrive in rising order, so an equal score goes behind those already there.  A score at least as large as entry
// i - 1 and one between two entries are both the median of the two and z.
template <int TOP>
__device__ inline void insert(float (&tv)[TOP], int (&tp)[TOP], float z, int place) {
    bool above = z > tv[TOP - 1];
#pragma unroll
    for (int i = TOP - 1; i > 0; --i) {
        const bool shift = z > tv[i - 1];
        tp[i] = shift ? tp[i - 1] : above ? place : tp[i];
        tv[i] = __builtin_amdgcn_fmed3f(z, tv[i - 1], tv[i]);
        above = shift;
    }
    tp[0] = above ? place : tp[0];
    tv[0] = fmaxf(z, tv[0]);
}

// NP: pieces of a value (bank_tiles.h).  GENERAL: with weights, with a list (its order is that of the scores), or with hardly any scale; see
// softmax_state.h for the two forms of the state.  The sign of the scale goes into the owners' fragments where the state is kept of the products.
//
// Tiles of 32 bank rows; in step n the wave multiplies tile n + 1 while it takes the products of tile n into the state, so that matrix cores
// and vector units work side by side.  Two tiles in LDS (n + 1, and n + 2 on its way), one barrier a step.
//
// Measured.  32768 x 15976 x 128 bf16: 202 us, 664 TF; the matrix instructions take 101 us, the vector units (10 operations a score, one of them
// the exponential, four times as long) about 160.  10007 x 3678 x 128 f32: 60 us, with weights for every pair 73; the six products of a pair 43.
// 8000 x 13416 x 128 f32 with a list of five: 203 us (the six products 124), with one of 16 350: insertions.  (The matrix instructions for f32 took
// 351 us for the former: see bank_tiles.h.)
template <int NP, int CP, int TOP, bool GENERAL>
__global__ __launch_bounds__(256, NP * CP > 512 ? 1 : 2) void bank_forward_kernel(BankArgs a) {
    typedef Tile<CP> L;
    constexpr int NT = TOP > 0 ? TOP : 1, NKF = CP / kFragK;
    __shared__ __attribute__((aligned(16))) char lds0[NP * L::BYTES];
    __shared__ __attribute__((aligned(16))) char lds1[NP * L::BYTES];
    __shared__ int s_again;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 5;
    const int part = (int)(blockIdx.x % a.parts);
    const int own0 = (int)(blockIdx.x / a.parts) * 128 + wave * 32, row = own0 + (lane & 31);
    const bool live = row < a.n_own;
    u32x4 q[NP][NKF];
    own_fragments<NP, CP>(q, a, own0, lane, !GENERAL && a.scale < 0.0f);
    const float* w = a.weights ? a.weights + (live ? row : 0) * a.ldw : nullptr;
    const long long tl = live ? a.targets[row] : -1;
    const int target = tl >= 0 && tl < a.n_other ? (int)tl : -1;
    const float scale = GENERAL ? a.scale : __builtin_fabsf(a.scale);
    const float k = a.out.k, unit = GENERAL ? kLog2e : 1.0f;
    SoftmaxState st;
    float tv[NT];
    int tp[NT];

    auto load_weights = [&](float (&wv)[16], int tile) __attribute__((always_inline)) {
        if (GENERAL && w) row_weights(wv, w, tile * 32, g, a.n_other);
    };
    // a product, or the score if GENERAL
    auto value = [&](const f32x16_t& pr, const float (&wv)[16], int i) __attribute__((always_inline)) {
        return !GENERAL ? pr[i] : w ? score(pr[i], scale, wv[i]) : score(pr[i], scale);
    };
    auto peak_of = [&](const float (&v)[16]) __attribute__((always_inline)) {
        float peak = v[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) peak = fmaxf(peak, v[i]);
        return peak;
    };
    // adds a value to the state.  SAFE: also right where a difference of two products is beyond the range of f32
    auto add = [&](float v, auto safe_tag) __attribute__((always_inline)) {
        constexpr bool SAFE = decltype(safe_tag)::value || GENERAL;
        const float x = GENERAL ? (v - st.m) * kLog2e : __builtin_fmaf(k, v, -st.m), e = exp2_fast(x);
        st.s += e;
        st.t += e * (SAFE ? fmaxf(x, -200.0f) : x);                    // 0 where e is 0, also where x is -inf
    };
    // what only some tiles have: the target's score, entries for the list
    auto note = [&](const float (&v)[16], int tile) __attribute__((always_inline)) {
        const int j0 = tile * 32;
        if (__any(target >= j0 && target < j0 + 32)) {
            const int at = target - j0 - 4 * g;
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (at == 8 * (i >> 2) + (i & 3)) a.z_target[row] = v[i];
        }
        if (TOP > 0) {
            // nothing below the worst entry of either list of the row belongs to its best
            const float bar = fmaxf(tv[NT - 1], __shfl_xor(tv[NT - 1], 32));
            if (__any(peak_of(v) > bar)) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (__any(v[i] > bar)) insert(tv, tp, v[i] > bar ? v[i] : neg_inf(), j0 + 8 * (i >> 2) + 4 * g + (i & 3));
            }
        }
    };
    const int tiles = (a.n_other + 31) / 32;
    const int t0 = part * a.part_tiles, t1 = min(tiles, t0 + a.part_tiles);
    const Stager<NP, CP> stager(a, wave, lane);
    auto stage = [&](char* lds, int tile) __attribute__((always_inline)) { stager.copy(lds, tile); };
    auto start = [&]() __attribute__((always_inline)) {
        st = empty_state();
#pragma unroll
        for (int i = 0; i < NT; ++i) { tv[i] = neg_inf(); tp[i] = kNoPlace; }
    };
    // tiles from `t` on one step after the other, with every precaution
    auto plain_pass = [&](int t) __attribute__((always_inline)) {
        for (; t < t1; ++t) {
            publish_lds();
            stage(lds0, t);
            float wv[16], v[16];
            load_weights(wv, t);
            publish_lds();
            const f32x16_t pr = products<NP, CP>(lds0, q, lane);
            const int left = a.n_other - t * 32 - 4 * g;               // registers whose row 8 b + i is at least this are beyond the end
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = 8 * (i >> 2) + (i & 3) >= left ? neg_inf() : value(pr, wv, i);
            const float peak = peak_of(v);
            raise(st, fmaxf(st.m, GENERAL ? peak : k * peak), unit);
#pragma unroll
            for (int i = 0; i < 16; ++i) add(v[i], std::true_type{});
            note(v, t);
        }
    };
    start();
    // the last tile of the bank may be cut short: it is left to the plain pass
    const int whole = t1 == tiles && a.n_other % 32 != 0 && t1 > t0 ? t1 - 1 : t1;
    if (t0 < whole) {
        stage(lds0, t0);
        publish_lds();
        f32x16_t pr = products<NP, CP>(lds0, q, lane);
        stage(lds1, t0 + 1);
        // `next` holds tile t + 1; `after` held tile t, whose products are in pr.  A slice: a fragment is read (two slices ahead of its use),
        // multiplied, and a share of the 18 units of tile t is done: the largest product, the state raised to it, 16 products added.  Weights
        // may arrive during the first half of the slices.
        auto step = [&](int t, const char* next, char* after) __attribute__((always_inline)) {
            publish_lds();                                             // tile t + 1 is there; nobody reads tile t any more
            stage(after, t + 2);                                       // also behind the part's last tile, to no effect: no branch
            float wv[16], v[16];
            load_weights(wv, t);
            f32x16_t nxt = {};
            constexpr int UNITS = 18, FRAGS = NKF * NP, SLICES = NKF * Pairs<NP>::N;
            float peak = 0.0f;
            u32x4 f[3];
            auto read = [&](int n) __attribute__((always_inline)) {
                if (n < FRAGS) f[n % 3] = row_fragment<CP>(next + n % NP * L::BYTES, n / NP, lane);
            };
            read(0);
            read(1);
#pragma unroll
            for (int i = 0; i < SLICES; ++i) {
                const int kf = i / Pairs<NP>::N, pair = i % Pairs<NP>::N, n = kf * NP + Pairs<NP>::first(pair);
                if (Pairs<NP>::second(pair) == 0) {
                    read(n + 2);
                    settle(f[n % 3]);
                }
                wide_mma(nxt, f[n % 3], q[Pairs<NP>::second(pair)][kf]);
                const int from = GENERAL ? (2 * i < SLICES ? 0 : (2 * i - SLICES) * UNITS / SLICES) : i * UNITS / SLICES;
                const int to = GENERAL ? (2 * i + 2 < SLICES ? 0 : (2 * i + 2 - SLICES) * UNITS / SLICES) : (i + 1) * UNITS / SLICES;
#pragma unroll
                for (int u = from; u < to; ++u) {
                    if (u == 0) {
#pragma unroll
                        for (int e = 0; e < 16; ++e) v[e] = value(pr, wv, e);
                        peak = peak_of(v);
                        settle(peak);
                    }
                    if (u == 1) {
                        raise(st, fmaxf(st.m, GENERAL ? peak : k * peak), unit);
                        settle(st.m);
                        settle(st.s);
                    }
                    if (u >= 2) {
                        add(v[u - 2], std::false_type{});
                        settle(st.s);
                        settle(st.t);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            note(v, t);
            pr = nxt;
        };
        int t = t0;                                                    // no way out of the loop's middle: it would cost copies of registers
        for (; t + 2 <= whole; t += 2) {
            step(t, lds1, lds0);
            step(t + 1, lds0, lds1);
        }
        if (t < whole) step(t, lds1, lds0);
        wait_for_copies();                                             // of the tiles behind the last one: no wave ends before they are there
    }
    plain_pass(whole);
    if (!GENERAL) {
        // a difference beyond the range, times the 0 that its exponential is, would have spoilt t alone
        if (threadIdx.x == 0) s_again = 0;
        __syncthreads();
        if (st.t != st.t && st.s == st.s) s_again = 1;
        __syncthreads();
        if (s_again) {
            start();
            plain_pass(t0);
        }
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

// A list takes registers and insertions for all the places it has, used or not, so there is a short and a long one.  Measured in us, 1 / 5 best (short),
// 6 / 16 (long): 8000 x 13416 x 128 f32 213 / 203, 324 / 349, bf16 145 / 147, 297 / 341; 10007 x 3678 x 128 f32 97 / 100, 148 / 175; 300 x 1118 x 64
// f32 28 / 28, 28 / 32.
template <int NP, int CP>
static void launch(const BankArgs& a, hipStream_t st) {
    const dim3 grid((unsigned)((a.n_own + 127) / 128 * a.parts));
    const int top = a.out.top;
    if (a.out.k != 0.0f) hipLaunchKernelGGL((bank_forward_kernel<NP, CP, 0, false>), grid, dim3(256), 0, st, a);
    else if (top == 0) hipLaunchKernelGGL((bank_forward_kernel<NP, CP, 0, true>), grid, dim3(256), 0, st, a);
    else if (top <= 5) hipLaunchKernelGGL((bank_forward_kernel<NP, CP, 5, true>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((bank_forward_kernel<NP, CP, 16, true>), grid, dim3(256), 0, st, a);
}

template <> void launch_bank_forward<NEMO_ELEMENT>(const BankArgs& a, hipStream_t st) {
    constexpr int NP = sizeof(NEMO_ELEMENT) == 4 ? 3 : 1;
    switch (padded_channels(a.channels)) {
        case 64: launch<NP, 64>(a, st); break;
        case 128: launch<NP, 128>(a, st); break;
        default: launch<NP, 256>(a, st);
    }
}

}  // namespace nemo
