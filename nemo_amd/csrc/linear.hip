// y = act(alpha x W^T + bias) + beta r and its gradients.
//
// One tiled product serves the forward pass and both weight- and input-gradients.  It computes
//     C[q][p] = sum_k P(p, k) Q(q, k)
// where p, the column of the result that is contiguous in memory, is the FIRST operand of the matrix instruction, so that a lane ends
// up with four consecutive columns of one row.  An operand is "plain" when k is contiguous in
// memory and "transposed" when its row index is:
//     y  = x W^T       p = output channel (W plain),  q = row of x (plain),          k = input channel
//     dx = dz W        p = input channel (W transposed), q = row of dz (plain),      k = output channel
//     dW = dz^T x      p = input channel (x transposed), q = output channel (dz transposed), k = row
//
// Tiles go straight from global memory to LDS (16 bytes a lane, no registers), two buffers, one barrier per 128-byte step of k.  LDS
// rows of a plain operand are 128 bytes = 8 chunks; chunk c of row r lies at position c ^ (r & 7), so that the 16-byte reads of a
// fragment (same c, consecutive rows) touch all banks.  A transposed operand lies in LDS as it does in memory (rows of k); 16-bit
// fragments are read with the transposing LDS read, 32 bytes of a row at a time, and those 32-byte pieces are spread over the banks by
// an exclusive-or with the k row.
//
// The copies to LDS need operands that start on 16 bytes, with rows that do and a contiguous extent of whole 16 bytes; others are first copied into
// the workspace with padded rows (pack_kernel).  Bias, residual and results may start at any element.
//
// Measured (a call).  8192 x 4096 x 4096 bf16 with gelu, bias and residual: 261 us, 1053 TF; the bare product of a library 207 us, 1326 TF.
// 160000 x 128 x 2048 bf16 with relu and bias (696 MB): 188 us, 3.7 TB/s.  5590 x 15976 x 128 f32 with a residual: 267 us, 86 TF and 2.7 TB/s:
// the f32 matrix instructions alone take 149 us, reading and writing the 714 MB alone 150, and little of the two overlaps.
// 8191 x 1001 x 515 f16, rows off 16 bytes, silu, bias, residual: packing 6, product 31 us; backward: packing 6, slope 20, column sums 4,
// products 23 and 20 + 6 (join).
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <algorithm>
#include <type_traits>

#include "../../include/nemo_hip.h"
#include "dense.h"
#include "errors.h"

namespace nemo {

__device__ const u32x4 g_zero_chunk = {0, 0, 0, 0};                    // what the lanes beyond the end of k copy

enum { ACT_NONE = 0, ACT_RELU = 1, ACT_GELU = 2, ACT_SILU = 3 };

// erfc(a), a >= 0, to 1.5e-7: the rational approximation 7.1.26 of Abramowitz and Stegun, a quarter of erff's instructions.  For the 16-bit types, whose
// own rounding is 2^-11 at best; f32 takes erff.
__device__ inline float erfc_short(float a) {
    const float t = __builtin_amdgcn_rcpf(1.0f + 0.3275911f * a);
    const float p = t * (0.254829592f + t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f))));
    return p * __builtin_amdgcn_exp2f(-1.44269504088896341f * a * a);
}
// Standard normal distribution function at z.
template <typename T> __device__ inline float normal_cdf(float z) {
    if constexpr (sizeof(T) == 4) return 0.5f * (1.0f + erff(z * 0.70710678118654752f));
    const float half = 0.5f * erfc_short(__builtin_fabsf(z) * 0.70710678118654752f);
    return z < 0.0f ? half : 1.0f - half;
}
template <typename T> __device__ inline float logistic(float z) {
    if constexpr (sizeof(T) == 4) return 1.0f / (1.0f + expf(-z));
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504088896341f * z));
}

template <typename T> __device__ inline float activate(float z, int act) {
    switch (act) {
        case ACT_RELU: return z > 0.0f ? z : (z != z ? z : 0.0f);
        case ACT_GELU: return z * normal_cdf<T>(z);
        case ACT_SILU: return z * logistic<T>(z);
        default: return z;
    }
}

// d act / d z.  relu's slope at 0 is 0.  Far out gelu's exp(-z^2 / 2) and silu's s underflow to 0; 1 - s is taken as the function of -z.
template <typename T> __device__ inline float activate_slope(float z, int act) {
    switch (act) {
        case ACT_RELU: return z > 0.0f ? 1.0f : (z != z ? z : 0.0f);
        case ACT_GELU: return normal_cdf<T>(z) + z * __builtin_amdgcn_exp2f(-0.72134752044448170f * z * z) * 0.39894228040143268f;
        case ACT_SILU: return logistic<T>(z) * (1.0f + z * logistic<T>(-z));
        default: return 1.0f;
    }
}

struct Epilogue {
    float alpha, beta;
    int act;
    const void* bias;          // [np] or null
    const void* residual;      // [nq][ldr] or null
    long ldr;
    void* out;                 // [nq][ldo]
    long ldo;
    void* pre;                 // [nq][ldo]: alpha acc + bias, or null
};

struct GemmArgs {
    const void* P;
    const void* Q;
    long ldp, ldq;             // elements
    int np, nq, nk;
    int bp, bq, tiles_p, tiles_q, splits, k_split; // sides of a tile; k of one split, whole steps
    float* partial;            // [splits][nq][np4] when splits > 1
    int np4;
    Epilogue e;
};

// The stored pre-activation: rounds to T so that the slopes stay those of the value before rounding.  A finite value beyond T's largest is kept as
// that one (an infinity would make the slopes of gelu and silu 0 x infinity; out there they are 0 and 1), and one that f16 rounds to zero keeps
// its sign as the smallest subnormal (relu).
template <typename T> __device__ inline T round_pre(float z) {
    if constexpr (sizeof(T) == 4) return z;
    constexpr bool F16 = std::is_same<T, f16>::value;
    constexpr float most = F16 ? 65504.0f : 3.3895313892515355e38f;
    const float cut = __builtin_amdgcn_fmed3f(z, -most, most);
    const T h = (T)(__builtin_fabsf(z) <= __FLT_MAX__ ? cut : z);
    if (F16 && h == (T)0.0f && z != 0.0f) return z > 0.0f ? (T)5.9604644775390625e-8f : (T)-5.9604644775390625e-8f;
    return h;
}

template <typename T, int N> __device__ inline void activate_all(float (&v)[N], int act) {
    if (act == ACT_NONE) return;
    if (act == ACT_RELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = activate<T>(v[i], ACT_RELU);
    } else if (act == ACT_GELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = activate<T>(v[i], ACT_GELU);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = activate<T>(v[i], ACT_SILU);
    }
}

// Up to N consecutive columns from p on of row q, those below np.
template <typename T, int N>
__device__ inline void epilogue_tail(const Epilogue& e, const float (&acc)[N], int q, int p, int np) {
    float v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = p + i < np && e.bias ? e.alpha * acc[i] + to_f32(((const T*)e.bias)[p + i]) : e.alpha * acc[i];
    if (e.pre) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (p + i < np) ((T*)e.pre)[(size_t)q * e.ldo + p + i] = round_pre<T>(v[i]);
    }
    activate_all<T, N>(v, e.act);
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (p + i < np) {
            const float r = e.residual ? v[i] + e.beta * to_f32(((const T*)e.residual)[(size_t)q * e.ldr + p + i]) : v[i];
            ((T*)e.out)[(size_t)q * e.ldo + p + i] = from_f32<T>(r);
        }
}

// Exclusive-or of the 16-byte chunk index of k row `k` in a transposed 16-bit tile: the 16 rows that one fragment read touches (8 g + 0..3
// or 8 g + 4..7) get different pairs of chunks as far as the row has them.
template <int CPR> __device__ inline int swizzle_t(int k) { return (2 * (((k >> 3) & 3) * 4 + (k & 3))) & (CPR - 1); }

template <typename T> constexpr int kstep() { return 128 / (int)sizeof(T); }

// What a lane copies of every tile of ROWS rows x 128 bytes of k, WAVES waves sharing the work: 32-bit offsets from an address that all lanes share and
// that moves on from tile to tile.  Rows beyond the last are replaced by the last one (their results are not stored).
template <typename T, int ROWS, bool TR, int WAVES> struct Copier {
    static constexpr int EPC = 16 / (int)sizeof(T), N = ROWS * 8 / 64 / WAVES, BK = kstep<T>();
    static_assert(N * 64 * WAVES == ROWS * 8, "every wave copies the same number of kilobytes");
    const char* base;                      // of the tile's first row (TR: first column), k = 0
    long step;                             // bytes from tile to tile
    uint32_t off[N];
    int wave, lane;
    // k of copy i within the tile
    __device__ inline int k_of(int i) const {
        const int idx = (i * WAVES + wave) * 64 + lane, r = idx >> 3;
        return TR ? idx / (ROWS / EPC) : ((idx & 7) ^ (r & 7)) * EPC;
    }
    __device__ inline Copier(const void* m, long ld, int row0, int rows, int wave_, int lane_) : wave(wave_), lane(lane_) {
        base = (const char*)m + (TR ? (long)row0 : (long)row0 * ld) * (long)sizeof(T);
        step = (TR ? BK * ld : BK) * (long)sizeof(T);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int idx = (i * WAVES + wave) * 64 + lane;
            if (!TR) {
                const int r = idx >> 3, c = (idx & 7) ^ (r & 7);
                off[i] = (uint32_t)(min(r, rows - 1 - row0) * (int)ld + c * EPC) * (uint32_t)sizeof(T);
            } else {
                constexpr int CPR = ROWS / EPC;
                const int kr = idx / CPR, c = (idx & (CPR - 1)) ^ (sizeof(T) == 2 ? swizzle_t<CPR>(kr) : 0);
                off[i] = (uint32_t)(kr * (int)ld + min(c * EPC, (rows - 1 - row0) / EPC * EPC)) * (uint32_t)sizeof(T);
            }
        }
    }
    // Tile number t.
    __device__ inline void copy(char* lds, int t) const {
        const char* tile = base + (long)t * step;
#pragma unroll
        for (int i = 0; i < N; ++i) copy_to_lds(tile + off[i], lds + (i * WAVES + wave) * 1024);
    }
    // Tile number t, of which k below `left` exists; the rest is zero.
    __device__ inline void copy_part(char* lds, int t, int left) const {
        const char* tile = base + (long)t * step;
#pragma unroll
        for (int i = 0; i < N; ++i)
            copy_to_lds(k_of(i) < left ? (const void*)(tile + off[i]) : (const void*)&g_zero_chunk, lds + (i * WAVES + wave) * 1024);
    }
};

// Fragment kf (of the tile's 128 bytes of k) of the FR rows that start at `row`.
template <typename T, int ROWS, bool TR>
__device__ inline u32x4 fragment(const char* lds, int row, int kf, int lane) {
    constexpr int FR = Mma<T>::FR, NG = Mma<T>::NG;
    const int r = row + (lane & (FR - 1)), g = lane / FR;
    if constexpr (!TR) {
        const int c = kf * NG + g;
        return *(const u32x4*)(lds + r * 128 + ((c ^ (r & 7)) << 4));
    } else if constexpr (sizeof(T) == 4) {
        u32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = *(const uint32_t*)(lds + ((kf * 8 + 4 * g + i) * ROWS + r) * 4);
        return v;
    } else {
        constexpr int CPR = ROWS / 8;
        // lane i of a group of 16 supplies the address of columns 4 (i % 4) .. + 3 of k row i / 4 and receives column i of the four rows
        const int i = lane & 15, k = kf * 32 + 8 * g + (i >> 2);
        const int col = row + 4 * (i & 3);
        const int s = swizzle_t<CPR>(k);                               // the same for k + 4
        const char* at = lds + k * (ROWS * 2) + ((((col >> 3) ^ s) << 4) | ((col & 7) << 1));
        union { i16x4 h[2]; u32x4 v; } u;
        u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((NEMO_LDS i16x4*)at);
        u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((NEMO_LDS i16x4*)(at + 4 * (ROWS * 2)));
        return u.v;
    }
}

// The tile of a step is multiplied in two halves of its k.  Both halves' fragments are in registers before the barrier that frees the tile's
// buffer; behind it, while the second half is multiplied, the tile after the next one is copied into that buffer and the first half of the
// next tile is read.  So the matrix cores have work across the barrier, and a copy could have a whole step to arrive.  As compiled it has that in
// every other step only: the compiler does not tell the two buffers apart.  In the 16-bit forms it waits for the copies just made before it
// reads the other buffer; in the f32 forms it moves them down to the next barrier, which waits for them.
template <typename T, int BP, int BQ, int WP, int WQ, bool PT, bool QT>
__global__ __launch_bounds__(64 * WP * WQ, BP == 256 ? 1 : BQ == 128 ? 2 : BQ == 64 ? 3 : 4) void gemm_kernel(GemmArgs a) {
    typedef Mma<T> M;
    constexpr int WAVES = WP * WQ, TP = BP / WP, TQ = BQ / WQ, NP = TP / M::FR, NQ = TQ / M::FR;
    constexpr int BK = kstep<T>(), HALF = BK / M::KF / 2;               // fragments of k in half a tile
    __shared__ __attribute__((aligned(16))) char lds0[(BP + BQ) * 128];
    __shared__ __attribute__((aligned(16))) char lds1[(BP + BQ) * 128];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wp = wave % WP, wq = wave / WP;

    // Workgroups are dealt to the eight XCDs in turn; renumbered so that an XCD gets consecutive tiles, and tiles run through eight
    // rows of q tiles before the next p tile, so that the XCD's L2 holds what its workgroups share.
    const int per_split = a.tiles_p * a.tiles_q, total = per_split * a.splits;
    int id = blockIdx.x;
    {
        const int x = id & 7, w = id >> 3, base = total >> 3, rest = total & 7;
        id = x * base + min(x, rest) + w;
    }
    const int split = id / per_split;
    id -= split * per_split;
    constexpr int GROUP = 8;
    const int group = id / (GROUP * a.tiles_p), first = group * GROUP, size = min(a.tiles_q - first, GROUP);
    const int in = id - group * GROUP * a.tiles_p;
    const int q0 = (first + in % size) * BQ, p0 = (in / size) * BP;

    const int k_begin = split * a.k_split, k_end = min(a.nk, k_begin + a.k_split), nt = (k_end - k_begin + BK - 1) / BK;
    typename M::Acc acc[NP][NQ];
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
        for (int j = 0; j < NQ; ++j) acc[i][j] = {};

    if (nt > 0) {
        const Copier<T, BP, PT, WAVES> cp(a.P, a.ldp, p0, a.np, wave, lane);
        const Copier<T, BQ, QT, WAVES> cq(a.Q, a.ldq, q0, a.nq, wave, lane);
        const int t0 = k_begin / BK;
        const int full = (k_end - k_begin) / BK;                       // tiles that are not cut short
        auto load = [&](char* lds, int t) __attribute__((always_inline)) {
            cp.copy(lds, t0 + t);
            cq.copy(lds + BP * 128, t0 + t);
        };
        auto load_any = [&](char* lds, int t) __attribute__((always_inline)) {
            if (t < full) {
                load(lds, t);
            } else if (t < nt) {
                cp.copy_part(lds, t0 + t, k_end - k_begin - t * BK);
                cq.copy_part(lds + BP * 128, t0 + t, k_end - k_begin - t * BK);
            }
        };
        u32x4 pf[2][HALF][NP], qf[2][HALF][NQ];
        // Fragment n of the HALF (NP + NQ) of half h.
        auto read = [&](const char* lds, int h, int n) __attribute__((always_inline)) {
            const int f = n / (NP + NQ), i = n % (NP + NQ);
            if (i < NP) pf[h][f][i < NP ? i : 0] = fragment<T, BP, PT>(lds, wp * TP + i * M::FR, h * HALF + f, lane);
            else qf[h][f][i < NP ? 0 : i - NP] = fragment<T, BQ, QT>(lds + BP * 128, wq * TQ + (i - NP) * M::FR, h * HALF + f, lane);
        };
        // Multiplies half h and, in between, reads half o of the tile in `lds`: a few fragments beside each row of products.
        auto multiply = [&](int h, const char* lds, int o) __attribute__((always_inline)) {
            constexpr int ROWS = HALF * NP, FRAGS = HALF * (NP + NQ);
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
#pragma unroll
                for (int n = r * FRAGS / ROWS; n < (r + 1) * FRAGS / ROWS; ++n) read(lds, o, n);
#pragma unroll
                for (int j = 0; j < NQ; ++j) M::run(acc[r % NP][j], pf[h][r / NP][r % NP], qf[h][r / NP][j]);
                if (sizeof(T) == 2) __builtin_amdgcn_sched_barrier(0);
            }
        };
        auto step = [&](char* here, const char* next, int t, auto any_tag) __attribute__((always_inline)) {
            multiply(0, here, 1);
            publish_lds();                                             // the next tile is there, nobody reads this one any more
            if constexpr (decltype(any_tag)::value) load_any(here, t + 2);
            else load(here, t + 2);
            multiply(1, next, 0);                                      // behind the last tile what is read is of no use, and none is made of it
        };
        load_any(lds0, 0);
        publish_lds();
        load_any(lds1, 1);
#pragma unroll
        for (int n = 0; n < HALF * (NP + NQ); ++n) read(lds0, 0, n);
        int t = 0;
        for (; t + 3 < full; t += 2) {                                 // straight code: no tile that is cut short, none missing
            step(lds0, lds1, t, std::false_type{});
            step(lds1, lds0, t + 1, std::false_type{});
        }
        for (; t < nt; t += 2) {
            step(lds0, lds1, t, std::true_type{});
            if (t + 1 < nt) step(lds1, lds0, t + 1, std::true_type{});
        }
    }

    // Through LDS into rows: a wave writes its results there (f32, in the buffers that held the tiles) and takes them back E consecutive columns
    // a lane, so that a row goes to memory in one piece, whatever its start, and the code that finishes a value stands here once.  Chunk c
    // (16 bytes) of row r lies at c ^ (r & FLIP).
    constexpr int FLIP = TP / 4 < 16 ? TP / 4 - 1 : 15;
    constexpr int E = 16 / (int)sizeof(T), REGION = (BP + BQ) * 256 / WAVES, ROWS = REGION / (TP * 4), PASSES = TQ / ROWS > 0 ? TQ / ROWS : 1;
    constexpr int FRAGS = NQ / PASSES, LANES = TP / E, ITERS = FRAGS * M::FR * LANES / 64, BATCH = ITERS < 4 ? ITERS : 4;
    static_assert(FRAGS * M::FR * TP * 4 <= REGION && ITERS % BATCH == 0, "a pass fits the wave's share of LDS");
    char* region = (wave < WAVES / 2 ? lds0 : lds1) + wave % (WAVES / 2) * REGION;
    const T* bias = (const T*)a.e.bias;
    const T* res = (const T*)a.e.residual;
    const int c0 = lane % LANES * E, p = p0 + wp * TP + c0, whole = p + E <= a.np;
    typename Loose<T, E>::V bv = {};
    if (bias && whole) bv = load_loose<E>(bias + p);
#pragma unroll
    for (int pass = 0; pass < PASSES; ++pass) {
        __syncthreads();                                               // nobody reads the tiles, or the pass before, any more
#pragma unroll
        for (int j = 0; j < FRAGS; ++j)
#pragma unroll
            for (int i = 0; i < NP; ++i)
#pragma unroll
                for (int b = 0; b < M::QUADS; ++b) {
                    const typename M::Acc& v = acc[i][pass * FRAGS + j];
                    const int r = j * M::FR + (lane & (M::FR - 1)), c = (i * M::FR + b * 8 + 4 * (lane / M::FR)) / 4;
                    *(f32x4*)(region + r * (TP * 4) + ((c ^ (r & FLIP)) << 4)) = (f32x4){v[4 * b], v[4 * b + 1], v[4 * b + 2], v[4 * b + 3]};
                }
        __syncthreads();
#pragma unroll 1
        for (int it = 0; it < ITERS; it += BATCH) {
            typename Loose<T, E>::V rv[BATCH] = {};
            if (res && whole) {
#pragma unroll
                for (int n = 0; n < BATCH; ++n) {
                    const int q = min(q0 + wq * TQ + pass * FRAGS * M::FR + ((it + n) * 64 + lane) / LANES, a.nq - 1);
                    rv[n] = load_loose<E>(res + (size_t)q * a.e.ldr + p);
                }
            }
#pragma unroll
            for (int n = 0; n < BATCH; ++n) {
                const int r = ((it + n) * 64 + lane) / LANES, q = q0 + wq * TQ + pass * FRAGS * M::FR + r;
                float v[E];
#pragma unroll
                for (int k = 0; k < E / 4; ++k) {
                    const f32x4 t = *(const f32x4*)(region + r * (TP * 4) + (((c0 / 4 + k) ^ (r & FLIP)) << 4));
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[4 * k + i] = t[i];
                }
                if (q >= a.nq || p >= a.np) continue;
                if (a.splits > 1) {
#pragma unroll
                    for (int k = 0; k < E / 4; ++k)
                        if (p + 4 * k < a.np)
                            *(f32x4*)(a.partial + ((size_t)split * a.nq + q) * a.np4 + p + 4 * k) = (f32x4){v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]};
                    continue;
                }
                if (!whole) {
                    epilogue_tail<T>(a.e, v, q, p, a.np);
                    continue;
                }
                const size_t at = (size_t)q * a.e.ldo + p;
                typename Loose<T, E>::V t;
#pragma unroll
                for (int i = 0; i < E; ++i) v[i] = a.e.alpha * v[i] + to_f32(bv[i]);
                if (a.e.pre) {
#pragma unroll
                    for (int i = 0; i < E; ++i) t[i] = round_pre<T>(v[i]);
                    store_loose<E>((T*)a.e.pre + at, t);
                }
                activate_all<T, E>(v, a.e.act);
#pragma unroll
                for (int i = 0; i < E; ++i) t[i] = from_f32<T>(res ? v[i] + a.e.beta * to_f32(rv[n][i]) : v[i]);
                store_loose<E>((T*)a.e.out + at, t);
            }
        }
    }
}

// Sums the splits in their order and applies the epilogue; four columns a thread.
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(GemmArgs a) {
    const uint32_t quads = a.np4 >> 2, id = blockIdx.x * 256u + threadIdx.x;       // splits are of less than 256 tiles
    if (id >= quads * (uint32_t)a.nq) return;
    const uint32_t row = id / quads;
    const int q = (int)row, p = 4 * (int)(id - row * quads);
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int s = 0; s < a.splits; ++s) {
        const f32x4 t = *(const f32x4*)(a.partial + ((size_t)s * a.nq + q) * a.np4 + p);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += t[i];
    }
    epilogue_tail<T>(a.e, v, q, p, a.np);
}

// Copies with padded rows of one or two matrices: rows x cols (row stride ld, any start) -> rows x ld_out on 16 bytes, the columns beyond cols
// zero; 16 bytes of the copy a thread.  The first `groups` workgroups take the first matrix.
struct PackJob { const void* src; long ld; uint32_t rows; int cols; void* dst; int ld_out; };
template <typename T>
__global__ __launch_bounds__(256) void pack_kernel(PackJob first, PackJob second, uint32_t groups) {
    constexpr int E = 16 / (int)sizeof(T);
    const bool other = blockIdx.x >= groups;
    const PackJob j = other ? second : first;
    const uint32_t per_row = j.ld_out / E;
    const uint32_t id = (blockIdx.x - (other ? groups : 0)) * 256u + threadIdx.x;
    const uint32_t r = id / per_row;
    if (r >= j.rows) return;
    const int c = (int)(id - r * per_row) * E;
    const T* s = (const T*)j.src + (long)r * j.ld + c;
    typename Loose<T, E>::V v = {};
    if (c + E <= j.cols) {
        v = load_loose<E>(s);
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (c + i < j.cols) v[i] = s[i];
    }
    *(typename Loose<T, E>::V*)((T*)j.dst + (long)r * j.ld_out + c) = v;
}

// dz = dy act'(pre), dr = beta dy, and per block of rows the column sums of the unrounded dz (for the bias).  dz is rounded to T because the matrix
// cores take T (a second piece would double both products), and pre is kept in T because it is a result's worth of memory between the two
// passes: 8191 x 1001 x 515 f16 with silu, gradients of x and weight off by 3.0e-4 of their norm, 2.1e-4 with both in f32 (the result's own
// rounding).  A workgroup takes 256 columns x kSlopeRows rows: 32 threads of eight columns, eight rows at a time.  Bound by the latency of
// its loads: 8191 x 1001 f16 (49 MB) 20 us with 32 rows a workgroup, 25 with 64; 18 where rows start on 16 bytes.
constexpr int kSlopeRows = 32;
template <typename T>
__global__ __launch_bounds__(256) void slope_kernel(const T* dy, long ldg, const T* pre, long ldpre, long m, int n, int act, float beta,
                                                    T* dz, int ldz, T* dr, float* col_partial, int np4) {
    typedef typename Loose<T, 8>::V T8;
    const int c = blockIdx.x * 256 + (threadIdx.x & 31) * 8, ry = threadIdx.x >> 5;
    const long r0 = (long)blockIdx.y * kSlopeRows;
    const long r1 = r0 + kSlopeRows < m ? r0 + kSlopeRows : m;
    float sum[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if (c + 8 <= n) {
#pragma unroll 4
        for (long r = r0 + ry; r < r1; r += 8) {
            const T8 g = load_loose<8>(dy + r * ldg + c);
            T8 p = {}, d;
            if (act != ACT_NONE) p = load_loose<8>(pre + r * ldpre + c);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x = act == ACT_NONE ? to_f32(g[i]) : to_f32(g[i]) * activate_slope<T>(to_f32(p[i]), act);
                sum[i] += x;
                d[i] = from_f32<T>(x);
            }
            if (dz) store_loose<8>(dz + r * (long)ldz + c, d);
            if (dr) {
                T8 t;
#pragma unroll
                for (int i = 0; i < 8; ++i) t[i] = from_f32<T>(beta * to_f32(g[i]));
                store_loose<8>(dr + r * (long)n + c, t);
            }
        }
    } else if (c < (dz ? ldz : n)) {
        for (long r = r0 + ry; r < r1; r += 8) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (c + i < n) {
                    const float g = to_f32(dy[r * ldg + c + i]);
                    const float x = act == ACT_NONE ? g : g * activate_slope<T>(to_f32(pre[r * ldpre + c + i]), act);
                    sum[i] += x;
                    if (dz) dz[r * (long)ldz + c + i] = from_f32<T>(x);
                    if (dr) dr[r * (long)n + c + i] = from_f32<T>(beta * g);
                } else if (dz && c + i < ldz) {
                    dz[r * (long)ldz + c + i] = (T)0.0f;
                }
            }
        }
    }
    if (!col_partial) return;
    __shared__ float s[8][256 + 8];
#pragma unroll
    for (int i = 0; i < 8; ++i) s[ry][(threadIdx.x & 31) * 8 + i] = sum[i];
    __syncthreads();
    const int col = blockIdx.x * 256 + threadIdx.x;
    if (col < np4) {
        float t = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) t += s[i][threadIdx.x];
        col_partial[(size_t)blockIdx.y * np4 + col] = t;
    }
}

template <typename T>
__global__ __launch_bounds__(256) void column_sum_kernel(const float* partial, int blocks, int np4, int n, T* out) {
    // 32 columns a workgroup, eight threads each
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), part = threadIdx.x >> 5;
    float t = 0.0f;
    if (c < n)
#pragma unroll 4
        for (int b = part; b < blocks; b += 8) t += partial[(size_t)b * np4 + c];
    __shared__ float s[8][32];
    s[part][threadIdx.x & 31] = t;
    __syncthreads();
    if (part == 0 && c < n) {
        for (int i = 1; i < 8; ++i) t += s[i][threadIdx.x];
        out[c] = from_f32<T>(t);
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------
static int elem_size(int dtype) { return dtype == NEMO_F32 ? 4 : 2; }
static int pad16(int64_t n, int es) { return (int)((n * es + 15) / 16 * 16 / es); }
static size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

static bool ready(const void* p, int64_t ld, int64_t cols, int es) {
    return ((uintptr_t)p & 15) == 0 && (ld * es) % 16 == 0 && (cols * es) % 16 == 0;
}

// Tiles of 256 x 256 (16-bit types, both operands plain, eight waves) where there are enough of them for every compute unit; else four waves on
// 128 columns x 128, 64 or 32 rows: fewer rows where there are no more, or where that gives no more than three tiles a unit and the sum is too
// short to be split (up to 32 steps).  The addresses of transposed fragments take too many registers for the largest tile.  Measured in us (128 x 128 /
// 128 x 64 / 128 x 32; f32 from a trace, 16-bit types a call within a graph):
//     both transposed (a weight's gradient), f16, 512 x 1000 x 8192, split: 26 / 26 / 27
//     f32   20 x 3678 x 128    15.5 / 11.0 /  7.4        bf16  20 x 3678 x 128      6.2 /  5.6 /  4.5
//           1000 x 1000 x 1000 39.4 / 34.8 / 26.6              1000 x 1000 x 1000  20.3 / 20.2 / 10.5
//           2000 x 2000 x 2048  145 /  140 /  145              2000 x 2000 x 2048  30.7 / 27.0 / 37.3
//           8192 x 1024 x 2048  262 /  269 /  281              8192 x 1024 x 2048  41.1 / 51.6 / 62.4
//     and 8192 x 4096 x 4096 bf16 228 with 256 x 256, 271 with 128 x 128.  f32 sums over at most 256 k leave so little to multiply in a tile
//     that three workgroups a unit hide more of its ends (128 / 64 rows): 5590 x 15976 x 128 239 / 224, with a residual 300 / 280, 20000 x 2048 x 64
//     74 / 68, 8192 x 8192 x 64 117 / 109, x 128 181 / 169, x 200 279 / 265, x 256 297 / 289, 30000 x 1000 x 256 with a residual 165 / 146; beyond that
//     it fades (8192 x 8192 x 512 541 / 537) and turns (8192 x 1024 x 2048 above).
// Splits of k for a product with too few tiles to fill 256 compute units: as many as bring it to about two workgroups each, of at least four
// steps of k.  Measured in us, f32 (bf16), unsplit / two steps / four / eight: 1 x 4096 x 4096 93 / 19.6 / 19.4 / 19.5 (33 / 8.8 / 8.7 / 9.5),
// 256 x 256 x 4096 265 / 25.8 / 22.9 / 27.1 (37 / 14.0 / 11.8 / 12.0), 700 x 700 x 2100 154 / 41 / 40 / 53 (43 / 26 / 25 / 24); aiming at one or
// four workgroups a unit: 38.7 / 40.4 for the last, 83 / 90 against 83 for 1000 x 500 x 8000.
struct Shape { int bp, bq, tiles_p, tiles_q, splits, k_split; };
static Shape shape_of(int64_t np, int64_t nq, int64_t nk, int dtype, bool transposed) {
    Shape s;
    const int step = 128 / elem_size(dtype);
    const bool big = dtype != NEMO_F32 && !transposed && np > 192 && nq > 192 && ((np + 255) / 256) * ((nq + 255) / 256) >= 240;
    s.bp = big ? 256 : 128;
    s.tiles_p = (int)((np + s.bp - 1) / s.bp);
    const int64_t steps = (nk + step - 1) / step;
    auto few = [&](int bq) { return nq <= bq || (steps <= 32 && s.tiles_p * ((nq + bq - 1) / bq) <= 3 * 256); };
    s.bq = big ? 256 : few(32) ? 32 : few(64) || (dtype == NEMO_F32 && nk <= 256) ? 64 : 128;
    s.tiles_q = (int)((nq + s.bq - 1) / s.bq);
    const int64_t tiles = (int64_t)s.tiles_p * s.tiles_q;
    int64_t want = tiles >= 256 || big ? 1 : 512 / tiles;
    if (want > steps / 4) want = steps / 4;
    if (want < 1) want = 1;
    const int64_t per = steps > 0 ? (steps + want - 1) / want : 1;
    s.splits = steps > 0 ? (int)((steps + per - 1) / per) : 1;
    s.k_split = (int)(per * step);
    return s;
}
static size_t partial_bytes(int64_t np, int64_t nq, const Shape& s) {
    return s.splits > 1 ? align256((size_t)s.splits * nq * (((size_t)np + 3) / 4 * 4) * 4) : 0;
}

template <typename T, bool PT, bool QT>
static void launch_gemm_typed(const GemmArgs& a, hipStream_t st) {
    const long wgs = (long)a.tiles_p * a.tiles_q * a.splits;
    if (a.bp == 256) {
        if constexpr (sizeof(T) == 2 && !PT) hipLaunchKernelGGL((gemm_kernel<T, 256, 256, 2, 4, PT, QT>), dim3((unsigned)wgs), dim3(512), 0, st, a);
    } else if (a.bq == 128) {
        hipLaunchKernelGGL((gemm_kernel<T, 128, 128, 2, 2, PT, QT>), dim3((unsigned)wgs), dim3(256), 0, st, a);
    } else if (a.bq == 64) {
        hipLaunchKernelGGL((gemm_kernel<T, 128, 64, 2, 2, PT, QT>), dim3((unsigned)wgs), dim3(256), 0, st, a);
    } else {
        hipLaunchKernelGGL((gemm_kernel<T, 128, 32, 4, 1, PT, QT>), dim3((unsigned)wgs), dim3(256), 0, st, a);
    }
    if (a.splits > 1) {
        const long threads = (long)(a.np4 / 4) * a.nq;
        hipLaunchKernelGGL((join_kernel<T>), dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, st, a);
    }
}

template <typename T>
static void launch_gemm(const GemmArgs& a, bool pt, bool qt, hipStream_t st) {
    if (!pt && !qt) launch_gemm_typed<T, false, false>(a, st);
    else if (pt && !qt) launch_gemm_typed<T, true, false>(a, st);
    else launch_gemm_typed<T, true, true>(a, st);
}

static void launch_gemm(int dtype, const GemmArgs& a, bool pt, bool qt, hipStream_t st) {
    if (dtype == NEMO_F32) launch_gemm<float>(a, pt, qt, st);
    else if (dtype == NEMO_BF16) launch_gemm<bf16>(a, pt, qt, st);
    else launch_gemm<f16>(a, pt, qt, st);
}

template <typename T>
static void launch_pack(const PackJob* jobs, int n, hipStream_t st) {
    int64_t groups[2] = {0, 0};
    for (int i = 0; i < n; ++i) groups[i] = ((int64_t)jobs[i].rows * (jobs[i].ld_out / (16 / (int)sizeof(T))) + 255) / 256;
    if (groups[0] + groups[1] <= 1 << 23) {
        hipLaunchKernelGGL((pack_kernel<T>), dim3((unsigned)(groups[0] + groups[1])), dim3(256), 0, st, jobs[0], jobs[n - 1], (uint32_t)groups[0]);
        return;
    }
    for (int i = 0; i < n; ++i) {                                      // a launch holds 2^32 threads: in slices of rows
        const int64_t slice = (1LL << 31) / (jobs[i].ld_out / (16 / (int)sizeof(T)));
        for (int64_t r = 0; r < jobs[i].rows; r += slice) {
            PackJob j = jobs[i];
            j.rows = (uint32_t)std::min<int64_t>(slice, jobs[i].rows - r);
            j.src = (const T*)j.src + r * j.ld;
            j.dst = (T*)j.dst + r * j.ld_out;
            const unsigned wgs = (unsigned)(((int64_t)j.rows * (j.ld_out / (16 / (int)sizeof(T))) + 255) / 256);
            hipLaunchKernelGGL((pack_kernel<T>), dim3(wgs), dim3(256), 0, st, j, j, wgs);
        }
    }
}

// Operands as the tiles want them: where they lie, or packed copies taken from the workspace, made in one launch.
struct Operand { const void* p; int64_t ld; };
struct Packer {
    int dtype, n = 0;
    PackJob jobs[2];
    Operand operand(const void* p, int64_t ld, int64_t rows, int64_t cols, char*& ws) {
        const int es = elem_size(dtype);
        if (rows == 0 || ready(p, ld, cols, es)) return {p, ld};
        const int ld_out = pad16(cols, es);
        void* dst = ws;
        ws += align256((size_t)rows * ld_out * es);
        jobs[n++] = {p, (long)ld, (uint32_t)rows, (int)cols, dst, ld_out};
        return {dst, ld_out};
    }
    void launch(hipStream_t st) const {
        if (n == 0) return;
        if (dtype == NEMO_F32) launch_pack<float>(jobs, n, st);
        else launch_pack<bf16>(jobs, n, st);                           // bits of either 16-bit type
    }
};

static GemmArgs gemm_args(Operand P, Operand Q, int64_t np, int64_t nq, int64_t nk, const Shape& s, void* partial) {
    GemmArgs a = {};
    a.P = P.p; a.Q = Q.p; a.ldp = P.ld; a.ldq = Q.ld;
    a.np = (int)np; a.nq = (int)nq; a.nk = (int)nk;
    a.bp = s.bp; a.bq = s.bq; a.tiles_p = s.tiles_p; a.tiles_q = s.tiles_q; a.splits = s.splits; a.k_split = s.k_split;
    a.partial = (float*)partial;
    a.np4 = (int)((np + 3) / 4 * 4);
    a.e.alpha = 1.0f;
    return a;
}

static size_t packed_bytes(int64_t rows, int64_t cols, int es) { return align256((size_t)rows * pad16(cols, es) * es); }
static size_t operand_bytes(const void* p, int64_t ld, int64_t rows, int64_t cols, int es) {
    return ready(p, ld, cols, es) ? 0 : packed_bytes(rows, cols, es);
}
static size_t column_bytes(int64_t M, int64_t N) { return align256((size_t)((M + kSlopeRows - 1) / kSlopeRows) * ((N + 3) / 4 * 4) * 4); }

static int check_linear(const char* who, int64_t M, int64_t N, int64_t K, int dtype, int act) {
    if (M < 0 || N < 0 || K < 0) return fail(NEMO_ERR_INVALID, "%s: negative size", who);
    if (dtype != NEMO_F32 && dtype != NEMO_BF16 && dtype != NEMO_F16) return fail(NEMO_ERR_INVALID, "%s: unknown element type %d", who, dtype);
    if (act < 0 || act > 3) return fail(NEMO_ERR_INVALID, "%s: unknown activation %d", who, act);
    // a launch holds 2^32 threads: at least 64 x 64 results a workgroup of 256
    const int64_t pairs[3][2] = {{M, N}, {M, K}, {N, K}};
    for (const auto& p : pairs)
        if (p[0] > 0x7FFFF000 || p[1] > 0x7FFFF000 || p[0] * p[1] > (1LL << 34) || ((p[0] + 63) / 64) * ((p[1] + 63) / 64) > (1LL << 23))
            return fail(NEMO_ERR_UNSUPPORTED, "%s: a matrix of %lld x %lld is too large for one launch", who, (long long)p[0], (long long)p[1]);
    return NEMO_OK;
}

// Offsets within a tile of 256 rows are 32-bit: rows lie at most 4 MiB apart.  cols: the contiguous extent, what a packed copy has.
constexpr int64_t kRowBytes = 1 << 22;
static int check_stride(const char* who, const void* p, int64_t ld, int64_t cols, int dtype) {
    const int es = elem_size(dtype);
    if ((ready(p, ld, cols, es) ? ld : pad16(cols, es)) * es > kRowBytes) return fail(NEMO_ERR_UNSUPPORTED, "%s: rows more than 4 MiB apart", who);
    return NEMO_OK;
}

}  // namespace nemo

using namespace nemo;

extern "C" size_t nemo_linear_workspace(const void* x, int64_t ldx, const void* weight, int64_t ldw, int64_t M, int64_t N, int64_t K,
                                        int32_t dtype) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    const int es = elem_size(dtype);
    return operand_bytes(x, ldx, M, K, es) + operand_bytes(weight, ldw, N, K, es) + partial_bytes(N, M, shape_of(N, M, K, dtype, false));
}

extern "C" int nemo_linear(const void* x, int64_t ldx, const void* weight, int64_t ldw, const void* bias, const void* residual, int64_t ldr,
                           int64_t M, int64_t N, int64_t K, int32_t dtype, int32_t activation, float alpha, float beta, void* y, void* pre,
                           void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check_linear("nemo_linear", M, N, K, dtype, activation);
    if (rc) return rc;
    if (M == 0 || N == 0) return NEMO_OK;
    if (!y || (K > 0 && (!x || !weight))) return fail(NEMO_ERR_INVALID, "nemo_linear: null argument");
    if ((K > 0 && (ldx < K || ldw < K)) || (residual && ldr < N)) return fail(NEMO_ERR_INVALID, "nemo_linear: a row stride shorter than the row");
    if (K > 0 && ((rc = check_stride("nemo_linear", x, ldx, K, dtype)) || (rc = check_stride("nemo_linear", weight, ldw, K, dtype)))) return rc;
    const size_t need = nemo_linear_workspace(x, ldx, weight, ldw, M, N, K, dtype);
    if (workspace_bytes < need || (need && !workspace))
        return fail(NEMO_ERR_INVALID, "nemo_linear: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    if (need && ((uintptr_t)workspace & 15)) return fail(NEMO_ERR_INVALID, "nemo_linear: the workspace must start on 16 bytes");
    hipStream_t st = (hipStream_t)stream;
    char* ws = (char*)workspace;
    Operand P = {weight, ldw}, Q = {x, ldx};
    if (K > 0) {
        Packer pack = {dtype};
        P = pack.operand(weight, ldw, N, K, ws);
        Q = pack.operand(x, ldx, M, K, ws);
        pack.launch(st);
    }
    const Shape s = shape_of(N, M, K, dtype, false);
    GemmArgs a = gemm_args(P, Q, N, M, K, s, ws);
    a.e = {alpha, beta, activation, bias, residual, ldr, y, N, pre};
    launch_gemm(dtype, a, false, false, st);
    HIP_TRY(hipGetLastError());
    return NEMO_OK;
}

// dz is the incoming gradient itself where there is no activation and its rows suit the tiles; else it is written with padded rows.
static bool slope_needed(const void* grad_y, int64_t ldg, int64_t N, int dtype, int act) {
    return act != ACT_NONE || !ready(grad_y, ldg, N, elem_size(dtype)) || ldg * elem_size(dtype) > kRowBytes;
}

extern "C" size_t nemo_linear_backward_workspace(const void* grad_y, int64_t ldg, const void* x, int64_t ldx, const void* weight, int64_t ldw,
                                                 int64_t M, int64_t N, int64_t K, int32_t dtype, int32_t activation) {
    if (M <= 0 || N <= 0) return 0;
    if (K <= 0) return column_bytes(M, N);
    const int es = elem_size(dtype);
    const size_t dx = partial_bytes(K, M, shape_of(K, M, N, dtype, true)), dw = partial_bytes(K, N, shape_of(K, N, M, dtype, true));
    return (slope_needed(grad_y, ldg, N, dtype, activation) ? packed_bytes(M, N, es) : 0) + operand_bytes(x, ldx, M, K, es) +
           operand_bytes(weight, ldw, N, K, es) + (dx > dw ? dx : dw) + column_bytes(M, N);
}

template <typename T>
static void launch_slope(const void* dy, int64_t ldg, const void* pre, int64_t M, int64_t N, int act, float beta, void* dz, int ldz, void* dr,
                         float* partial, void* grad_bias, hipStream_t st) {
    const int np4 = (int)((N + 3) / 4 * 4);
    const int width = dz ? ldz : (int)N;
    // grid.y holds 65535 blocks; taller inputs go in slices
    const int64_t blocks = (M + kSlopeRows - 1) / kSlopeRows;
    for (int64_t b0 = 0; b0 < blocks; b0 += 65535) {
        const int64_t nb = blocks - b0 < 65535 ? blocks - b0 : 65535, r0 = b0 * kSlopeRows;
        hipLaunchKernelGGL((slope_kernel<T>), dim3((width + 255) / 256, (unsigned)nb), dim3(256), 0, st, (const T*)dy + r0 * ldg, (long)ldg,
                           pre ? (const T*)pre + r0 * N : (const T*)nullptr, (long)N, (long)(M - r0), (int)N, act, beta,
                           dz ? (T*)dz + r0 * ldz : (T*)nullptr, ldz, dr ? (T*)dr + r0 * N : (T*)nullptr,
                           partial ? partial + (size_t)b0 * np4 : (float*)nullptr, np4);
    }
    if (grad_bias)
        hipLaunchKernelGGL((column_sum_kernel<T>), dim3((unsigned)((N + 31) / 32)), dim3(256), 0, st, partial, (int)blocks, np4, (int)N,
                           (T*)grad_bias);
}

extern "C" int nemo_linear_backward(const void* grad_y, int64_t ldg, const void* x, int64_t ldx, const void* weight, int64_t ldw,
                                    const void* pre, int64_t M, int64_t N, int64_t K, int32_t dtype, int32_t activation, float alpha, float beta,
                                    void* grad_x, void* grad_weight, void* grad_bias, void* grad_residual, void* workspace,
                                    size_t workspace_bytes, void* stream) {
    int rc = check_linear("nemo_linear_backward", M, N, K, dtype, activation);
    if (rc) return rc;
    if (M > 0 && N > 0 && !grad_y) return fail(NEMO_ERR_INVALID, "nemo_linear_backward: null gradient");
    if (M > 0 && N > 0 && ldg < N) return fail(NEMO_ERR_INVALID, "nemo_linear_backward: a row stride shorter than the row");
    if (!grad_x && !grad_weight && !grad_bias) activation = ACT_NONE;        // the residual's gradient passes the activation by
    if (activation != ACT_NONE && M > 0 && N > 0 && !pre) return fail(NEMO_ERR_INVALID, "nemo_linear_backward: the activation needs `pre`");
    if (M > 0 && N > 0 && K > 0 && ((grad_x && (!weight || ldw < K)) || (grad_weight && (!x || ldx < K))))
        return fail(NEMO_ERR_INVALID, "nemo_linear_backward: null operand or a row stride shorter than the row");
    if (M > 0 && N > 0 && K > 0 && (grad_x || grad_weight)) {
        if (pad16(N, elem_size(dtype)) * (int64_t)elem_size(dtype) > kRowBytes)
            return fail(NEMO_ERR_UNSUPPORTED, "nemo_linear_backward: rows of grad_y longer than 4 MiB");
        if ((grad_x && (rc = check_stride("nemo_linear_backward", weight, ldw, K, dtype))) ||
            (grad_weight && (rc = check_stride("nemo_linear_backward", x, ldx, K, dtype))))
            return rc;
    }
    const size_t need = nemo_linear_backward_workspace(grad_y, ldg, x, ldx, weight, ldw, M, N, K, dtype, activation);
    if (workspace_bytes < need || (need && !workspace))
        return fail(NEMO_ERR_INVALID, "nemo_linear_backward: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    if (need && ((uintptr_t)workspace & 15)) return fail(NEMO_ERR_INVALID, "nemo_linear_backward: the workspace must start on 16 bytes");
    hipStream_t st = (hipStream_t)stream;
    const int es = elem_size(dtype);
    char* ws = (char*)workspace;
    const bool products = (grad_x || grad_weight) && K > 0;
    Operand dz = {grad_y, ldg};
    void* dz_out = nullptr;
    const int ldz = pad16(N, es);
    if (products && M > 0 && N > 0 && slope_needed(grad_y, ldg, N, dtype, activation)) {
        dz_out = ws;
        ws += packed_bytes(M, N, es);
        dz = {dz_out, ldz};
    }
    float* col_partial = nullptr;
    if (grad_bias && M > 0) {
        col_partial = (float*)ws;
        ws += column_bytes(M, N);
    }
    if (N > 0 && ((M > 0 && (dz_out || grad_residual)) || grad_bias)) {
        if (dtype == NEMO_F32)
            launch_slope<float>(grad_y, ldg, pre, M, N, activation, beta, dz_out, ldz, grad_residual, col_partial, grad_bias, st);
        else if (dtype == NEMO_BF16)
            launch_slope<bf16>(grad_y, ldg, pre, M, N, activation, beta, dz_out, ldz, grad_residual, col_partial, grad_bias, st);
        else
            launch_slope<f16>(grad_y, ldg, pre, M, N, activation, beta, dz_out, ldz, grad_residual, col_partial, grad_bias, st);
    }
    Operand W = {weight, ldw}, X = {x, ldx};
    if (K > 0) {
        Packer pack = {dtype};
        if (grad_x && M > 0) W = pack.operand(weight, ldw, N, K, ws);
        if (grad_weight && N > 0) X = pack.operand(x, ldx, M, K, ws);
        pack.launch(st);
    }
    if (grad_x && M > 0 && K > 0) {
        const Shape s = shape_of(K, M, N, dtype, true);
        GemmArgs a = gemm_args(W, dz, K, M, N, s, ws);
        a.e = {alpha, 0.0f, ACT_NONE, nullptr, nullptr, 0, grad_x, K, nullptr};
        launch_gemm(dtype, a, true, false, st);
    }
    if (grad_weight && N > 0 && K > 0) {
        const Shape s = shape_of(K, N, M, dtype, true);
        GemmArgs a = gemm_args(X, dz, K, N, M, s, ws);
        a.e = {alpha, 0.0f, ACT_NONE, nullptr, nullptr, 0, grad_weight, K, nullptr};
        launch_gemm(dtype, a, true, true, st);
    }
    HIP_TRY(hipGetLastError());
    return NEMO_OK;
}
