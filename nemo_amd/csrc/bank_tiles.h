// What the kernels of bank_forward.hip and bank_gradient.hip share: arguments, tiles in LDS, the first product.
//
// 32 "owner" rows, whose fragments a wave keeps in registers, are multiplied with tiles of 32 "other" rows that the workgroup's four waves share in
// LDS (copied from global memory without registers), on v_mfma_f32_32x32x16_bf16 with the other rows as first operand.  Register 4 b + i of lane l
// then holds the product of owner row l % 32 with other row 8 b + 4 (l / 32) + i: a lane sees one owner row only.
//
// f32 rows are three bf16 pieces, x = h + m + l, each the rounding of what the ones before leave (24 bits together, the range of f32), written by a
// kernel of its own in front.  A product is h h' + h m' + m h' + m m' + h l' + l h'; what is left out is below 2^-26 of it, less than f32's own
// rounding, and sums are f32 sums.  Six bf16 instructions take 3/8 of the time of the f32 matrix instructions, which moreover share their
// multipliers with the vector units, so that nothing runs beside them (8000 x 13416 x 128 with a list: 351 us on those).
#pragma once
#include <type_traits>

#include "softmax_state.h"

namespace nemo {

static __device__ const u32x4 g_zero_row = {0, 0, 0, 0};

// 32 x 32 products; a fragment is 16 bytes a lane, k of 16: lane group g = lane / 32 holds 8 g .. 8 g + 7.
constexpr int kFragK = 16;
__device__ inline void wide_mma(f32x16_t& acc, const u32x4& p, const u32x4& q) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, p), __builtin_bit_cast(bf16x8, q), acc, 0, 0, 0);
}
// NP pieces a value (1 or 3): piece i of one operand meets pieces 0 .. NP - 1 - i of the other.  The pairs in the order in which they are multiplied.
template <int NP> struct Pairs {
    static constexpr int N = NP * (NP + 1) / 2;
    static __device__ constexpr int first(int u) { return NP == 1 ? 0 : u < 3 ? 0 : u < 5 ? 1 : 2; }
    static __device__ constexpr int second(int u) { return NP == 1 ? 0 : u < 3 ? u : u < 5 ? u - 3 : 0; }
};

struct BankArgs {
    const bf16* own;               // rows whose fragments stay in registers: [n_own][ld_own], piece n at n CP
    const bf16* other;
    long ld_own, ld_other;         // elements
    int n_own, n_other, channels;  // channels beyond which rows hold nothing (a multiple of 8)
    int grad_channels;             // of the gradient's rows
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
    const float* coef;             // [K_COUNT][features]
    float* partial;                // [parts][n_own][CP] when parts > 1
    void* grad;                    // [n_own][grad_channels]
};

// A tile of 32 rows in LDS.  Each instruction of a copy writes 1024 bytes, RPI rows, and 16 bytes of padding are left behind them; chunk c (16 bytes)
// of row r lies at c ^ flip(r) within its row.  Padding and flip put what one LDS read touches into different banks: the same chunk of 16
// consecutive rows (row_fragment), and 64 bytes of four consecutive rows (the transposing reads of the second product).  flip reaches the
// bits MASK of a chunk index only, so that most addresses of a lane differ by constants, which need no registers.
template <int CP> struct Tile {
    static constexpr int RB = CP * 2, CPR = RB / 16, RPI = 1024 / RB, PITCH = 1024 + 16;
    static constexpr int MASK = RPI == 8 ? 7 : RPI == 4 ? 12 : 8;
    static constexpr int ROWS = 32, COPIES = ROWS / RPI, BYTES = COPIES * PITCH;       // BYTES of one piece
    static __device__ constexpr int flip(int r) { return RPI == 8 ? r & 7 : RPI == 4 ? (r & 3) << 2 : (r & 1) << 3; }
    static __device__ constexpr int row(int r) { return r / RPI * PITCH + r % RPI * RB; }
    // Byte offset of chunk a + b (no bit in common; a a constant) in a row whose flip is f.
    static __device__ constexpr int chunk(int a, int b, int f) { return ((((a & MASK) | (b & MASK)) ^ f) + (a & ~MASK) + (b & ~MASK)) << 4; }
};

// What a lane copies of every tile: its chunk of row `row` of the tile, or zeros (rows beyond the last, channels beyond the last).
template <int NP, int CP> struct Stager {
    typedef Tile<CP> L;
    static constexpr int N = L::COPIES / 4;                            // copies of a wave and piece
    const bf16* src[N];
    int row[N];
    long step;                                                         // elements from tile to tile
    int rows, wave;
    __device__ inline Stager(const BankArgs& a, int wave_, int lane) : step(32 * a.ld_other), rows(a.n_other), wave(wave_) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r = (i * 4 + wave) * L::RPI + lane / L::CPR, c = (lane & (L::CPR - 1)) ^ L::flip(r);
            src[i] = a.other + (long)r * a.ld_other + c * 8;
            row[i] = c * 8 < a.channels ? r : 0x40000000;
        }
    }
    __device__ inline void copy(char* lds, int tile) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const bf16* p = src[i] + (long)tile * step;
            const bool in = tile * 32 + row[i] < rows;
#pragma unroll
            for (int n = 0; n < NP; ++n)
                copy_to_lds(in ? (const void*)(p + n * CP) : (const void*)&g_zero_row, lds + n * L::BYTES + (i * 4 + wave) * L::PITCH);
        }
    }
    // A tile of the first n of the rows in `list`, zeros behind them.
    __device__ inline void gather(char* lds, const BankArgs& a, const int* list, int n, int lane) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r = (i * 4 + wave) * L::RPI + lane / L::CPR, c = (lane & (L::CPR - 1)) ^ L::flip(r);
            const bool in = r < n && c * 8 < a.channels;
            const bf16* p = a.other + (in ? (long)list[r] : 0) * a.ld_other + c * 8;
#pragma unroll
            for (int k = 0; k < NP; ++k)
                copy_to_lds(in ? (const void*)(p + k * CP) : (const void*)&g_zero_row, lds + k * L::BYTES + (i * 4 + wave) * L::PITCH);
        }
    }
};

// Fragment kf of the tile's rows, one piece.
template <int CP>
__device__ inline u32x4 row_fragment(const char* lds, int kf, int lane) {
    typedef Tile<CP> L;
    const int r = lane & 31;
    return *(const u32x4*)(lds + L::row(r) + L::chunk(2 * kf, lane >> 5, L::flip(r)));
}

// Fragments of owner rows straight from memory.
template <int NP, int CP>
__device__ inline void own_fragments(u32x4 (&q)[NP][CP / kFragK], const BankArgs& a, int own0, int lane, bool negate) {
    const uint32_t flip = negate ? 0x80008000u : 0u;
    const int row = own0 + (lane & 31);
#pragma unroll
    for (int n = 0; n < NP; ++n)
#pragma unroll
        for (int kf = 0; kf < CP / kFragK; ++kf) {
            const int c = (kf * 2 + (lane >> 5)) * 8;
            q[n][kf] = row < a.n_own && c < a.channels ? *(const u32x4*)(a.own + (size_t)row * a.ld_own + n * CP + c) : u32x4{0, 0, 0, 0};
            q[n][kf] ^= flip;
        }
}

template <int NP, int CP>
__device__ inline f32x16_t products(const char* lds, const u32x4 (&q)[NP][CP / kFragK], int lane) {
    f32x16_t acc = {};
#pragma unroll
    for (int kf = 0; kf < CP / kFragK; ++kf) {
        u32x4 f[NP];
#pragma unroll
        for (int n = 0; n < NP; ++n) f[n] = row_fragment<CP>(lds + n * Tile<CP>::BYTES, kf, lane);
#pragma unroll
        for (int u = 0; u < Pairs<NP>::N; ++u) wide_mma(acc, f[Pairs<NP>::first(u)], q[Pairs<NP>::second(u)][kf]);
        if (kf % 4 == 3) __builtin_amdgcn_sched_barrier(0);            // reads no further ahead: registers
    }
    return acc;
}

// Keeps the compiler from moving the computation of x behind this point (it would put it where x is used, out of reach of the matrix
// instructions that it is meant to run beside).
__device__ inline void settle(u32x4& x) { asm volatile("" : "+v"(x)); }
__device__ inline void settle(float& x) { asm volatile("" : "+v"(x)); }

struct __attribute__((packed, aligned(4))) LooseQuad { f32x4 v; };

// Weights of the lane's 16 other rows j0 + 8 b + 4 g + i, +inf (left out) beyond `end`; w: the row of weights of the lane's feature row.
__device__ inline void row_weights(float wv[16], const float* w, int j0, int g, int end) {
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        const int j = j0 + 8 * b + 4 * g;
        if (j0 + 32 <= end) {
            const f32x4 q = ((const LooseQuad*)(w + j))->v;
#pragma unroll
            for (int i = 0; i < 4; ++i) wv[4 * b + i] = q[i];
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) wv[4 * b + i] = j + i < end ? w[j + i] : __builtin_inff();
        }
    }
}


template <typename T> void launch_bank_forward(const BankArgs& a, hipStream_t st);
template <typename T> void launch_bank_gradient(const BankArgs& a, bool own_bank, hipStream_t st);
template <> void launch_bank_forward<float>(const BankArgs& a, hipStream_t st);
template <> void launch_bank_forward<bf16>(const BankArgs& a, hipStream_t st);
template <> void launch_bank_gradient<float>(const BankArgs& a, bool own_bank, hipStream_t st);
template <> void launch_bank_gradient<bf16>(const BankArgs& a, bool own_bank, hipStream_t st);

// The six arrays that the gradient kernels need of every feature row; rows beyond the last have p = 0 and no target.
enum { K_M, K_LOG2_S, K_C, K_G2, K_LOGP, K_TARGET, K_COUNT };
constexpr int coef_rows(int64_t rows) { return (int)((rows + 63) / 64 * 64 + 192); }

inline int padded_channels(int c) { return c <= 64 ? 64 : c <= 128 ? 128 : 256; }

}  // namespace nemo
