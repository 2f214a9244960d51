// What the dense operators (linear.hip, log_probs.hip, the bank kernels) share: element types, accesses at any element, the matrix-core fragments
// of linear.hip, the direct copy from global memory to LDS, reductions over a wave.
//
// A fragment is 16 bytes a lane, for either operand of a product:
//   16-bit types  v_mfma_f32_16x16x32: lane = (row r = lane % 16, group g = lane / 16), elements k = 8 g .. 8 g + 7 of a block of 32;
//   f32           v_mfma_f32_32x32x2 (four of them): lane = (row r = lane % 32, group g = lane / 32), elements k = 4 g .. 4 g + 3 of a
//                 block of 8.  The hardware pairs element i of one operand with element i of the other; which k that is does not
//                 matter as long as both operands agree, so four consecutive f32 are loaded at once.
// Results: lane % FR is the row of the SECOND operand (q); the FIRST operand's rows (p) run through the registers, four consecutive
// ones at a time: register 4 b + i holds p = 8 b + 4 (lane / 32) + i (f32) or 4 (lane / 16) + i (16-bit types).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace nemo {

typedef __bf16 bf16;
typedef _Float16 f16;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x8_t __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

#define NEMO_LDS __attribute__((address_space(3)))
#define NEMO_GLOBAL __attribute__((address_space(1)))

template <typename T> __device__ inline float to_f32(T x) { return (float)x; }
template <typename T> __device__ inline T from_f32(float x) { return (T)x; }       // round to nearest even

__device__ inline float neg_inf() { return -__builtin_inff(); }

// N elements at any element's address: 8- and 16-byte accesses need no alignment on this hardware.
template <typename T, int N> struct __attribute__((packed, aligned(sizeof(T)))) Loose {
    typedef T V __attribute__((ext_vector_type(N)));
    V v;
};
template <int N, typename T> __device__ inline typename Loose<T, N>::V load_loose(const T* p) { return ((const Loose<T, N>*)p)->v; }
template <int N, typename T> __device__ inline void store_loose(T* p, typename Loose<T, N>::V v) { ((Loose<T, N>*)p)->v = v; }

// ---- matrix cores ---------------------------------------------------------------------------------------------------------------
template <typename T> struct Mma;

template <> struct Mma<float> {
    typedef f32x16_t Acc;
    static constexpr int FR = 32, NG = 2, KF = 8, QUADS = 4;           // rows of a fragment, lane groups, k of a fragment, p quads of a result
    static __device__ inline void run(Acc& acc, const u32x4& p, const u32x4& q) {
        const f32x4 a = __builtin_bit_cast(f32x4, p), b = __builtin_bit_cast(f32x4, q);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], acc, 0, 0, 0);
    }
};

template <> struct Mma<bf16> {
    typedef f32x4 Acc;
    static constexpr int FR = 16, NG = 4, KF = 32, QUADS = 1;
    static __device__ inline void run(Acc& acc, const u32x4& p, const u32x4& q) {
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, p), __builtin_bit_cast(bf16x8, q), acc, 0, 0, 0);
    }
};

template <> struct Mma<f16> {
    typedef f32x4 Acc;
    static constexpr int FR = 16, NG = 4, KF = 32, QUADS = 1;
    static __device__ inline void run(Acc& acc, const u32x4& p, const u32x4& q) {
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, p), __builtin_bit_cast(f16x8_t, q), acc, 0, 0, 0);
    }
};

// 64 lanes copy 16 bytes each from their own global addresses to 1024 consecutive bytes of LDS at `lds` (the same for all lanes).
__device__ inline void copy_to_lds(const void* g, void* lds) {
    __builtin_amdgcn_global_load_lds((NEMO_GLOBAL void*)g, (NEMO_LDS void*)lds, 16, 0, 0);
}

// The same with 4 bytes a lane, 256 bytes of LDS.
__device__ inline void copy_words_to_lds(const void* g, void* lds) {
    __builtin_amdgcn_global_load_lds((NEMO_GLOBAL void*)g, (NEMO_LDS void*)lds, 4, 0, 0);
}

// The copies are asynchronous: a wave waits here for its own.
__device__ inline void wait_for_copies() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// A barrier behind which other waves read what this one has copied or written to LDS, or copy over what it has read.  __syncthreads alone does not wait
// for copies, and around a loop not always for writes either: the compiler leaves the wait out in front of a barrier whose copies it has not
// seen yet when it gets there, those of the loop's last turn.
__device__ inline void publish_lds() {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __syncthreads();
}

// ---- reductions -----------------------------------------------------------------------------------------------------------------
// Over the 64 lanes of a wave, all of them active, with the lane permutations of the vector units (a tenth of the latency of exchanges through
// LDS): within four, eight and sixteen lanes, then lane 15 of a row of sixteen into the next one, lane 31 into the upper half; lane 63 has it all.
template <int CTRL, int ROWS = 0xF> __device__ inline int permuted(int v, int other_rows) {
    return __builtin_amdgcn_update_dpp(other_rows, v, CTRL, ROWS, 0xF, false);
}
template <int CTRL, int ROWS = 0xF> __device__ inline float permuted(float v, float other_rows) {
    return __builtin_bit_cast(float, permuted<CTRL, ROWS>(__builtin_bit_cast(int, v), __builtin_bit_cast(int, other_rows)));
}
template <typename V, typename Op> __device__ inline V wave_reduce(V v, V neutral, Op op) {
    v = op(v, permuted<0xB1>(v, neutral));                             // lanes 1 0 3 2
    v = op(v, permuted<0x4E>(v, neutral));                             // lanes 2 3 0 1
    v = op(v, permuted<0x141>(v, neutral));                            // eight lanes mirrored
    v = op(v, permuted<0x140>(v, neutral));                            // sixteen lanes mirrored
    v = op(v, permuted<0x142, 0xA>(v, neutral));
    v = op(v, permuted<0x143, 0xC>(v, neutral));
    const int last = __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63);
    return __builtin_bit_cast(V, last);
}
__device__ inline float wave_sum(float v) {
    return wave_reduce(v, 0.0f, [](float a, float b) { return a + b; });
}
__device__ inline float wave_max(float v) {
    return wave_reduce(v, neg_inf(), [](float a, float b) { return fmaxf(a, b); });
}
__device__ inline int wave_min(int v) {
    return wave_reduce(v, 0x7FFFFFFF, [](int a, int b) { return min(a, b); });
}

}  // namespace nemo
