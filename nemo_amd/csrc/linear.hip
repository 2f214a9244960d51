// y = act(alpha x W^T + bias) + beta r and its gradients.
//
// One tiled product serves the forward pass and both weight- and input-gradients.  It computes
//     C[q][p] = sum_k P(p, k) Q(q, k)
// where p, the column of the result that is contiguous in memory, is the FIRST operand of the matrix instruction, so that a lane ends
// up with four consecutive columns of one row and stores them with one instruction.  An operand is "plain" when k is contiguous in
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
// Operands must start on 16 bytes, have rows that start on 16 bytes and a contiguous extent of whole 16 bytes; others are first copied
// into the workspace with padded rows (pack_kernel).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/nemo_hip.h"
#include "dense.h"
#include "errors.h"

namespace nemo {

__device__ const u32x4 g_zero_chunk = {0, 0, 0, 0};                    // what the lanes beyond the end of k copy

enum { ACT_NONE = 0, ACT_RELU = 1, ACT_GELU = 2, ACT_SILU = 3 };

__device__ inline float activate(float z, int act) {
    switch (act) {
        case ACT_RELU: return z > 0.0f ? z : (z != z ? z : 0.0f);
        case ACT_GELU: return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
        case ACT_SILU: return z / (1.0f + expf(-z));
        default: return z;
    }
}

// d act / d z.  relu's slope at 0 is 0.  For large negative z: gelu's exp(-z^2 / 2) underflows to 0 and silu's s to 0, for large
// positive ones 1 + z (1 - s) is 1 because 1 - s is written as the sigmoid of -z.
__device__ inline float activate_slope(float z, int act) {
    switch (act) {
        case ACT_RELU: return z > 0.0f ? 1.0f : (z != z ? z : 0.0f);
        case ACT_GELU: return 0.5f * (1.0f + erff(z * 0.70710678118654752f)) + z * expf(-0.5f * z * z) * 0.39894228040143268f;
        case ACT_SILU: {
            const float s = 1.0f / (1.0f + expf(-z)), r = 1.0f / (1.0f + expf(z));
            return s * (1.0f + z * r);
        }
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
    int vec;                   // rows of out, pre and residual start on four elements, and so does their end
};

struct GemmArgs {
    const void* P;
    const void* Q;
    long ldp, ldq;             // elements
    int np, nq, nk;
    int tiles_p, tiles_q, splits, k_split;         // k_split: k of one split, whole steps
    float* partial;            // [splits][nq][np4] when splits > 1
    int np4;
    Epilogue e;
};

// Rounds to T; for the stored pre-activation of f16 a value that rounds to zero keeps its sign as the smallest subnormal, so that relu's
// slope is that of the value before rounding.
template <typename T> __device__ inline T round_pre(float z) { return (T)z; }
template <> __device__ inline f16 round_pre<f16>(float z) {
    const f16 h = (f16)z;
    if (h == (f16)0.0f && z != 0.0f) return z > 0.0f ? (f16)5.9604644775390625e-8f : (f16)-5.9604644775390625e-8f;
    return h;
}

// Four consecutive columns p .. p + 3 of row q.
template <typename T>
__device__ inline void epilogue4(const Epilogue& e, const float v[4], int q, int p, int np) {
    const int n = np - p < 4 ? np - p : 4;
    const T* bias = (const T*)e.bias;
    const T* res = e.residual ? (const T*)e.residual + (size_t)q * e.ldr + p : nullptr;
    T* out = (T*)e.out + (size_t)q * e.ldo + p;
    T* pre = e.pre ? (T*)e.pre + (size_t)q * e.ldo + p : nullptr;
    float z[4], r[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    typedef T T4 __attribute__((ext_vector_type(4)));
    if (e.vec) {
        if (bias) {
            const T4 b = *(const T4*)(bias + p);
#pragma unroll
            for (int i = 0; i < 4; ++i) z[i] = e.alpha * v[i] + to_f32(b[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) z[i] = e.alpha * v[i];
        }
        if (res) {
            const T4 t = *(const T4*)res;
#pragma unroll
            for (int i = 0; i < 4; ++i) r[i] = to_f32(t[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            z[i] = e.alpha * v[i];
            if (bias && i < n) z[i] += to_f32(bias[p + i]);
            if (res && i < n) r[i] = to_f32(res[i]);
        }
    }
    if (pre) {
        if (e.vec) {
            T4 t;
#pragma unroll
            for (int i = 0; i < 4; ++i) t[i] = round_pre<T>(z[i]);
            *(T4*)pre = t;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i < n) pre[i] = round_pre<T>(z[i]);
        }
    }
    if (e.act != ACT_NONE) {
#pragma unroll
        for (int i = 0; i < 4; ++i) z[i] = activate(z[i], e.act);
    }
    if (res) {
#pragma unroll
        for (int i = 0; i < 4; ++i) z[i] += e.beta * r[i];
    }
    if (e.vec) {
        T4 t;
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] = from_f32<T>(z[i]);
        *(T4*)out = t;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < n) out[i] = from_f32<T>(z[i]);
    }
}

// Exclusive-or of the 16-byte chunk index of k row `k` in a transposed 16-bit tile: the 16 rows that one fragment read touches (8 g + 0..3
// or 8 g + 4..7) get different pairs of chunks as far as the row has them.
template <int CPR> __device__ inline int swizzle_t(int k) { return (2 * (((k >> 3) & 3) * 4 + (k & 3))) & (CPR - 1); }

template <typename T> constexpr int kstep() { return 128 / (int)sizeof(T); }

// A tile of ROWS rows x 128 bytes of k into `lds` by WAVES waves.
template <typename T, int ROWS, bool TR, int WAVES>
__device__ inline void stage(char* lds, const T* base, long ld, int row0, int rows, int k0, int nk, int wave, int lane) {
    constexpr int EPC = 16 / (int)sizeof(T);                           // elements of a chunk
    constexpr int CHUNKS = ROWS * 8;
    static_assert(CHUNKS % (64 * WAVES) == 0, "every wave copies the same number of kilobytes");
#pragma unroll
    for (int i = 0; i < CHUNKS / 64 / WAVES; ++i) {
        const int j = i * WAVES + wave, idx = j * 64 + lane;
        const T* src;
        bool in;
        if (!TR) {
            const int r = idx >> 3, c = (idx & 7) ^ (r & 7);
            const int row = min(row0 + r, rows - 1), k = k0 + c * EPC;
            in = k < nk;
            src = base + (size_t)row * ld + k;
        } else {
            constexpr int CPR = ROWS / EPC;
            const int kr = idx / CPR;
            const int c = (idx & (CPR - 1)) ^ (sizeof(T) == 2 ? swizzle_t<CPR>(kr) : 0);
            const int col = row0 + c * EPC, k = k0 + kr;
            in = k < nk && col < rows;
            src = base + (size_t)k * ld + col;
        }
        copy_to_lds(in ? (const void*)src : (const void*)&g_zero_chunk, lds + j * 1024);
    }
}

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

template <typename T, int BP, int BQ, int WP, int WQ, bool PT, bool QT>
__global__ __launch_bounds__(64 * WP * WQ, 2) void gemm_kernel(GemmArgs a) {
    typedef Mma<T> M;
    constexpr int WAVES = WP * WQ, TP = BP / WP, TQ = BQ / WQ, NP = TP / M::FR, NQ = TQ / M::FR;
    constexpr int BK = kstep<T>(), NKF = BK / M::KF;
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

    const int k_begin = split * a.k_split, k_end = min(a.nk, k_begin + a.k_split);
    const T* P = (const T*)a.P;
    const T* Q = (const T*)a.Q;
    typename M::Acc acc[NP][NQ];
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
        for (int j = 0; j < NQ; ++j) acc[i][j] = {};

    auto load = [&](char* lds, int k) {
        stage<T, BP, PT, WAVES>(lds, P, a.ldp, p0, a.np, k, k_end, wave, lane);
        stage<T, BQ, QT, WAVES>(lds + BP * 128, Q, a.ldq, q0, a.nq, k, k_end, wave, lane);
    };
    auto multiply = [&](const char* lds) {
#pragma unroll
        for (int kf = 0; kf < NKF; ++kf) {
            u32x4 pf[NP], qf[NQ];
#pragma unroll
            for (int i = 0; i < NP; ++i) pf[i] = fragment<T, BP, PT>(lds, wp * TP + i * M::FR, kf, lane);
#pragma unroll
            for (int j = 0; j < NQ; ++j) qf[j] = fragment<T, BQ, QT>(lds + BP * 128, wq * TQ + j * M::FR, kf, lane);
#pragma unroll
            for (int i = 0; i < NP; ++i)
#pragma unroll
                for (int j = 0; j < NQ; ++j) M::run(acc[i][j], pf[i], qf[j]);
        }
    };

    if (k_begin < k_end) load(lds0, k_begin);
    for (int k = k_begin; k < k_end; k += 2 * BK) {
        __syncthreads();                                               // the tile in lds0 is there, lds1 is free
        if (k + BK < k_end) load(lds1, k + BK);
        multiply(lds0);
        if (k + BK >= k_end) break;
        __syncthreads();
        if (k + 2 * BK < k_end) load(lds0, k + 2 * BK);
        multiply(lds1);
    }

    const int g = lane / M::FR;
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
        const int q = q0 + wq * TQ + j * M::FR + (lane & (M::FR - 1));
        if (q >= a.nq) continue;
#pragma unroll
        for (int i = 0; i < NP; ++i)
#pragma unroll
            for (int b = 0; b < M::QUADS; ++b) {
                const int p = p0 + wp * TP + i * M::FR + b * 8 + 4 * g;
                if (p >= a.np) continue;
                const float v[4] = {acc[i][j][4 * b], acc[i][j][4 * b + 1], acc[i][j][4 * b + 2], acc[i][j][4 * b + 3]};
                if (a.splits > 1)
                    *(f32x4*)(a.partial + ((size_t)split * a.nq + q) * a.np4 + p) = (f32x4){v[0], v[1], v[2], v[3]};
                else
                    epilogue4<T>(a.e, v, q, p, a.np);
            }
    }
}

// Sums the splits in their order and applies the epilogue; four columns a thread.
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(GemmArgs a) {
    const int quads = a.np4 >> 2;
    const long id = (long)blockIdx.x * 256 + threadIdx.x;
    if (id >= (long)quads * a.nq) return;
    const int q = (int)(id / quads), p = 4 * (int)(id % quads);
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = 0; s < a.splits; ++s) {
        const f32x4 t = *(const f32x4*)(a.partial + ((size_t)s * a.nq + q) * a.np4 + p);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += t[i];
    }
    epilogue4<T>(a.e, v, q, p, a.np);
}

// rows x cols (row stride ld) -> rows x ld_out, the columns beyond cols zero; 32-bit words of the copy a thread, ld_out a multiple of 16 bytes.
template <typename T>
__global__ __launch_bounds__(256) void pack_kernel(const T* src, long ld, long rows, int cols, T* dst, int ld_out) {
    constexpr int E = 16 / (int)sizeof(T);
    const int per_row = ld_out / E;
    const long id = (long)blockIdx.x * 256 + threadIdx.x;
    if (id >= rows * per_row) return;
    const long r = id / per_row;
    const int c = (int)(id % per_row) * E;
    const T* s = src + r * ld + c;
    union { T t[E]; u32x4 v; } u;
#pragma unroll
    for (int i = 0; i < E; ++i) u.t[i] = c + i < cols ? s[i] : (T)0.0f;
    *(u32x4*)(dst + r * (long)ld_out + c) = u.v;
}

// dz = dy act'(pre) (rounded to T because the matrix cores take T), dr = beta dy, and per block of rows the column sums of the unrounded
// dz (for the bias).  A workgroup takes 64 columns x ROWS rows: 16 threads of four columns, 16 rows at a time.
constexpr int kSlopeRows = 256;
template <typename T>
__global__ __launch_bounds__(256) void slope_kernel(const T* dy, long ldg, const T* pre, long ldpre, long m, int n, int act, float beta,
                                                    T* dz, int ldz, T* dr, float* col_partial, int np4) {
    const int c = blockIdx.x * 64 + (threadIdx.x & 15) * 4, ry = threadIdx.x >> 4;
    const long r0 = (long)blockIdx.y * kSlopeRows;
    const long r1 = r0 + kSlopeRows < m ? r0 + kSlopeRows : m;
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (long r = r0 + ry; r < r1; r += 16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (c + i < n) {
                const float g = to_f32(dy[r * ldg + c + i]);
                const float d = act == ACT_NONE ? g : g * activate_slope(to_f32(pre[r * ldpre + c + i]), act);
                sum[i] += d;
                if (dz) dz[r * (long)ldz + c + i] = from_f32<T>(d);
                if (dr) dr[r * (long)n + c + i] = from_f32<T>(beta * g);
            } else if (dz && c + i < ldz) {
                dz[r * (long)ldz + c + i] = (T)0.0f;
            }
        }
    }
    if (!col_partial) return;
    __shared__ float s[16][64];
#pragma unroll
    for (int i = 0; i < 4; ++i) s[ry][(threadIdx.x & 15) * 4 + i] = sum[i];
    __syncthreads();
    if (threadIdx.x < 64 && blockIdx.x * 64 + threadIdx.x < np4) {
        float t = 0.0f;
        for (int i = 0; i < 16; ++i) t += s[i][threadIdx.x];
        col_partial[(size_t)blockIdx.y * np4 + blockIdx.x * 64 + threadIdx.x] = t;
    }
}

template <typename T>
__global__ __launch_bounds__(256) void column_sum_kernel(const float* partial, int blocks, int np4, int n, T* out) {
    // 32 columns a workgroup, eight threads each
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), part = threadIdx.x >> 5;
    float t = 0.0f;
    if (c < n)
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

// Splits of k for a product with too few tiles to fill 256 compute units: as many as bring it to about two workgroups each, of at least
// four steps of k.
struct Shape { int big, tiles_p, tiles_q, splits, k_split; };
static Shape shape_of(int64_t np, int64_t nq, int64_t nk, int dtype) {
    Shape s;
    const int step = 128 / elem_size(dtype);
    s.big = 128;
    s.tiles_p = (int)((np + s.big - 1) / s.big);
    s.tiles_q = (int)((nq + s.big - 1) / s.big);
    const int64_t tiles = (int64_t)s.tiles_p * s.tiles_q, steps = (nk + step - 1) / step;
    int64_t want = tiles >= 256 ? 1 : 512 / tiles;
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
    hipLaunchKernelGGL((gemm_kernel<T, 128, 128, 2, 2, PT, QT>), dim3((unsigned)wgs), dim3(256), 0, st, a);
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
static void launch_pack(const void* src, int64_t ld, int64_t rows, int64_t cols, void* dst, int ld_out, hipStream_t st) {
    const long threads = rows * (ld_out / (16 / (long)sizeof(T)));
    hipLaunchKernelGGL((pack_kernel<T>), dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, st, (const T*)src, ld, rows, (int)cols, (T*)dst,
                       ld_out);
}

// An operand as the tiles want it: where it lies, or its packed copy taken from the workspace.
struct Operand { const void* p; int64_t ld; };
static Operand operand(int dtype, const void* p, int64_t ld, int64_t rows, int64_t cols, char*& ws, hipStream_t st) {
    const int es = elem_size(dtype);
    if (ready(p, ld, cols, es)) return {p, ld};
    const int ld_out = pad16(cols, es);
    void* dst = ws;
    ws += align256((size_t)rows * ld_out * es);
    if (dtype == NEMO_F32) launch_pack<float>(p, ld, rows, cols, dst, ld_out, st);
    else if (dtype == NEMO_BF16) launch_pack<bf16>(p, ld, rows, cols, dst, ld_out, st);
    else launch_pack<f16>(p, ld, rows, cols, dst, ld_out, st);
    return {dst, ld_out};
}

static GemmArgs gemm_args(Operand P, Operand Q, int64_t np, int64_t nq, int64_t nk, const Shape& s, void* partial) {
    GemmArgs a = {};
    a.P = P.p; a.Q = Q.p; a.ldp = P.ld; a.ldq = Q.ld;
    a.np = (int)np; a.nq = (int)nq; a.nk = (int)nk;
    a.tiles_p = s.tiles_p; a.tiles_q = s.tiles_q; a.splits = s.splits; a.k_split = s.k_split;
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
    // a launch holds 2^32 threads: 16 bytes of a copy a thread, a tile of 64 x 64 results a workgroup of 256
    const int64_t pairs[3][2] = {{M, N}, {M, K}, {N, K}};
    for (const auto& p : pairs)
        if (p[0] > 0x7FFFF000 || p[1] > 0x7FFFF000 || p[0] * p[1] > (1LL << 34) || ((p[0] + 63) / 64) * ((p[1] + 63) / 64) > (1LL << 23))
            return fail(NEMO_ERR_UNSUPPORTED, "%s: a matrix of %lld x %lld is too large for one launch", who, (long long)p[0], (long long)p[1]);
    return NEMO_OK;
}

}  // namespace nemo

using namespace nemo;

extern "C" size_t nemo_linear_workspace(const void* x, int64_t ldx, const void* weight, int64_t ldw, int64_t M, int64_t N, int64_t K,
                                        int32_t dtype) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    const int es = elem_size(dtype);
    return operand_bytes(x, ldx, M, K, es) + operand_bytes(weight, ldw, N, K, es) + partial_bytes(N, M, shape_of(N, M, K, dtype));
}

extern "C" int nemo_linear(const void* x, int64_t ldx, const void* weight, int64_t ldw, const void* bias, const void* residual, int64_t ldr,
                           int64_t M, int64_t N, int64_t K, int32_t dtype, int32_t activation, float alpha, float beta, void* y, void* pre,
                           void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check_linear("nemo_linear", M, N, K, dtype, activation);
    if (rc) return rc;
    if (M == 0 || N == 0) return NEMO_OK;
    if (!y || (K > 0 && (!x || !weight))) return fail(NEMO_ERR_INVALID, "nemo_linear: null argument");
    if ((K > 0 && (ldx < K || ldw < K)) || (residual && ldr < N)) return fail(NEMO_ERR_INVALID, "nemo_linear: a row stride shorter than the row");
    const size_t need = nemo_linear_workspace(x, ldx, weight, ldw, M, N, K, dtype);
    if (workspace_bytes < need || (need && !workspace))
        return fail(NEMO_ERR_INVALID, "nemo_linear: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    hipStream_t st = (hipStream_t)stream;
    const int es = elem_size(dtype);
    char* ws = (char*)workspace;
    Operand P = {weight, ldw}, Q = {x, ldx};
    if (K > 0) {
        P = operand(dtype, weight, ldw, N, K, ws, st);
        Q = operand(dtype, x, ldx, M, K, ws, st);
    }
    const Shape s = shape_of(N, M, K, dtype);
    GemmArgs a = gemm_args(P, Q, N, M, K, s, ws);
    a.e = {alpha, beta, activation, bias, residual, ldr, y, N, pre, 0};
    a.e.vec = N % 4 == 0 && ((uintptr_t)y & (4 * es - 1)) == 0 && (!pre || ((uintptr_t)pre & (4 * es - 1)) == 0) &&
              (!bias || ((uintptr_t)bias & (4 * es - 1)) == 0) && (!residual || (((uintptr_t)residual & (4 * es - 1)) == 0 && ldr % 4 == 0));
    launch_gemm(dtype, a, false, false, st);
    HIP_TRY(hipGetLastError());
    return NEMO_OK;
}

// dz is the incoming gradient itself where there is no activation and its rows suit the tiles.
static bool slope_needed(const void* grad_y, int64_t ldg, int64_t N, int dtype, int act) {
    return act != ACT_NONE || !ready(grad_y, ldg, N, elem_size(dtype));
}

extern "C" size_t nemo_linear_backward_workspace(const void* grad_y, int64_t ldg, const void* x, int64_t ldx, const void* weight, int64_t ldw,
                                                 int64_t M, int64_t N, int64_t K, int32_t dtype, int32_t activation) {
    if (M <= 0 || N <= 0) return 0;
    if (K <= 0) return column_bytes(M, N);
    const int es = elem_size(dtype);
    const size_t dx = partial_bytes(K, M, shape_of(K, M, N, dtype)), dw = partial_bytes(K, N, shape_of(K, N, M, dtype));
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
        hipLaunchKernelGGL((slope_kernel<T>), dim3((width + 63) / 64, (unsigned)nb), dim3(256), 0, st, (const T*)dy + r0 * ldg, (long)ldg,
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
    if (activation != ACT_NONE && M > 0 && N > 0 && !pre) return fail(NEMO_ERR_INVALID, "nemo_linear_backward: the activation needs `pre`");
    if (M > 0 && N > 0 && K > 0 && ((grad_x && (!weight || ldw < K)) || (grad_weight && (!x || ldx < K))))
        return fail(NEMO_ERR_INVALID, "nemo_linear_backward: null operand or a row stride shorter than the row");
    const size_t need = nemo_linear_backward_workspace(grad_y, ldg, x, ldx, weight, ldw, M, N, K, dtype, activation);
    if (workspace_bytes < need || (need && !workspace))
        return fail(NEMO_ERR_INVALID, "nemo_linear_backward: workspace of %zu bytes, %zu needed", workspace_bytes, need);
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
    if (grad_x && M > 0 && K > 0) {
        Operand W = N > 0 ? operand(dtype, weight, ldw, N, K, ws, st) : Operand{weight, ldw};
        const Shape s = shape_of(K, M, N, dtype);
        GemmArgs a = gemm_args(W, dz, K, M, N, s, ws);
        a.e = {alpha, 0.0f, ACT_NONE, nullptr, nullptr, 0, grad_x, K, nullptr, 0};
        a.e.vec = K % 4 == 0 && ((uintptr_t)grad_x & (4 * es - 1)) == 0;
        launch_gemm(dtype, a, true, false, st);
    }
    if (grad_weight && N > 0 && K > 0) {
        Operand X = M > 0 ? operand(dtype, x, ldx, M, K, ws, st) : Operand{x, ldx};
        const Shape s = shape_of(K, N, M, dtype);
        GemmArgs a = gemm_args(X, dz, K, N, M, s, ws);
        a.e = {alpha, 0.0f, ACT_NONE, nullptr, nullptr, 0, grad_weight, K, nullptr, 0};
        a.e.vec = K % 4 == 0 && ((uintptr_t)grad_weight & (4 * es - 1)) == 0;
        launch_gemm(dtype, a, true, true, st);
    }
    HIP_TRY(hipGetLastError());
    return NEMO_OK;
}
