// Log probabilities of given places of rows of logits, with entropy, log-sum-exp and the best entries; and the gradient of the logits.
//
// Both directions read each logit once.  Forward: a wave or a workgroup of four waves takes a row (or one of its parts), a lane takes 16 bytes
// at a time, four of them under way at once, and keeps the state of softmax_state.h; states are joined across lanes, waves and parts in
// a fixed order.  For the best entries a lane keeps its best one; a wave takes the best of its lanes k times, and the lane it came from
// looks through its share of the row again for the next one, together with the whole wave.  Waves' lists, sorted, are merged.
// Rows need not be aligned: 16-byte accesses at any element are in order on this hardware.
//
// Measured.  4096 x 100003 bf16 (819 MB): forward 213 us, 3.9 TB/s, the vector units 71 % busy (7.5 instructions a score, one of them the
// exponential, four times as long); backward 352 us for as much read and written, 4.7 TB/s, what a copy reaches.  8000 x 13416 f32 with the five
// best (429 MB): 91 us, 4.7 TB/s; with weights for every place, without a list (858 MB): 170 us, 5.1 TB/s.  One row of 1118 f32 with the five
// best: 7.5 us, the latency of a launch, of a few dependent loads and of five selections.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <algorithm>
#include <type_traits>

#include "../../include/nemo_hip.h"
#include "errors.h"
#include "softmax_state.h"

namespace nemo {

struct LogProbArgs {
    const void* logits;
    long ld;
    const float* weights;          // null, or rows with stride ldw (0: one row for all)
    long ldw;
    const long long* targets;
    long rows;
    int cols;
    float scale;
    int parts, part_cols;          // columns of a part, whole chunks
    float* part_state;             // [3][parts][rows]
    float* part_z;                 // [parts][rows][top]
    int* part_place;
    RowOut out;
};

template <typename T> struct Chunk {
    static constexpr int N = 16 / (int)sizeof(T);
    typename Loose<T, N>::V v;
    f32x4 w[N / 4];
    // Logits and, with W, weights of N places from column j on, all of which exist.
    template <bool W> __device__ inline void load(const T* row, const float* weights, int j) {
        v = load_loose<N>(row + j);
        if (W) {
#pragma unroll
            for (int q = 0; q < N / 4; ++q) w[q] = load_loose<4>(weights + j + 4 * q);
        }
    }
    template <bool W> __device__ inline void scores(float scale, float* z) const {
#pragma unroll
        for (int i = 0; i < N; ++i) z[i] = W ? score(to_f32(v[i]), scale, w[i / 4][i % 4]) : score(to_f32(v[i]), scale);
    }
};

// Scores of up to N places from column j on; places at or beyond `end` are -inf.
template <bool W, typename T>
__device__ inline void chunk_scores(const T* row, const float* w, float scale, int j, int end, float z[Chunk<T>::N]) {
    constexpr int N = Chunk<T>::N;
    if (j + N <= end) {
        Chunk<T> c;
        c.template load<W>(row, w, j);
        c.template scores<W>(scale, z);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            z[i] = j + i >= end ? neg_inf() : W ? score(to_f32(row[j + i]), scale, w[j + i]) : score(to_f32(row[j + i]), scale);
    }
}

// N scores into a state: one rescaling for all of them.
template <int N>
__device__ inline void add_scores(SoftmaxState& a, const float* z) {
    float m = a.m;
#pragma unroll
    for (int i = 0; i < N; ++i) m = fmaxf(m, z[i]);
    raise(a, m, kLog2e);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float x = (z[i] - m) * kLog2e, e = exp2_fast(x);
        a.s += e;
        a.t += e * fmaxf(x, -200.0f);                                  // 0 where e is 0, also where x is -inf
    }
}

// The same with fewer operations: x = fma(z, log2 e, -u) against the rounded u = m log2 e, which drops out when the state is turned into the
// other form.  Scores beyond 2^126 and, without LEFT_OUT, scores of -inf make s 0 or s or t NaN; the wave then goes through its share again.
// (4096 x 100003 bf16: 224 us with the other form, of which the vector units were busy 150; 8000 x 13416 f32 with a list 99 against 91.)
// Off from 64 bits by 1.7e-7 of the results' norm at 8000 x 13416, the same operations one by one in 32 bits by 7e-8.
struct QuickState {
    float m = -0x1p126f, u = -0x1p126f * kLog2e, s = 0.0f, t = 0.0f;       // u exact: a lane without scores stays 0
    template <int N, bool LEFT_OUT> __device__ inline void add(const float* z) {
#pragma unroll
        for (int i = 0; i < N; ++i) m = fmaxf(m, z[i]);
        const float up = m * kLog2e, d = u - up, f = exp2_fast(d);
        t = f * (t + fmaxf(d, -1.0e4f) * s);
        s *= f;
        u = up;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float x = __builtin_fmaf(z[i], kLog2e, -u), e = exp2_fast(x);
            s += e;
            t += e * (LEFT_OUT ? fmaxf(x, -200.0f) : x);
        }
    }
    __device__ inline SoftmaxState state() const {
        const float d = -__builtin_fmaf(m, kLog2e, -u), f = exp2_fast(d);
        return {m, s * f, f * (t + d * s)};
    }
};

// WAVES waves a row, ROWS rows a workgroup (WAVES * ROWS = 4).
template <typename T, int WAVES, bool TOP, bool W>
__global__ __launch_bounds__(256) void log_probs_kernel(LogProbArgs a) {
    constexpr int N = Chunk<T>::N, ROWS = 4 / WAVES, LANES = 64 * WAVES, UNROLL = 4;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int part = (int)(blockIdx.x % a.parts);
    const long row = (long)(blockIdx.x / a.parts) * ROWS + wave / WAVES;
    const bool live = row < a.rows;                                    // all four waves of a workgroup meet at the barriers below
    const int wr = wave % WAVES;
    const int begin = part * a.part_cols, end = min(a.cols, begin + a.part_cols);
    const T* logits = (const T*)a.logits + (live ? row : 0) * a.ld;
    const float* w = W ? a.weights + (live ? row : 0) * a.ldw : nullptr;
    const int first = begin + (wr * 64 + lane) * N;
    QuickState quick;
    Entry best = no_entry();
    if (live) {
        // places rise within a lane: the first of equal ones stays
        auto keep = [&](float z, int place) __attribute__((always_inline)) {
            if (TOP && z > best.z) best = {z, place};
        };
        // UNROLL loads under way at once
        int j = first;
        for (; j + (UNROLL - 1) * LANES * N + N <= end; j += UNROLL * LANES * N) {
            Chunk<T> c[UNROLL];
            float z[UNROLL * N];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) c[u].template load<W>(logits, w, j + u * LANES * N);
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) c[u].template scores<W>(a.scale, z + u * N);
            quick.add<UNROLL * N, W>(z);
#pragma unroll
            for (int i = 0; i < UNROLL * N; ++i) keep(z[i], j + i / N * (LANES * N) + i % N);
        }
        for (; j < end; j += LANES * N) {
            float z[N];
            chunk_scores<W>(logits, w, a.scale, j, end, z);
            quick.add<N, true>(z);
#pragma unroll
            for (int i = 0; i < N; ++i) keep(z[i], j + i);
        }
    }
    SoftmaxState st = wave_join(quick.state(), kLog2e);
    if (live && !(st.s > 0.0f && st.t == st.t)) {                      // nothing counted, or a value that QuickState does not take
        st = empty_state();
        for (int j = first; j < end; j += LANES * N) {
            float z[N];
            chunk_scores<W>(logits, w, a.scale, j, end, z);
            add_scores<N>(st, z);
        }
        st = wave_join(st, kLog2e);
    }
    __shared__ SoftmaxState s_state[4];
    __shared__ Entry s_top[TOP ? 4 : 1][kMaxTop];
    const int top = a.out.top;
    if (TOP && live) {
        for (int i = 0; i < top; ++i) {
            const Entry e = wave_best(best);
            if (lane == 0) s_top[wave][i] = e;
            if (i + 1 == top || e.z == neg_inf()) {
                if (lane == 0)
                    for (int r = i + 1; r < top; ++r) s_top[wave][r] = no_entry();
                break;
            }
            // the owner's share again: the best entry behind e
            const int owner = ((e.place - begin) / N) & 63;
            Entry next = no_entry();
            for (int j = begin + (wr * 64 + owner) * N + lane * LANES * N; j < end; j += 64 * LANES * N) {
                float z[N];
                chunk_scores<W>(logits, w, a.scale, j, end, z);
#pragma unroll
                for (int q = 0; q < N; ++q) {
                    const Entry c = {z[q], j + q};
                    if (ahead(e, c) && ahead(c, next)) next = c;
                }
            }
            next = wave_best(next);
            if (lane == owner) best = next;
        }
    }
    if (WAVES > 1) {
        if (lane == 0) s_state[wave] = st;
        __syncthreads();
        if (wr != 0 || !live) return;
        st = s_state[wave];
#pragma unroll
        for (int i = 1; i < WAVES; ++i) st = join_states(st, s_state[wave + i], kLog2e);
    } else {
        if (TOP) __syncthreads();
        if (!live) return;
    }
    // the wave that is left merges the waves' lists: lane i < WAVES walks list i
    if (a.parts > 1) {
        const size_t at = (size_t)part * a.rows + row, plane = (size_t)a.parts * a.rows;
        if (lane == 0) {
            a.part_state[at] = st.m;
            a.part_state[plane + at] = st.s;
            a.part_state[2 * plane + at] = st.t;
        }
    } else if (lane == 0) {
        const long long t = a.targets[row];
        float zt = 0.0f;
        if (t >= 0 && t < a.cols) zt = W ? score(to_f32(logits[t]), a.scale, w[t]) : score(to_f32(logits[t]), a.scale);
        write_row(a.out, row, st, t, a.cols, zt);
    }
    if (TOP) {
        int walk = 0;
        for (int i = 0; i < top; ++i) {
            const Entry mine = lane < WAVES && walk < top ? s_top[wave + lane][walk] : no_entry();
            const Entry e = wave_best(mine);
            if (mine.place == e.place && mine.z == e.z) ++walk;
            if (lane == 0) {
                if (a.parts > 1) {
                    const size_t at = ((size_t)part * a.rows + row) * top + i;
                    a.part_z[at] = e.z;
                    a.part_place[at] = e.place;
                } else {
                    write_top(a.out, row, i, st, e);
                }
            }
        }
    }
}

// Joins the parts of a row (at most 64): a wave a row, a lane a part.
template <typename T>
__global__ __launch_bounds__(256) void log_probs_join_kernel(LogProbArgs a) {
    const int lane = threadIdx.x & 63;
    const long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= a.rows) return;
    const size_t at = (size_t)lane * a.rows + row, plane = (size_t)a.parts * a.rows;
    SoftmaxState st = empty_state();
    if (lane < a.parts) st = {a.part_state[at], a.part_state[plane + at], a.part_state[2 * plane + at]};
    st = wave_join(st, kLog2e);
    if (lane == 0) {
        const long long t = a.targets[row];
        float zt = 0.0f;
        if (t >= 0 && t < a.cols) {
            const float x = to_f32(((const T*)a.logits)[row * a.ld + t]);
            zt = a.weights ? score(x, a.scale, a.weights[row * a.ldw + t]) : score(x, a.scale);
        }
        write_row(a.out, row, st, t, a.cols, zt);
    }
    int walk = 0;
    for (int i = 0; i < a.out.top; ++i) {
        Entry mine = no_entry();
        if (lane < a.parts && walk < a.out.top) mine = {a.part_z[at * a.out.top + walk], a.part_place[at * a.out.top + walk]};
        const Entry e = wave_best(mine);
        if (mine.place == e.place && mine.z == e.z) ++walk;
        if (lane == 0) write_top(a.out, row, i, st, e);
    }
}

// d logits: 256 threads x 16 bytes a step of a row.
template <typename T, bool W>
__global__ __launch_bounds__(256) void log_probs_backward_kernel(LogProbArgs a, const float* stats, const float* g_logp, const float* g_entropy,
                                                                 const float* g_lse, T* grad) {
    constexpr int N = Chunk<T>::N;
    for (long row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const RowCoef k = row_coef(stats, g_logp, g_entropy, g_lse, a.targets, row, a.cols);
        const T* logits = (const T*)a.logits + row * a.ld;
        const float* w = W ? a.weights + row * a.ldw : nullptr;
        T* out = grad + row * (long)a.cols;
#pragma unroll 2
        for (int j = (blockIdx.x * 256 + threadIdx.x) * N; j < a.cols; j += gridDim.x * 256 * N) {
            float z[N];
            chunk_scores<W>(logits, w, a.scale, j, a.cols, z);
            typename Loose<T, N>::V c;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                float d = prob_gradient(__builtin_fmaf(z[i] - k.m, kLog2e, -k.log2_s), k.c, k.g2);
                if (j + i == k.target) d += k.g_logp;
                if (z[i] == neg_inf()) d = 0.0f;
                c[i] = from_f32<T>(a.scale * d);
            }
            if (j + N <= a.cols) {
                store_loose<N>(out + j, c);
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (j + i < a.cols) out[j + i] = c[i];
            }
        }
    }
}

static size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

// Parts of a row where there are too few rows to fill the device: four workgroups a compute unit, at least 8192 columns a part, rows of at least
// four of them (the join is a launch).  Measured in us, f32, parts of 2048 / 8192 / 32768 columns: 16 x 20000 6.3 / 6.7 / 5.9 (one part),
// 128 x 16384 6.8 / 6.6 / 5.0 (one part), 16 x 130000 7.0 / 6.7 / 10.1, 1 x 130000 with the five best 11.9 / 12.5 / 16.1.
static int parts_of(int64_t rows, int64_t cols) {
    if (rows <= 0 || cols < 4 * 8192) return 1;
    return (int)std::max<int64_t>(1, std::min<int64_t>(64, std::min(1024 / rows, cols / 8192)));
}

static int check_log_probs(const char* who, int64_t rows, int64_t cols, int dtype, int top) {
    if (rows < 0 || cols < 0) return fail(NEMO_ERR_INVALID, "%s: negative size", who);
    if (dtype != NEMO_F32 && dtype != NEMO_BF16 && dtype != NEMO_F16) return fail(NEMO_ERR_INVALID, "%s: unknown element type %d", who, dtype);
    if (top < 0 || top > kMaxTop) return fail(NEMO_ERR_UNSUPPORTED, "%s: %d best entries (takes 0 to %d)", who, top, kMaxTop);
    if (rows >= (1LL << 24) || cols > (1LL << 30)) return fail(NEMO_ERR_UNSUPPORTED, "%s: more than 2^24 - 1 rows or 2^30 columns", who);
    return NEMO_OK;
}

template <typename T>
static void launch_log_probs(const LogProbArgs& a, hipStream_t st) {
    // One wave a row where there is a row for every SIMD and it is no longer than 32 KB; else four waves a row.  Measured in us, four waves / one:
    // f32 2048 x 500 5.4 / 4.0, 8000 x 1118 with the five best 43.7 / 20.4, 32768 x 4000 with them 192 / 123, 8000 x 8000 with them 64 / 60, 8000 x 13416
    // with them 93 / 95, 16000 x 16384 183 / 194, 1024 x 8000 8.2 / 9.0; bf16 8000 x 13416 with the five best 80 / 56, 4096 x 60000 95 / 97.
    const bool narrow = a.rows >= 1024 && (int64_t)a.cols * (int64_t)sizeof(T) <= 32768;
    const unsigned wgs = narrow ? (unsigned)((a.rows + 3) / 4) : (unsigned)(a.rows * a.parts);
    auto launch = [&](auto top, auto weighted) {
        constexpr bool TOP = decltype(top)::value, W = decltype(weighted)::value;
        if (narrow) hipLaunchKernelGGL((log_probs_kernel<T, 1, TOP, W>), dim3(wgs), dim3(256), 0, st, a);
        else hipLaunchKernelGGL((log_probs_kernel<T, 4, TOP, W>), dim3(wgs), dim3(256), 0, st, a);
    };
    const std::true_type yes;
    const std::false_type no;
    if (a.out.top) a.weights ? launch(yes, yes) : launch(yes, no);
    else a.weights ? launch(no, yes) : launch(no, no);
    if (a.parts > 1) hipLaunchKernelGGL((log_probs_join_kernel<T>), dim3((unsigned)((a.rows + 3) / 4)), dim3(256), 0, st, a);
}

}  // namespace nemo

using namespace nemo;

extern "C" size_t nemo_log_probs_workspace(int64_t rows, int64_t cols, int32_t top) {
    const int parts = parts_of(rows, cols);
    if (rows <= 0 || parts <= 1 || top < 0 || top > kMaxTop) return 0;
    return align256((size_t)3 * parts * rows * 4) + align256((size_t)parts * rows * top * 4) * 2;
}

extern "C" int nemo_log_probs(const void* logits, int64_t ld, const float* weights, int64_t ldw, const int64_t* targets, int64_t rows,
                              int64_t cols, int32_t dtype, float scale, int32_t top, float* out_logp, float* out_entropy, float* out_lse,
                              float* out_stats, float* out_top_logp, int64_t* out_top_index, void* workspace, size_t workspace_bytes,
                              void* stream) {
    int rc = check_log_probs("nemo_log_probs", rows, cols, dtype, top);
    if (rc) return rc;
    if (rows == 0) return NEMO_OK;
    if (!targets || (cols > 0 && !logits) || (top > 0 && (!out_top_logp || !out_top_index)))
        return fail(NEMO_ERR_INVALID, "nemo_log_probs: null argument");
    if (ld < cols || (weights && ldw != 0 && ldw < cols)) return fail(NEMO_ERR_INVALID, "nemo_log_probs: a row stride shorter than the row");
    if ((uintptr_t)out_stats & 15) return fail(NEMO_ERR_INVALID, "nemo_log_probs: out_stats must start on 16 bytes");
    const size_t need = nemo_log_probs_workspace(rows, cols, top);
    if (workspace_bytes < need || (need && !workspace))
        return fail(NEMO_ERR_INVALID, "nemo_log_probs: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    if (need && ((uintptr_t)workspace & 15)) return fail(NEMO_ERR_INVALID, "nemo_log_probs: the workspace must start on 16 bytes");
    LogProbArgs a = {};
    a.logits = logits; a.ld = ld; a.weights = weights; a.ldw = ldw; a.targets = (const long long*)targets;
    a.rows = rows; a.cols = (int)cols; a.scale = scale;
    a.parts = parts_of(rows, cols);
    a.part_cols = (int)(((cols + a.parts - 1) / a.parts + 7) / 8 * 8);
    if (a.parts > 1) {
        char* ws = (char*)workspace;
        a.part_state = (float*)ws;
        ws += align256((size_t)3 * a.parts * rows * 4);
        a.part_z = (float*)ws;
        a.part_place = (int*)(ws + align256((size_t)a.parts * rows * top * 4));
    }
    a.out = {out_logp, out_entropy, out_lse, out_stats, out_top_logp, (long long*)out_top_index, top, 0.0f};
    hipStream_t st = (hipStream_t)stream;
    if (dtype == NEMO_F32) launch_log_probs<float>(a, st);
    else if (dtype == NEMO_BF16) launch_log_probs<bf16>(a, st);
    else launch_log_probs<f16>(a, st);
    HIP_TRY(hipGetLastError());
    return NEMO_OK;
}

template <typename T>
static void launch_log_probs_backward(const LogProbArgs& a, const float* stats, const float* g_logp, const float* g_entropy, const float* g_lse,
                                      void* grad, hipStream_t st) {
    const int per = 256 * Chunk<T>::N;
    const int slabs = (a.cols + 2 * per - 1) / (2 * per);              // two steps a thread
    const dim3 grid(slabs, (unsigned)(a.rows < 65535 ? a.rows : 65535));
    if (a.weights)
        hipLaunchKernelGGL((log_probs_backward_kernel<T, true>), grid, dim3(256), 0, st, a, stats, g_logp, g_entropy, g_lse, (T*)grad);
    else
        hipLaunchKernelGGL((log_probs_backward_kernel<T, false>), grid, dim3(256), 0, st, a, stats, g_logp, g_entropy, g_lse, (T*)grad);
}

extern "C" int nemo_log_probs_backward(const void* logits, int64_t ld, const float* weights, int64_t ldw, const int64_t* targets,
                                       const float* stats, const float* g_logp, const float* g_entropy, const float* g_lse, int64_t rows,
                                       int64_t cols, int32_t dtype, float scale, void* grad_logits, void* stream) {
    int rc = check_log_probs("nemo_log_probs_backward", rows, cols, dtype, 0);
    if (rc) return rc;
    if (rows == 0 || cols == 0) return NEMO_OK;
    if (!logits || !targets || !stats || !grad_logits) return fail(NEMO_ERR_INVALID, "nemo_log_probs_backward: null argument");
    if (ld < cols || (weights && ldw != 0 && ldw < cols)) return fail(NEMO_ERR_INVALID, "nemo_log_probs_backward: a row stride shorter than the row");
    if ((uintptr_t)stats & 15) return fail(NEMO_ERR_INVALID, "nemo_log_probs_backward: stats must start on 16 bytes");
    LogProbArgs a = {};
    a.logits = logits; a.ld = ld; a.weights = weights; a.ldw = ldw; a.targets = (const long long*)targets;
    a.rows = rows; a.cols = (int)cols; a.scale = scale; a.parts = 1;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == NEMO_F32) launch_log_probs_backward<float>(a, stats, g_logp, g_entropy, g_lse, grad_logits, st);
    else if (dtype == NEMO_BF16) launch_log_probs_backward<bf16>(a, stats, g_logp, g_entropy, g_lse, grad_logits, st);
    else launch_log_probs_backward<f16>(a, stats, g_logp, g_entropy, g_lse, grad_logits, st);
    HIP_TRY(hipGetLastError());
    return NEMO_OK;
}
