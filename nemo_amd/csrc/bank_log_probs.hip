// The log probabilities of log_probs.hip straight from features and bank, z = scale <feature, bank row> - weight, without ever writing the
// [rows, bank rows] matrix: owners (bank_tiles.h) are the feature rows, others the bank; the softmax state of a row and its best entries live
// in the lane, no exchange until the end.  The bank is split where there are too few feature rows to fill the device; states and lists of the
// parts, and of the two lanes of a row, are joined by a second kernel in a fixed order.  The gradients are in bank_gradient.hip.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/nemo_hip.h"
#include "bank_tiles.h"
#include "errors.h"

namespace nemo {

// Puts v into the list, ordered by v * order (the score; a score is not smaller where the product is not, but may be equal).  Places arrive
// in rising order, so an equal score goes behind those already there.
template <int TOP>
__device__ inline void insert(float (&tv)[TOP], int (&tp)[TOP], float v, int place, float order) {
    const float z = v * order;
#pragma unroll
    for (int i = TOP - 1; i >= 0; --i) {
        const bool above = z > tv[i] * order;
        const bool shift = i > 0 && z > tv[i > 0 ? i - 1 : 0] * order;
        if (above) {
            tv[i] = shift ? tv[i > 0 ? i - 1 : 0] : v;
            tp[i] = shift ? tp[i > 0 ? i - 1 : 0] : place;
        }
    }
}

// GENERAL: with weights, or with a scale of 0; see softmax_state.h for the two forms of the state.  The sign of the scale goes into the
// owners' fragments where the state is kept of the products.
template <typename T, int CP, int TOP, bool GENERAL>
__global__ __launch_bounds__(256, CP * sizeof(T) >= 1024 ? 1 : 2) void bank_forward_kernel(BankArgs a) {
    constexpr int BJ = Tile<T, CP>::ROWS, NT = TOP > 0 ? TOP : 1;
    __shared__ __attribute__((aligned(16))) char lds0[Tile<T, CP>::BYTES];
    __shared__ __attribute__((aligned(16))) char lds1[Tile<T, CP>::BYTES];
    __shared__ int s_again;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 5;
    const int part = (int)(blockIdx.x % a.parts);
    const int own0 = (int)(blockIdx.x / a.parts) * 128 + wave * 32, row = own0 + (lane & 31);
    const bool live = row < a.n_own;
    u32x4 q[CP / Wide<T>::KF];
    own_fragments<T, CP>(q, a, own0, lane, !GENERAL && a.scale < 0.0f);
    const float* w = a.weights ? a.weights + (live ? row : 0) * a.ldw : nullptr;
    const long long tl = live ? a.targets[row] : -1;
    const int target = tl >= 0 && tl < a.n_other ? (int)tl : -1;
    const float scale = GENERAL ? a.scale : __builtin_fabsf(a.scale);
    const float k = a.out.k, order = GENERAL ? 1.0f : scale;
    SoftmaxState st;
    float tv[NT];
    int tp[NT];

    // SAFE: also right where a difference of two products is beyond the range of f32
    auto consume = [&](const char* lds, int j_tile, auto safe_tag) __attribute__((always_inline)) {
        constexpr bool SAFE = decltype(safe_tag)::value || GENERAL;
#pragma unroll
        for (int s = 0; s < BJ / 32; ++s) {
            const int j0 = j_tile + s * 32;
            float wv[16];
            if (GENERAL && w) row_weights(wv, w, j0, g, a.n_other);
            const f32x16_t acc = products<T, CP>(lds, s * 32, q, lane);
            float v[16];                                               // products, or scores if GENERAL
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = !GENERAL ? acc[i] : w ? score(acc[i], scale, wv[i]) : score(acc[i], scale);
            const int left = a.n_other - j0 - 4 * g;                   // registers whose row 8 b + i is at least this are beyond the end
            const bool tail = j0 + 32 > a.n_other;
            if (tail) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (8 * (i >> 2) + (i & 3) >= left) v[i] = neg_inf();
            }
            float peak = v[0];
#pragma unroll
            for (int i = 1; i < 16; ++i) peak = fmaxf(peak, v[i]);
            const float m = GENERAL ? peak : k * peak;
            if (__any(m > st.m)) raise(st, fmaxf(st.m, m), GENERAL ? kLog2e : 1.0f);
            if (SAFE || tail) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float x = GENERAL ? (v[i] - st.m) * kLog2e : __builtin_fmaf(k, v[i], -st.m), e = exp2_fast(x);
                    st.s += e;
                    st.t += e * fmaxf(x, -200.0f);                     // 0 where e is 0, also where x is -inf
                }
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float x = __builtin_fmaf(k, v[i], -st.m), e = exp2_fast(x);
                    st.s += e;
                    st.t += e * x;
                }
            }
            if (__any(target >= j0 && target < j0 + 32)) {
                const int at = target - j0 - 4 * g;
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (at == 8 * (i >> 2) + (i & 3)) a.z_target[row] = v[i];
            }
            if (TOP > 0) {
                if (__any(peak * order > tv[NT - 1] * order)) {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (__any(v[i] * order > tv[NT - 1] * order)) insert(tv, tp, v[i], j0 + 8 * (i >> 2) + 4 * g + (i & 3), order);
                }
            }
        }
    };
    const int tiles = (a.n_other + BJ - 1) / BJ;
    const int t0 = part * a.part_tiles, t1 = min(tiles, t0 + a.part_tiles);
    const T* other = (const T*)a.other;
    auto pass = [&](auto safe_tag) __attribute__((always_inline)) {
        st = empty_state();
#pragma unroll
        for (int i = 0; i < NT; ++i) { tv[i] = neg_inf(); tp[i] = kNoPlace; }
        if (t0 < t1) stage_rows<T, CP>(lds0, other, a.ld_other, t0 * BJ, a.n_other, a.channels, wave, lane);
        for (int t = t0; t < t1; t += 2) {
            __syncthreads();
            if (t + 1 < t1) stage_rows<T, CP>(lds1, other, a.ld_other, (t + 1) * BJ, a.n_other, a.channels, wave, lane);
            consume(lds0, t * BJ, safe_tag);
            if (t + 1 >= t1) break;
            __syncthreads();
            if (t + 2 < t1) stage_rows<T, CP>(lds0, other, a.ld_other, (t + 2) * BJ, a.n_other, a.channels, wave, lane);
            consume(lds1, (t + 1) * BJ, safe_tag);
        }
    };
    pass(std::false_type{});
    if (!GENERAL) {
        // 0 times the infinity that such a difference is would have spoilt t alone
        if (threadIdx.x == 0) s_again = 0;
        __syncthreads();
        if (st.t != st.t && st.s == st.s) s_again = 1;
        __syncthreads();
        if (s_again) pass(std::true_type{});
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
    st = wave_join(st, state_unit(a.out));
    if (lane == 0) {
        const long long t = a.targets[row];
        write_row(a.out, row, st, t, a.n_other, t >= 0 && t < a.n_other ? a.z_target[row] : 0.0f);
    }
    const float order = a.out.k == 0.0f ? 1.0f : __builtin_fabsf(a.scale);
    int walk = 0;
    for (int i = 0; i < top; ++i) {
        float v = neg_inf();
        Entry mine = no_entry();
        if (lane < n && walk < top) {
            v = a.part_z[at * top + walk];
            mine = {v * order, a.part_place[at * top + walk]};
        }
        const Entry e = wave_best(mine);
        const bool owner = mine.place == e.place && e.place != kNoPlace;
        if (owner) ++walk;
        if (owner || (e.place == kNoPlace && lane == 0)) write_top(a.out, row, i, st, {v, e.place});
    }
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

// The state's form: 0 with weights (or hardly any scale), else what turns a product into its score in units of log 2.
static float product_unit(const float* weights, float scale) {
    const float s = scale < 0.0f ? -scale : scale;
    return weights || !(s >= 1.0e-30f) ? 0.0f : s * kLog2e;
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
    const bool general = a.out.k == 0.0f;
    if (top == 0) {
        if (general) hipLaunchKernelGGL((bank_forward_kernel<T, CP, 0, true>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((bank_forward_kernel<T, CP, 0, false>), grid, dim3(256), 0, st, a);
    } else if (top <= 5) {
        if (general) hipLaunchKernelGGL((bank_forward_kernel<T, CP, 5, true>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((bank_forward_kernel<T, CP, 5, false>), grid, dim3(256), 0, st, a);
    } else {
        if (general) hipLaunchKernelGGL((bank_forward_kernel<T, CP, 16, true>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((bank_forward_kernel<T, CP, 16, false>), grid, dim3(256), 0, st, a);
    }
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
    a.out = {out_logp, out_entropy, out_lse, out_stats, out_top_logp, (long long*)out_top_index, top, product_unit(weights, scale)};
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
    return pack_bytes(features, ldf, rows, channels, dtype) + pack_bytes(bank, ldb, cols, channels, dtype) + align256((size_t)K_COUNT * coef_rows(rows) * 4) +
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
    ws += align256((size_t)K_COUNT * coef_rows(rows) * 4);
    const float unit = product_unit(weights, scale);
    launch_bank_coef(stats, g_logp, g_entropy, g_lse, (const long long*)targets, (int)rows, (int)cols, coef, unit != 0.0f && dtype == NEMO_BF16, st);
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
        a.out.k = unit;
        a.coef = coef; a.partial = (float*)ws; a.grad = grad;
        launch_bank_gradient(a, dtype, own_bank, st);
    }
    HIP_TRY(hipGetLastError());
    return NEMO_OK;
}
