// Entry points of the bank kernels (bank_forward.hip, bank_gradient.hip) and their small companions: the join of the parts of a row, what the
// gradient needs of a row, rows copied to where they start on 16 bytes.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/nemo_hip.h"
#include "bank_tiles.h"
#include "errors.h"

namespace nemo {

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
    int walk = 0;
    for (int i = 0; i < top; ++i) {
        Entry mine = no_entry();
        if (lane < n && walk < top) mine = {a.part_z[at * top + walk], a.part_place[at * top + walk]};
        const Entry e = wave_best(mine);
        if (mine.place == e.place && mine.z == e.z) ++walk;
        if (lane == 0) write_top(a.out, row, i, st, e);
    }
}

// What the gradients need of a row, as arrays over the rows; the rows behind the last, up to whole tiles, give nothing.
struct CoefArgs {
    const float *stats, *g_logp, *g_entropy, *g_lse;
    const long long* targets;
    float* coef;
    int rows, cols;
    bool join_m;
};
__device__ void write_coef(const CoefArgs& a, int row) {
    const int n = coef_rows(a.rows);
    if (row >= n) return;
    RowCoef k = {0.0f, kNoProbability, 0.0f, 0.0f, 0.0f, -1};
    if (row < a.rows) k = row_coef(a.stats, a.g_logp, a.g_entropy, a.g_lse, a.targets, row, a.cols);
    a.coef[K_M * n + row] = a.join_m ? k.m + k.log2_s : k.m;
    a.coef[K_LOG2_S * n + row] = k.log2_s;
    a.coef[K_C * n + row] = k.c;
    a.coef[K_G2 * n + row] = k.g2;
    a.coef[K_LOGP * n + row] = k.g_logp;
    a.coef[K_TARGET * n + row] = __builtin_bit_cast(float, k.target);
}

// Rows as the kernels take them: `rows_a` rows of one matrix, then `rows_b` of another (written behind them), channels padded with zeros to cp.
// bf16: one piece, a copy for rows that do not start on 16 bytes.  f32: three pieces a row, each the rounding of what the ones before leave; a
// value beyond bf16's largest is cut to it first, an infinity or NaN is the first piece alone.  Eight channels a thread.
// The first workgroups write the coefficients instead (a backward call's; none in a forward call): one launch for all that comes before.
struct RowsOf { const void* p; long ld; int rows; };
template <typename T>
__global__ __launch_bounds__(256) void bank_rows_kernel(RowsOf a, RowsOf b, int channels, int cp, bf16* out_a, bf16* out_b, CoefArgs k, uint32_t k_groups) {
    constexpr int NP = sizeof(T) == 4 ? 3 : 1;
    if (blockIdx.x < k_groups) return write_coef(k, (int)(blockIdx.x * 256 + threadIdx.x));
    const uint32_t per_row = cp / 8, id = (blockIdx.x - k_groups) * 256u + threadIdx.x;          // fewer than 2^31 threads: see check_bank
    const uint32_t r = id / per_row;
    const int c = (int)(id - r * per_row) * 8;
    if (r >= (uint32_t)(a.rows + b.rows)) return;
    const bool second = r >= (uint32_t)a.rows;
    const long row = second ? r - a.rows : r;
    const T* src = (const T*)(second ? b.p : a.p) + row * (second ? b.ld : a.ld) + c;
    bf16* dst = (second ? out_b : out_a) + row * (long)(NP * cp) + c;
    float v[8] = {};
    if (c + 8 <= channels) {
        const typename Loose<T, 8>::V t = load_loose<8>(src);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_f32(t[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < channels) v[i] = to_f32(src[i]);
    }
#pragma unroll
    for (int n = 0; n < NP; ++n) {
        bf16x8 piece;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float most = 3.3895313892515355e38f;
            float h = (float)(bf16)v[i];
            if (NP > 1 && n == 0 && __builtin_fabsf(v[i]) > most && __builtin_fabsf(v[i]) <= FLT_MAX) h = v[i] > 0.0f ? most : -most;
            piece[i] = (bf16)h;
            v[i] = __builtin_fabsf(h) <= FLT_MAX ? v[i] - h : 0.0f;
        }
        *(bf16x8*)(dst + n * cp) = piece;
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------
static size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }
static bool aligned_rows(const void* p, int64_t ld, int64_t cols, int es) {
    return ((uintptr_t)p & 15) == 0 && (ld * es) % 16 == 0 && (cols * es) % 16 == 0;
}
// Bytes of the rows' copy in the workspace.
static size_t rows_bytes(const void* p, int64_t ld, int64_t rows, int64_t cols, int dtype) {
    if (dtype == NEMO_BF16 && aligned_rows(p, ld, cols, 2)) return 0;
    return align256((size_t)rows * padded_channels((int)cols) * 2 * (dtype == NEMO_F32 ? 3 : 1));
}

// Parts of the other axis, at most 32: while the card is not full, parts down to `least` tiles, a workgroup a compute unit; beyond that
// `per_cu` workgroups a unit (what a kernel's registers leave room for), of at least four tiles.  Measured (a call in us, f32, 128 channels,
// parts of one tile / four): forward 17 rows of 643 11.3 / 17.1, 1000 of 1000 16.2 / 20.3, 4096 of 643 26.5 / 25.1; backward, whose parts
// are written out and joined, with two tiles / four / one: 128 of 1024 72 / 86 / 71, 1000 of 1000 81 / 88 / 90.
struct Parts { int parts, tiles; };
static Parts parts_of_bank(int64_t owners, int64_t others, int per_cu, int least) {
    const int64_t groups = owners > 0 ? (owners + 127) / 128 : 1, tiles = (others + 31) / 32;
    const int64_t few = std::min(256 / groups, tiles / least), many = std::min(256 * per_cu / groups, tiles / 4);
    const int64_t p = std::max<int64_t>(1, std::min<int64_t>(32, std::max(few, many)));
    const int64_t per = tiles > 0 ? (tiles + p - 1) / p : 1;
    return {(int)(tiles > 0 ? (tiles + per - 1) / per : 1), (int)per};
}
static Parts forward_parts(int64_t rows, int64_t cols, int cp, int dtype) {
    return parts_of_bank(rows, cols, dtype == NEMO_F32 ? (cp == 64 ? 3 : cp == 128 ? 2 : 1) : cp <= 128 ? 4 : 2, 1);
}
static Parts gradient_parts(int64_t owners, int64_t others, int cp, int dtype) {
    return parts_of_bank(owners, others, dtype == NEMO_F32 ? (cp == 64 ? 2 : 1) : cp <= 128 ? 2 : 1, 2);
}

// The state's form: 0 where it is kept of the scores, else what turns a product into its score in units of log 2 (with hardly any scale it would be
// inexact, with the largest ones infinite).
static float product_unit(const float* weights, float scale, int top) {
    const float s = scale < 0.0f ? -scale : scale;
    return weights || top > 0 || !(s >= 1.0e-30f && s <= 1.0e30f) ? 0.0f : s * kLog2e;
}

static int check_bank(const char* who, int64_t rows, int64_t cols, int64_t channels, int dtype, int top) {
    if (rows < 0 || cols < 0 || channels <= 0) return fail(NEMO_ERR_INVALID, "%s: bad size", who);
    if (dtype != NEMO_F32 && dtype != NEMO_BF16) return fail(NEMO_ERR_UNSUPPORTED, "%s: element type %d (takes f32 and bf16)", who, dtype);
    if (channels > 256) return fail(NEMO_ERR_UNSUPPORTED, "%s: %lld channels (takes up to 256)", who, (long long)channels);
    if (top < 0 || top > kMaxTop) return fail(NEMO_ERR_UNSUPPORTED, "%s: %d best entries (takes 0 to %d)", who, top, kMaxTop);
    if (rows >= (1LL << 24) || cols >= (1LL << 24)) return fail(NEMO_ERR_UNSUPPORTED, "%s: 2^24 rows or more", who);
    return NEMO_OK;
}

struct RowsIn { const bf16* p; int64_t ld; };
static void rows_in(int dtype, const void* features, int64_t ldf, int64_t rows, const void* bank, int64_t ldb, int64_t cols, int64_t channels,
                    char*& ws, hipStream_t st, const CoefArgs& k, RowsIn* f, RowsIn* b) {
    const int cp = padded_channels((int)channels);
    *f = {(const bf16*)features, ldf};
    *b = {(const bf16*)bank, ldb};
    const size_t bytes_f = rows_bytes(features, ldf, rows, channels, dtype), bytes_b = rows_bytes(bank, ldb, cols, channels, dtype);
    const int64_t ld_out = (int64_t)cp * (dtype == NEMO_F32 ? 3 : 1);
    if (bytes_f) *f = {(bf16*)ws, ld_out};
    if (bytes_b) *b = {(bf16*)(ws + bytes_f), ld_out};
    ws += bytes_f + bytes_b;
    const int na = bytes_f ? (int)rows : 0, nb = bytes_b ? (int)cols : 0;
    const unsigned k_groups = k.coef ? (unsigned)(coef_rows(k.rows) + 255) / 256 : 0;
    const unsigned wgs = k_groups + (unsigned)(((int64_t)(na + nb) * (cp / 8) + 255) / 256);
    if (wgs == 0) return;
    const RowsOf ra = {features, (long)ldf, na}, rb = {bank, (long)ldb, nb};
    if (dtype == NEMO_F32)
        hipLaunchKernelGGL((bank_rows_kernel<float>), dim3(wgs), dim3(256), 0, st, ra, rb, (int)channels, cp, (bf16*)f->p, (bf16*)b->p, k, k_groups);
    else
        hipLaunchKernelGGL((bank_rows_kernel<bf16>), dim3(wgs), dim3(256), 0, st, ra, rb, (int)channels, cp, (bf16*)f->p, (bf16*)b->p, k, k_groups);
}

}  // namespace nemo

using namespace nemo;

extern "C" size_t nemo_bank_log_probs_workspace(const void* features, int64_t ldf, const void* bank, int64_t ldb, int64_t rows, int64_t cols,
                                                int64_t channels, int32_t dtype, int32_t top) {
    if (rows <= 0 || cols < 0 || channels <= 0 || channels > 256 || top < 0 || top > kMaxTop) return 0;
    const Parts p = forward_parts(rows, cols, padded_channels((int)channels), dtype);
    return rows_bytes(features, ldf, rows, channels, dtype) + rows_bytes(bank, ldb, cols, channels, dtype) +
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
    if (need && ((uintptr_t)workspace & 15)) return fail(NEMO_ERR_INVALID, "nemo_bank_log_probs: the workspace must start on 16 bytes");
    hipStream_t st = (hipStream_t)stream;
    char* ws = (char*)workspace;
    RowsIn f, b;
    rows_in(dtype, features, ldf, rows, bank, ldb, cols, channels, ws, st, CoefArgs{}, &f, &b);
    const Parts p = forward_parts(rows, cols, padded_channels((int)channels), dtype);
    BankArgs a = {};
    a.own = f.p; a.ld_own = f.ld; a.n_own = (int)rows;
    a.other = b.p; a.ld_other = b.ld; a.n_other = (int)cols;
    a.channels = (int)(channels + 7) / 8 * 8;
    a.weights = weights; a.ldw = ldw; a.targets = (const long long*)targets; a.scale = scale;
    a.parts = p.parts; a.part_tiles = p.tiles;
    a.part_state = (float*)ws;
    ws += align256((size_t)3 * 2 * p.parts * rows * 4);
    a.part_z = (float*)ws;
    ws += align256((size_t)2 * p.parts * rows * top * 4);
    a.part_place = (int*)ws;
    ws += align256((size_t)2 * p.parts * rows * top * 4);
    a.z_target = (float*)ws;
    a.out = {out_logp, out_entropy, out_lse, out_stats, out_top_logp, (long long*)out_top_index, top, product_unit(weights, scale, top)};
    if (dtype == NEMO_F32) launch_bank_forward<float>(a, st);
    else launch_bank_forward<bf16>(a, st);
    hipLaunchKernelGGL(bank_join_kernel, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, a);
    HIP_TRY(hipGetLastError());
    return NEMO_OK;
}

extern "C" size_t nemo_bank_log_probs_backward_workspace(const void* features, int64_t ldf, const void* bank, int64_t ldb, int64_t rows,
                                                         int64_t cols, int64_t channels, int32_t dtype) {
    if (rows <= 0 || cols <= 0 || channels <= 0 || channels > 256) return 0;
    const int cp = padded_channels((int)channels);
    const Parts pf = gradient_parts(rows, cols, cp, dtype), pb = gradient_parts(cols, rows, cp, dtype);
    const size_t bf = pf.parts > 1 ? (size_t)pf.parts * rows * cp * 4 : 0, bb = pb.parts > 1 ? (size_t)pb.parts * cols * cp * 4 : 0;
    return rows_bytes(features, ldf, rows, channels, dtype) + rows_bytes(bank, ldb, cols, channels, dtype) + align256((size_t)K_COUNT * coef_rows(rows) * 4) +
           align256(bf > bb ? bf : bb);
}

extern "C" int nemo_bank_log_probs_backward(const void* features, int64_t ldf, const void* bank, int64_t ldb, const float* weights, int64_t ldw,
                                            const int64_t* targets, const float* stats, const float* g_logp, const float* g_entropy,
                                            const float* g_lse, int64_t rows, int64_t cols, int64_t channels, int32_t dtype, float scale,
                                            int32_t top, void* grad_features, void* grad_bank, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check_bank("nemo_bank_log_probs_backward", rows, cols, channels, dtype, top);
    if (rc) return rc;
    if (rows == 0 || cols == 0) return NEMO_OK;
    if (!features || !bank || !targets || !stats) return fail(NEMO_ERR_INVALID, "nemo_bank_log_probs_backward: null argument");
    if (ldf < channels || ldb < channels || (weights && ldw != 0 && ldw < cols))
        return fail(NEMO_ERR_INVALID, "nemo_bank_log_probs_backward: a row stride shorter than the row");
    if (weights && ldw > (1LL << 27)) return fail(NEMO_ERR_UNSUPPORTED, "nemo_bank_log_probs_backward: weights with rows more than 2^27 apart");
    if ((uintptr_t)stats & 15) return fail(NEMO_ERR_INVALID, "nemo_bank_log_probs_backward: stats must start on 16 bytes");
    const size_t need = nemo_bank_log_probs_backward_workspace(features, ldf, bank, ldb, rows, cols, channels, dtype);
    if (workspace_bytes < need || (need && !workspace))
        return fail(NEMO_ERR_INVALID, "nemo_bank_log_probs_backward: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    if (need && ((uintptr_t)workspace & 15)) return fail(NEMO_ERR_INVALID, "nemo_bank_log_probs_backward: the workspace must start on 16 bytes");
    hipStream_t st = (hipStream_t)stream;
    char* ws = (char*)workspace;
    const float unit = product_unit(weights, scale, top);
    float* coef = (float*)ws;
    ws += align256((size_t)K_COUNT * coef_rows(rows) * 4);
    RowsIn f, b;
    rows_in(dtype, features, ldf, rows, bank, ldb, cols, channels, ws, st,
            {stats, g_logp, g_entropy, g_lse, (const long long*)targets, coef, (int)rows, (int)cols, unit != 0.0f && dtype == NEMO_BF16}, &f, &b);
    const int cp = padded_channels((int)channels);
    for (int own_bank = 0; own_bank < 2; ++own_bank) {
        void* grad = own_bank ? grad_bank : grad_features;
        if (!grad) continue;
        const RowsIn own = own_bank ? b : f, other = own_bank ? f : b;
        const int64_t n_own = own_bank ? cols : rows, n_other = own_bank ? rows : cols;
        const Parts p = gradient_parts(n_own, n_other, cp, dtype);
        BankArgs a = {};
        a.own = own.p; a.ld_own = own.ld; a.n_own = (int)n_own;
        a.other = other.p; a.ld_other = other.ld; a.n_other = (int)n_other;
        a.channels = (int)(channels + 7) / 8 * 8;
        a.grad_channels = (int)channels;
        a.weights = weights; a.ldw = ldw; a.targets = (const long long*)targets; a.scale = scale;
        a.parts = p.parts; a.part_tiles = p.tiles;
        a.out.k = unit;
        a.coef = coef; a.partial = (float*)ws; a.grad = grad;
        if (dtype == NEMO_F32) launch_bank_gradient<float>(a, own_bank, st);
        else launch_bank_gradient<bf16>(a, own_bank, st);
    }
    HIP_TRY(hipGetLastError());
    return NEMO_OK;
}
