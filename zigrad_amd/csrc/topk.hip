// The k largest of a row, and the loss of a student against a teacher's k largest logits.
#include "reduce_device.h"

namespace zg {

// A float as an unsigned number of the same order: -0 like +0, every NaN above +inf.
__device__ __forceinline__ uint32_t order_key(float x) {
    uint32_t b = __float_as_uint(x);
    if (x != x) return 0xfffffffeu;  // below the largest number, which stands for "no limit"
    if (x == 0.f) b = 0u;
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
// Key of an element of a row: equal values order by column, the lower column being the larger key, so no two are equal.
__device__ __forceinline__ uint64_t element_key(uint32_t key, uint32_t col) { return ((uint64_t)key << 32) | (uint32_t)~col; }

struct MaxKey {
    using Acc = uint64_t;
    static __device__ __forceinline__ Acc init() { return 0; }
    static __device__ __forceinline__ Acc combine(Acc a, Acc b) { return a > b ? a : b; }
    static __device__ __forceinline__ Acc shfl_xor(Acc a, int m) { return (Acc)__shfl_xor((unsigned long long)a, m, kWave); }
};

__global__ __launch_bounds__(kBlock) void topk_rounds_kernel(const float* x, float* values, uint64_t* indices, size_t rows,
                                                              size_t cols, size_t k) {
    __shared__ uint64_t smem[kBlock / kWave];
    __shared__ uint64_t best;
    for (size_t r = blockIdx.x; r < rows; r += gridDim.x) {
        uint64_t below = ~(uint64_t)0;
        for (size_t j = 0; j < k; j++) {
            uint64_t m = 0;
            for (size_t c = threadIdx.x; c < cols; c += kBlock) {
                const uint64_t key = element_key(order_key(x[r * cols + c]), (uint32_t)c);
                if (key < below && key > m) m = key;
            }
            m = block_reduce<MaxKey>(m, smem);
            if (threadIdx.x == 0) {
                best = m;
                const uint32_t c = ~(uint32_t)m;
                values[r * k + j] = x[r * cols + c];
                indices[r * k + j] = c;
            }
            __syncthreads();
            below = best;
            __syncthreads();
        }
    }
}

// A row's chosen places in LDS: entry j holds its column (kNoCol: none), and only the first of the entries that name a
// column speaks for it.
constexpr uint32_t kNoCol = 0xffffffffu;
constexpr int kMaxK = ZG_HIP_TOPK_MAX_K;
__device__ __forceinline__ bool speaks(const uint32_t* col, int j) {
    const uint32_t c = col[j];
    if (c == kNoCol) return false;
    for (int i = 0; i < j; i++)
        if (col[i] == c) return false;
    return true;
}

template <bool ACC>
__global__ __launch_bounds__(kBlock) void topk_bwd_kernel(const uint64_t* indices, const float* y_g, float* x_g, size_t rows,
                                                           size_t cols, size_t k) {
    __shared__ uint32_t col[kMaxK];
    __shared__ float g[kMaxK];
    for (size_t r = blockIdx.x; r < rows; r += gridDim.x) {
        __syncthreads();
        for (int j = threadIdx.x; j < (int)k; j += kBlock) {
            const uint64_t c = indices[r * k + j];
            col[j] = c < cols ? (uint32_t)c : kNoCol;
            g[j] = y_g[r * k + j];
        }
        float* row = x_g + r * cols;
        if (!ACC)
            for (size_t c = threadIdx.x; c < cols; c += kBlock) row[c] = 0.f;
        __syncthreads();
        for (int j = threadIdx.x; j < (int)k; j += kBlock) {
            if (!speaks(col, j)) continue;
            float v = ACC ? __fadd_rn(row[col[j]], g[j]) : g[j];
            for (int i = j + 1; i < (int)k; i++)
                if (col[i] == col[j]) v = __fadd_rn(v, g[i]);
            row[col[j]] = v;
        }
    }
}

// ------------------------------------------------------------------------------------------------
// distillation
// ------------------------------------------------------------------------------------------------
struct MaxF {
    using Acc = float;
    static __device__ __forceinline__ Acc init() { return -INFINITY; }
    static __device__ __forceinline__ Acc combine(Acc a, Acc b) { return fmaxf(a, b); }
    static __device__ __forceinline__ Acc shfl_xor(Acc a, int m) { return __shfl_xor(a, m, kWave); }
};
template <class P>
__device__ __forceinline__ typename P::Acc block_all(typename P::Acc v, typename P::Acc* smem) {
    v = block_reduce<P>(v, smem);
    __syncthreads();
    if (threadIdx.x == 0) smem[0] = v;
    __syncthreads();
    v = smem[0];
    __syncthreads();
    return v;
}

struct DistillArgs {
    const float* x;
    const float* t;
    const uint64_t* idx;
    const float* w;
    float* stats;
    float* row_loss;
    float* grad;
    size_t rows, cols, k;
    float temp, inv_temp, mean;
};

// FWD: statistics and loss; BWD: gradient, added when ACC
template <bool FWD, bool BWD, bool ACC>
__global__ __launch_bounds__(kBlock) void distill_kernel(DistillArgs a) {
    __shared__ float smem[kBlock / kWave];
    __shared__ uint32_t col[kMaxK];
    __shared__ float q[kMaxK];
    for (size_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const float* x = a.x + r * a.cols;
        float* grad = BWD ? a.grad + r * a.cols : nullptr;
        const float w = a.w ? a.w[r] : a.mean;
        if (w == 0.f) {
            if (FWD && threadIdx.x == 0) {
                a.stats[2 * r] = a.stats[2 * r + 1] = 0.f;
                a.row_loss[r] = 0.f;
            }
            if (BWD && !ACC)
                for (size_t c = threadIdx.x; c < a.cols; c += kBlock) grad[c] = 0.f;
            continue;
        }
        // the student's statistics
        float m, ls;
        if (FWD) {
            float mx = -INFINITY;
            for (size_t c = threadIdx.x; c < a.cols; c += kBlock) mx = fmaxf(mx, x[c]);
            m = block_all<MaxF>(mx, smem);
            float s = 0.f;
            const float from = m == -INFINITY ? 0.f : m;
            for (size_t c = threadIdx.x; c < a.cols; c += kBlock) s += expf((x[c] - from) * a.inv_temp);
            s = block_all<SumAcc>(s, smem);
            ls = logf(s);
            if (m == -INFINITY) {
                if (s != 0.f) m = NAN;  // NaNs among logits of -inf
                else ls = 0.f;
            }
            if (threadIdx.x == 0) {
                a.stats[2 * r] = m;
                a.stats[2 * r + 1] = ls;
            }
        } else {
            m = a.stats[2 * r];
            ls = a.stats[2 * r + 1];
        }
        // the teacher's distribution
        float tm = -INFINITY;
        for (size_t j = threadIdx.x; j < a.k; j += kBlock) {
            const uint64_t c = a.idx[r * a.k + j];
            const bool held = c < a.cols;
            col[j] = held ? (uint32_t)c : kNoCol;
            if (held) tm = fmaxf(tm, a.t[r * a.k + j]);
        }
        tm = block_all<MaxF>(tm, smem);
        const float t_from = tm == -INFINITY ? 0.f : tm;
        float ts = 0.f;
        for (size_t j = threadIdx.x; j < a.k; j += kBlock) {
            q[j] = col[j] != kNoCol ? expf((a.t[r * a.k + j] - t_from) * a.inv_temp) : 0.f;
            ts += q[j];
        }
        ts = block_all<SumAcc>(ts, smem);
        const bool empty = ts == 0.f || m == -INFINITY;
        if (FWD) {
            const float lts = logf(ts);
            float part = 0.f;
            for (size_t j = threadIdx.x; j < a.k; j += kBlock)
                if (q[j] != 0.f && !empty) {
                    const float log_q = (a.t[r * a.k + j] - t_from) * a.inv_temp - lts;
                    const float log_p = (x[col[j]] - m) * a.inv_temp - ls;
                    part += q[j] / ts * (log_q - log_p);
                }
            part = block_all<SumAcc>(part, smem);
            if (threadIdx.x == 0) a.row_loss[r] = empty ? 0.f : part * a.temp * a.temp;
        }
        if (BWD) {
            if (empty) {
                if (!ACC)
                    for (size_t c = threadIdx.x; c < a.cols; c += kBlock) grad[c] = 0.f;
                __syncthreads();
                continue;
            }
            const float f = w * a.temp;
            __syncthreads();
            float old[kMaxK / kBlock];
            for (int u = 0; u < kMaxK / kBlock; u++) {
                const int j = threadIdx.x + u * kBlock;
                old[u] = (ACC && j < (int)a.k && col[j] != kNoCol) ? grad[col[j]] : 0.f;
            }
            __syncthreads();
            for (size_t c = threadIdx.x; c < a.cols; c += kBlock) {
                const float v = f * expf((x[c] - m) * a.inv_temp - ls);
                grad[c] = ACC ? grad[c] + v : v;
            }
            __syncthreads();
            for (int u = 0; u < kMaxK / kBlock; u++) {
                const int j = threadIdx.x + u * kBlock;
                if (j >= (int)a.k || !speaks(col, j)) continue;
                float sum = 0.f;
                for (int i = j; i < (int)a.k; i++)
                    if (col[i] == col[j]) sum += q[i];
                const float v = f * (expf((x[col[j]] - m) * a.inv_temp - ls) - sum / ts);
                grad[col[j]] = ACC ? old[u] + v : v;
            }
        }
        __syncthreads();
    }
}

static unsigned row_grid(size_t rows) { return (unsigned)(rows < 65536 ? rows : 65536); }

static int distill_check(const char* op, const float* logits, const float* teacher, const uint64_t* indices,
                         const float* row_weights, size_t rows, size_t cols, size_t k, float temperature) {
    ZG_REQUIRE(logits && teacher && indices, "%s: null pointer", op);
    ZG_REQUIRE(((uintptr_t)indices & 7u) == 0, "%s: indices are not on an 8-byte boundary", op);
    ZG_REQUIRE(cols < 0xffffffffull, "%s: %zu columns", op, cols);
    ZG_REQUIRE(mul_sat(rows, cols) < ((size_t)1 << 60) && mul_sat(rows, k) < ((size_t)1 << 60), "%s: %zu rows", op, rows);
    ZG_REQUIRE(k >= 1 && k <= kMaxK, "%s: k = %zu is not in 1 .. %d", op, k, kMaxK);
    ZG_REQUIRE(temperature > 0.f && temperature < INFINITY && 1.f / temperature < INFINITY, "%s: temperature %g", op, temperature);
    return ZG_HIP_OK;
}
// an output against the inputs of the loss
static int distill_clear(const char* op, const char* name, const void* out, size_t bytes, const float* logits,
                         const float* teacher, const uint64_t* indices, const float* row_weights, size_t rows, size_t cols,
                         size_t k) {
    ZG_REQUIRE(out, "%s: null %s", op, name);
    ZG_REQUIRE(!ranges_overlap(out, bytes, logits, rows * cols * 4) && !ranges_overlap(out, bytes, teacher, rows * k * 4) &&
                   !ranges_overlap(out, bytes, indices, rows * k * 8) && !ranges_overlap(out, bytes, row_weights, rows * 4),
               "%s: %s overlaps an input", op, name);
    return ZG_HIP_OK;
}
static int distill_total(zg_hip_ctx* ctx, const float* row_loss, const float* row_weights, float* loss, size_t rows) {
    if (row_weights) return flat_reduce<TermDot, 2>(ctx, row_loss, row_weights, rows, 0.f, FinStore{loss});
    return flat_reduce<TermId, 1>(ctx, row_loss, nullptr, rows, 0.f, FinDivN{loss, (float)rows});
}

}  // namespace zg

using namespace zg;

ZG_API int zg_hip_topk_fwd(zg_hip_ctx* ctx, const float* x, float* values, uint64_t* indices, size_t rows, size_t cols,
                           size_t k) {
    ZG_CTX(ctx);
    ZG_REQUIRE(k >= 1 && k <= cols && k <= kMaxK, "topk_fwd: k = %zu is not in 1 .. min(%zu, %d)", k, cols, kMaxK);
    ZG_REQUIRE(cols < 0xffffffffull, "topk_fwd: %zu columns", cols);
    if (rows == 0) return ZG_HIP_OK;
    ZG_REQUIRE(x && values && indices, "topk_fwd: null pointer");
    ZG_REQUIRE(((uintptr_t)indices & 7u) == 0, "topk_fwd: indices are not on an 8-byte boundary");
    ZG_REQUIRE(mul_sat(rows, cols) < ((size_t)1 << 60), "topk_fwd: %zu rows", rows);
    ZG_REQUIRE(!ranges_overlap(values, rows * k * 4, x, rows * cols * 4) && !ranges_overlap(indices, rows * k * 8, x, rows * cols * 4) &&
                   !ranges_overlap(indices, rows * k * 8, values, rows * k * 4),
               "topk_fwd: an output overlaps another operand");
    DeviceGuard guard(ctx);
    hipLaunchKernelGGL(topk_rounds_kernel, dim3(row_grid(rows)), dim3(kBlock), 0, ctx->stream, x, values, indices, rows, cols, k);
    ZG_LAUNCH_CHECK();
    return ZG_HIP_OK;
}

ZG_API int zg_hip_topk_bwd(zg_hip_ctx* ctx, const uint64_t* indices, const float* y_g, float* x_g, size_t rows, size_t cols,
                           size_t k, int accumulate) {
    ZG_CTX(ctx);
    ZG_REQUIRE(k >= 1 && k <= kMaxK, "topk_bwd: k = %zu is not in 1 .. %d", k, kMaxK);
    ZG_REQUIRE(cols < 0xffffffffull, "topk_bwd: %zu columns", cols);
    if (rows == 0 || cols == 0) return ZG_HIP_OK;
    ZG_REQUIRE(indices && y_g && x_g, "topk_bwd: null pointer");
    ZG_REQUIRE(((uintptr_t)indices & 7u) == 0, "topk_bwd: indices are not on an 8-byte boundary");
    ZG_REQUIRE(mul_sat(rows, cols) < ((size_t)1 << 60) && mul_sat(rows, k) < ((size_t)1 << 60), "topk_bwd: %zu rows", rows);
    ZG_REQUIRE(!ranges_overlap(x_g, rows * cols * 4, y_g, rows * k * 4) && !ranges_overlap(x_g, rows * cols * 4, indices, rows * k * 8),
               "topk_bwd: x_g overlaps an input");
    DeviceGuard guard(ctx);
    if (accumulate)
        hipLaunchKernelGGL(topk_bwd_kernel<true>, dim3(row_grid(rows)), dim3(kBlock), 0, ctx->stream, indices, y_g, x_g, rows, cols, k);
    else
        hipLaunchKernelGGL(topk_bwd_kernel<false>, dim3(row_grid(rows)), dim3(kBlock), 0, ctx->stream, indices, y_g, x_g, rows, cols, k);
    ZG_LAUNCH_CHECK();
    return ZG_HIP_OK;
}

namespace zg {
static int distill_entry(zg_hip_ctx* ctx, const char* op, const float* logits, const float* teacher, const uint64_t* indices,
                         const float* row_weights, float* stats, float* row_loss, float* loss, float* grad, size_t rows,
                         size_t cols, size_t k, float temperature, int accumulate, bool fwd, bool bwd) {
    if (int rc = distill_check(op, logits, teacher, indices, row_weights, rows, cols, k, temperature)) return rc;
    if (fwd) {
        if (int rc = distill_clear(op, "stats", stats, rows * 8, logits, teacher, indices, row_weights, rows, cols, k)) return rc;
        if (int rc = distill_clear(op, "row_loss", row_loss, rows * 4, logits, teacher, indices, row_weights, rows, cols, k)) return rc;
        if (int rc = distill_clear(op, "loss", loss, 4, logits, teacher, indices, row_weights, rows, cols, k)) return rc;
        ZG_REQUIRE(!ranges_overlap(stats, rows * 8, row_loss, rows * 4) && !ranges_overlap(loss, 4, row_loss, rows * 4) &&
                       !ranges_overlap(loss, 4, stats, rows * 8),
                   "%s: two outputs overlap", op);
    } else {
        ZG_REQUIRE(stats, "%s: null stats", op);
    }
    if (bwd) {
        if (int rc = distill_clear(op, "grad", grad, rows * cols * 4, logits, teacher, indices, row_weights, rows, cols, k)) return rc;
        ZG_REQUIRE(!ranges_overlap(grad, rows * cols * 4, stats, rows * 8) &&
                       (!fwd || (!ranges_overlap(grad, rows * cols * 4, row_loss, rows * 4) && !ranges_overlap(grad, rows * cols * 4, loss, 4))),
                   "%s: grad overlaps another operand", op);
    }
    DeviceGuard guard(ctx);
    DistillArgs a{logits, teacher, indices, row_weights, stats, row_loss, grad, rows, cols, k, temperature, 1.f / temperature,
                  1.f / (float)rows};
    const dim3 grid(row_grid(rows)), block(kBlock);
    if (fwd && !bwd) hipLaunchKernelGGL((distill_kernel<true, false, false>), grid, block, 0, ctx->stream, a);
    else if (!fwd && !accumulate) hipLaunchKernelGGL((distill_kernel<false, true, false>), grid, block, 0, ctx->stream, a);
    else if (!fwd) hipLaunchKernelGGL((distill_kernel<false, true, true>), grid, block, 0, ctx->stream, a);
    else if (!accumulate) hipLaunchKernelGGL((distill_kernel<true, true, false>), grid, block, 0, ctx->stream, a);
    else hipLaunchKernelGGL((distill_kernel<true, true, true>), grid, block, 0, ctx->stream, a);
    ZG_LAUNCH_CHECK();
    return fwd ? distill_total(ctx, row_loss, row_weights, loss, rows) : ZG_HIP_OK;
}
}  // namespace zg

ZG_API int zg_hip_distill_fwd(zg_hip_ctx* ctx, const float* logits, const float* teacher, const uint64_t* indices,
                              const float* row_weights, float* stats, float* row_loss, float* loss, size_t rows, size_t cols,
                              size_t k, float temperature) {
    ZG_CTX(ctx);
    ZG_REQUIRE(rows > 0 && cols > 0, "distill_fwd: empty matrix (%zu x %zu)", rows, cols);
    return distill_entry(ctx, "distill_fwd", logits, teacher, indices, row_weights, stats, row_loss, loss, nullptr, rows, cols, k,
                         temperature, 0, true, false);
}

ZG_API int zg_hip_distill_bwd(zg_hip_ctx* ctx, const float* logits, const float* teacher, const uint64_t* indices,
                              const float* row_weights, const float* stats, float* grad, size_t rows, size_t cols, size_t k,
                              float temperature, int accumulate) {
    ZG_CTX(ctx);
    if (rows == 0 || cols == 0) return ZG_HIP_OK;
    return distill_entry(ctx, "distill_bwd", logits, teacher, indices, row_weights, const_cast<float*>(stats), nullptr, nullptr, grad,
                         rows, cols, k, temperature, accumulate, false, true);
}

ZG_API int zg_hip_distill_fwd_bwd(zg_hip_ctx* ctx, const float* logits, const float* teacher, const uint64_t* indices,
                                  const float* row_weights, float* stats, float* row_loss, float* loss, float* grad, size_t rows,
                                  size_t cols, size_t k, float temperature, int accumulate) {
    ZG_CTX(ctx);
    ZG_REQUIRE(rows > 0 && cols > 0, "distill_fwd_bwd: empty matrix (%zu x %zu)", rows, cols);
    return distill_entry(ctx, "distill_fwd_bwd", logits, teacher, indices, row_weights, stats, row_loss, loss, grad, rows, cols, k,
                         temperature, accumulate, true, true);
}
