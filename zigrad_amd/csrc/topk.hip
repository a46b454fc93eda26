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

// The float whose key this is; numbers that are no float's key come out as NaN.
__device__ __forceinline__ float key_value(uint32_t key) {
    return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
}

constexpr int kMaxK = ZG_HIP_TOPK_MAX_K;

// ------------------------------------------------------------------------------------------------
// Selection.  NT threads (a wave, or a workgroup of four) own a row and read it once:
//   * the first NT x 4 x VPT values are held in registers as 4 NT groups, and the k-th largest of the groups' maxima is a
//     lower bound of the row's k-th largest value (k groups hold a value at least that large each).  It is found bit by
//     bit from the top, counting with ballots, and only to 16 bits: a bound that is a little low lets a few more through;
//   * values that reach the bound become candidates in LDS as 64-bit keys (value, then column), about k of them among the
//     first values and k / (4 NT VPT) of the rest of the row.  A thread looks at its single values only when their maximum
//     reaches the bound, so the row is read at the memory's rate;
//   * with more than kRankMost candidates the k largest are cut out by a radix selection over their keys (eight bits at a
//     time, as many digits as it takes to tell them apart), which also raises the bound for the rest of the row;
//   * a candidate's place in the result is the number of larger keys, which every thread counts for its own candidates.
// Keys are unique, so neither the order in which candidates arrive nor the variant taken changes the result.
// When a stretch of the row brings more candidates than LDS has room for (rows in rising order, rows of few different values) the
// row is read again in pieces that fit whatever they hold (select_slowly).
// ------------------------------------------------------------------------------------------------
typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));  // 16 bytes at any 4-byte alignment

template <int NT>
struct Select {
    static constexpr int kWaves = NT / kWave;
    static constexpr int kCap = NT == kWave ? 1024 : 4096;
    static constexpr uint32_t kRankMost = 384;
    uint64_t key[kCap + 2];
    uint32_t hist[256];
    uint32_t count[2][kWaves];
    uint32_t n;  // candidates asked for; those past kCap found no room
};

// orders the LDS accesses of the NT threads
template <int NT>
__device__ __forceinline__ void select_sync() {
    if constexpr (NT == kWave) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    } else {
        __syncthreads();
    }
}

__device__ __forceinline__ float larger(float a, float b) {  // NaN if either is
    return __builtin_elementwise_maximum(a, b);
}

// What a value has to reach: `low` for the quick look (NaN: every value passes), `key` exactly.
struct Bound {
    uint32_t key;
    float low;
};

// Four values from column col on; what lies behind the row's end is -inf, which loses to every value of the row.  ONCE: not
// read again.
template <bool ONCE>
__device__ __forceinline__ float4u row_piece(const float* row, uint32_t col, uint32_t cols) {
    if (col + 4 <= cols) {
        const float4u* p = reinterpret_cast<const float4u*>(row + col);
        return ONCE ? __builtin_nontemporal_load(p) : *p;
    }
    float4u v = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    if (col < cols) v.x = row[col];
    if (col + 1 < cols) v.y = row[col + 1];
    if (col + 2 < cols) v.z = row[col + 2];
    return v;
}

// Those of the four values that reach the bound become candidates.
template <int NT>
__device__ __forceinline__ void push_piece(Select<NT>& s, float4u v, uint32_t col, uint32_t cols, Bound bound) {
    if (larger(larger(v.x, v.y), larger(v.z, v.w)) < bound.low) return;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const uint32_t key = order_key(v[e]);
        if (key < bound.key || col + e >= cols) continue;
        const uint32_t at = atomicAdd(&s.n, 1u);
        if (at < (uint32_t)Select<NT>::kCap) s.key[at] = element_key(key, col + e);
    }
}

// Leaves the k largest of the s.n <= kCap candidates and returns the bound for values of later columns.  All threads call it
// after a sync and find the candidates in place when it returns.
template <int NT>
__device__ Bound select_cut(Select<NT>& s, uint32_t k, int tid) {
    const uint32_t n = s.n;
    const int lane = tid & (kWave - 1);
    uint64_t prefix = 0, mask = 0;
    uint32_t need = k;
    for (int shift = 56; shift >= 0; shift -= 8) {
        for (int i = tid; i < 256; i += NT) s.hist[i] = 0;
        select_sync<NT>();
        for (uint32_t i = tid; i < n; i += NT) {
            const uint64_t key = s.key[i];
            if ((key & mask) == prefix) atomicAdd(&s.hist[(key >> shift) & 255], 1u);
        }
        select_sync<NT>();
        // every wave finds the digit: lane l looks after the digits 255 - 4l .. 252 - 4l
        uint32_t h[4], sum = 0;
#pragma unroll
        for (int u = 0; u < 4; u++) {
            h[u] = s.hist[255 - 4 * lane - u];
            sum += h[u];
        }
        uint32_t incl = sum;
#pragma unroll
        for (int d = 1; d < kWave; d <<= 1) {
            const uint32_t o = (uint32_t)__shfl_up((int)incl, d, kWave);
            if (lane >= d) incl += o;
        }
        const int l = __builtin_ctzll(__ballot(incl >= need));
        uint32_t above = incl - sum, digit = 0, inside = 0;
        bool found = false;
#pragma unroll
        for (int u = 0; u < 4; u++) {
            if (!found && above + h[u] >= need) {
                found = true;
                digit = 255 - 4 * lane - u;
                inside = h[u];
            }
            if (!found) above += h[u];
        }
        above = (uint32_t)__builtin_amdgcn_readlane((int)above, l);
        digit = (uint32_t)__builtin_amdgcn_readlane((int)digit, l);
        inside = (uint32_t)__builtin_amdgcn_readlane((int)inside, l);
        prefix |= (uint64_t)digit << shift;
        mask |= (uint64_t)255 << shift;
        need -= above;
        select_sync<NT>();
        if (inside == need) break;  // exactly the keys from here on up
    }
    // moved down in place: what is kept of a stretch lands where keys have been read already
    if (tid == 0) s.n = 0;
    select_sync<NT>();
    for (uint32_t i0 = 0; i0 < n; i0 += NT) {
        const uint64_t mine = i0 + tid < n ? s.key[i0 + tid] : 0;
        select_sync<NT>();
        if (mine >= prefix && mine != 0) s.key[atomicAdd(&s.n, 1u)] = mine;
        select_sync<NT>();
    }
    // with the whole value told apart, later columns of the same value lose
    const uint32_t top = (uint32_t)(prefix >> 32);
    return {(uint32_t)mask ? top + 1 : top, key_value(top)};
}

// The row again, NT x 4 values at a time, with room made before each.
template <int NT>
__device__ void select_slowly(Select<NT>& s, const float* row, uint32_t cols, uint32_t k, int tid) {
    Bound bound{0u, NAN};
    select_sync<NT>();
    if (tid == 0) s.n = 0;
    select_sync<NT>();
    for (uint32_t c0 = 0; c0 < cols; c0 += 4 * NT) {
        if (s.n + 4 * NT > (uint32_t)Select<NT>::kCap) bound = select_cut<NT>(s, k, tid);
        select_sync<NT>();
        const uint32_t col = c0 + 4 * tid;
        push_piece<NT>(s, row_piece<false>(row, col, cols), col, cols, bound);
        select_sync<NT>();
    }
}

// The candidates of a row, at least k of them, its k largest among them.
template <int NT, int VPT>
__device__ __forceinline__ void select_row(Select<NT>& s, const float* row, uint32_t cols, uint32_t k, int tid) {
    constexpr uint32_t kTile = 4 * NT * VPT;
    constexpr int U = 4;                    // pieces in flight per thread behind the tile
    constexpr uint32_t kStretch = 4 * 4 * NT * U;  // columns between two looks at the number of candidates
    const int lane = tid & (kWave - 1), wave = tid / kWave;
    float4u v[VPT];
#pragma unroll
    for (int u = 0; u < VPT; u++) v[u] = row_piece<false>(row, 4 * (tid + u * NT), cols);
    float4u top = v[0];  // groups: the same component of a thread's pieces
#pragma unroll
    for (int u = 1; u < VPT; u++)
#pragma unroll
        for (int e = 0; e < 4; e++) top[e] = larger(top[e], v[u][e]);
    uint32_t group[4];
#pragma unroll
    for (int e = 0; e < 4; e++) group[e] = order_key(top[e]);
    if (tid == 0) s.n = 0;
    uint32_t t = 0;
#pragma unroll 1
    for (int bit = 31; bit >= 16; bit--) {
        const uint32_t c = t | (1u << bit);
        uint32_t reach = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) reach += (uint32_t)__popcll(__ballot(group[e] >= c));
        if constexpr (NT != kWave) {
            if (lane == 0) s.count[bit & 1][wave] = reach;
            __syncthreads();
            reach = 0;
#pragma unroll
            for (int w = 0; w < Select<NT>::kWaves; w++) reach += s.count[bit & 1][w];
        }
        if (reach >= k) t = c;
    }
    Bound bound{t, key_value(t)};
    select_sync<NT>();
    // a thread whose maximum reaches the bound reads its values again (from the caches): holding them costs the registers
    // of half the waves
    if (!(larger(larger(top[0], top[1]), larger(top[2], top[3])) < bound.low)) {
#pragma unroll 2
        for (uint32_t col = 4 * tid; col < kTile && col < cols; col += 4 * NT)
            push_piece<NT>(s, row_piece<false>(row, col, cols), col, cols, bound);
    }
    select_sync<NT>();
    for (uint32_t c0 = kTile; c0 < cols && s.n <= (uint32_t)Select<NT>::kCap;) {
        if (s.n > (uint32_t)Select<NT>::kCap / 2) {
            const Bound b = select_cut<NT>(s, k, tid);
            if (b.key > bound.key) bound = b;
        }
        select_sync<NT>();
        const uint32_t end = cols - c0 < kStretch ? cols : c0 + kStretch;
        for (; c0 < end; c0 += 4 * NT * U) {
            float4u w[U];
#pragma unroll
            for (int u = 0; u < U; u++) w[u] = row_piece<true>(row, c0 + 4 * (tid + u * NT), cols);
#pragma unroll
            for (int u = 0; u < U; u++) push_piece<NT>(s, w[u], c0 + 4 * (tid + u * NT), cols, bound);
        }
        select_sync<NT>();
    }
    if (s.n > (uint32_t)Select<NT>::kCap) select_slowly<NT>(s, row, cols, k, tid);
}

// The k largest candidates in order, by rank: emit(rank, key).
template <int NT, class Emit>
__device__ __forceinline__ void select_emit(Select<NT>& s, uint32_t k, int tid, Emit emit) {
    if (s.n > Select<NT>::kRankMost && s.n > k) select_cut<NT>(s, k, tid);
    const uint32_t n = s.n;
    if (tid < 2) s.key[n + tid] = 0;
    select_sync<NT>();
    for (uint32_t i = tid; i < n; i += NT) {
        const uint64_t mine = s.key[i];
        uint32_t rank = 0;
        for (uint32_t j = 0; j < n; j += 2) rank += (uint32_t)(s.key[j] > mine) + (uint32_t)(s.key[j + 1] > mine);
        if (rank < k) emit(rank, mine);
    }
}

template <int NT, int VPT>
__global__ __launch_bounds__(256, 4) void topk_kernel(const float* x, float* values, uint64_t* indices, size_t rows, uint32_t cols,
                                                   uint32_t k) {
    constexpr int kRows = 256 / NT;
    __shared__ Select<NT> mem[kRows];
    const int tid = threadIdx.x % NT, sub = threadIdx.x / NT;
    Select<NT>& s = mem[sub];
    for (size_t r = (size_t)blockIdx.x * kRows + sub; r < rows; r += (size_t)gridDim.x * kRows) {
        const float* row = x + r * cols;
        select_row<NT, VPT>(s, row, cols, k, tid);
        select_emit<NT>(s, k, tid, [&](uint32_t rank, uint64_t key) {
            const uint32_t c = ~(uint32_t)key;
            values[r * k + rank] = row[c];
            indices[r * k + rank] = c;
        });
        select_sync<NT>();
    }
}

// A row's chosen places in LDS: entry j holds its column (kNoCol: none), and only the first of the entries that name a
// column speaks for it.
constexpr uint32_t kNoCol = 0xffffffffu;
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
    ZG_REQUIRE(cols < ((size_t)1 << 31), "%s: %zu columns", op, cols);
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
    ZG_REQUIRE(cols < ((size_t)1 << 31), "topk_fwd: %zu columns", cols);
    if (rows == 0) return ZG_HIP_OK;
    ZG_REQUIRE(x && values && indices, "topk_fwd: null pointer");
    ZG_REQUIRE(((uintptr_t)indices & 7u) == 0, "topk_fwd: indices are not on an 8-byte boundary");
    ZG_REQUIRE(mul_sat(rows, cols) < ((size_t)1 << 60), "topk_fwd: %zu rows", rows);
    ZG_REQUIRE(!ranges_overlap(values, rows * k * 4, x, rows * cols * 4) && !ranges_overlap(indices, rows * k * 8, x, rows * cols * 4) &&
                   !ranges_overlap(indices, rows * k * 8, values, rows * k * 4),
               "topk_fwd: an output overlaps another operand");
    DeviceGuard guard(ctx);
    const uint32_t c32 = (uint32_t)cols, k32 = (uint32_t)k;
#define ZG_TOPK(NT, VPT)                                                                                                      \
    hipLaunchKernelGGL((topk_kernel<NT, VPT>), dim3(row_grid(ceil_div_sz(rows, 256 / (NT)))), dim3(256), 0, ctx->stream, x, values, \
                       indices, rows, c32, k32)
    // A wave per row up to 2048 columns, as far as its 256 groups can bound k; a workgroup per row beyond.
    if (cols <= 2048 && k <= 128) {
        if (cols <= 256) ZG_TOPK(64, 1);
        else if (cols <= 512) ZG_TOPK(64, 2);
        else if (cols <= 1024) ZG_TOPK(64, 4);
        else ZG_TOPK(64, 8);
    } else if (cols <= 2048) {
        ZG_TOPK(256, 2);
    } else {
        ZG_TOPK(256, 8);
    }
#undef ZG_TOPK
    ZG_LAUNCH_CHECK();
    return ZG_HIP_OK;
}

ZG_API int zg_hip_topk_bwd(zg_hip_ctx* ctx, const uint64_t* indices, const float* y_g, float* x_g, size_t rows, size_t cols,
                           size_t k, int accumulate) {
    ZG_CTX(ctx);
    ZG_REQUIRE(k >= 1 && k <= kMaxK, "topk_bwd: k = %zu is not in 1 .. %d", k, kMaxK);
    ZG_REQUIRE(cols < ((size_t)1 << 31), "topk_bwd: %zu columns", cols);
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
