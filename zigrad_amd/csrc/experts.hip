// Rows to experts and back: the order of the entries by expert, rows laid out in that order, their weighted sums.
#include "reduce_device.h"

namespace zg {

// ------------------------------------------------------------------------------------------------
// expert_sort: a stable counting sort.  A workgroup owns a run of entries, each of its waves a run of those; counters are
// integers in LDS, so their order of arrival changes nothing.  Up to kSortAlone entries one workgroup does everything in a launch;
// more are counted first, run by run, and every workgroup adds up for itself what lies before its run.  Latency bounds it
// throughout (65536 entries are 1 MiB in and out).
// ------------------------------------------------------------------------------------------------
constexpr int kSortThreads = 512;
constexpr int kSortWaves = kSortThreads / kWave;
constexpr size_t kSortAlone = 2048;
constexpr int kMaxExperts = ZG_HIP_EXPERTS_MAX;

__global__ __launch_bounds__(kSortThreads) void expert_count_kernel(const uint64_t* experts, uint32_t* counts, size_t n,
                                                                     size_t per_block, int n_experts) {
    __shared__ uint32_t hist[kMaxExperts];
    for (int e = threadIdx.x; e < n_experts; e += kSortThreads) hist[e] = 0;
    __syncthreads();
    const size_t lo = (size_t)blockIdx.x * per_block, hi = lo + per_block < n ? lo + per_block : n;
    for (size_t i = lo + threadIdx.x; i < hi; i += kSortThreads) {
        const uint64_t e = experts[i];
        if (e < (uint64_t)n_experts) atomicAdd(&hist[e], 1u);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < n_experts; e += kSortThreads) counts[(size_t)blockIdx.x * n_experts + e] = hist[e];
}

// counts (null with a single workgroup): what expert_count_kernel found for every workgroup's run
__global__ __launch_bounds__(kSortThreads) void expert_place_kernel(const uint64_t* experts, const uint32_t* counts,
                                                                     uint64_t* offsets, uint64_t* slots, size_t n,
                                                                     size_t per_block, int n_experts) {
    extern __shared__ uint32_t mem[];
    uint32_t* next = mem;                            // [wave][expert]: where the wave's next entry of the expert goes
    uint32_t* before = mem + kSortWaves * n_experts; // [expert]: entries of the expert in the workgroups before this one
    uint32_t* all = before + n_experts;              // [expert]: its entries, then those of all experts before it
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int i = threadIdx.x; i < (kSortWaves + 2) * n_experts; i += kSortThreads) mem[i] = 0;
    __syncthreads();
    const size_t lo = (size_t)blockIdx.x * per_block, hi = lo + per_block < n ? lo + per_block : n;
    const size_t per_wave = (per_block + kSortThreads - 1) / kSortThreads * kWave;
    const size_t w_lo = lo + wave * per_wave, w_hi = w_lo + per_wave < hi ? w_lo + per_wave : hi;
    for (size_t i = w_lo + lane; i < w_hi; i += kWave) {
        const uint64_t e = experts[i];
        if (e < (uint64_t)n_experts) atomicAdd(&next[wave * n_experts + e], 1u);
    }
    if (counts) {
        // a column of the counts per thread; with fewer experts than threads several threads share one, each with its own runs
        int wide = kSortThreads;
        while (wide / 2 >= n_experts) wide /= 2;
        const unsigned groups = kSortThreads / wide, group = threadIdx.x / wide;
        for (int e = threadIdx.x % wide; e < n_experts; e += wide) {
            uint32_t sum = 0, early = 0;
            for (unsigned b0 = group; b0 < gridDim.x; b0 += 16 * groups) {  // sixteen loads in flight: they come from other XCDs' writes
                uint32_t c[16];
#pragma unroll
                for (int u = 0; u < 16; u++) {
                    const unsigned b = b0 + u * groups;
                    c[u] = b < gridDim.x ? counts[(size_t)b * n_experts + e] : 0u;
                }
#pragma unroll
                for (int u = 0; u < 16; u++) {
                    sum += c[u];
                    early += b0 + u * groups < blockIdx.x ? c[u] : 0u;
                }
            }
            atomicAdd(&all[e], sum);
            atomicAdd(&before[e], early);
        }
    }
    __syncthreads();
    if (!counts) {
        for (int e = threadIdx.x; e < n_experts; e += kSortThreads) {
            uint32_t c = 0;
            for (int w = 0; w < kSortWaves; w++) c += next[w * n_experts + e];
            all[e] = c;
        }
        __syncthreads();
    }
    if (wave == 0) {  // exclusive sums over the experts, 64 at a time
        uint32_t carry = 0;
        for (int e0 = 0; e0 < n_experts; e0 += kWave) {
            const int e = e0 + lane;
            const uint32_t c = e < n_experts ? all[e] : 0u;
            uint32_t incl = c;
#pragma unroll
            for (int d = 1; d < kWave; d <<= 1) {
                const uint32_t o = (uint32_t)__shfl_up((int)incl, d, kWave);
                if (lane >= d) incl += o;
            }
            if (e < n_experts) all[e] = carry + incl - c;
            if (blockIdx.x == 0 && e < n_experts) offsets[e] = carry + incl - c;
            carry += (uint32_t)__builtin_amdgcn_readlane((int)incl, kWave - 1);
        }
        if (blockIdx.x == 0 && lane == 0) offsets[n_experts] = carry;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < n_experts; e += kSortThreads) {
        uint32_t at = all[e] + before[e];
        for (int w = 0; w < kSortWaves; w++) {
            const uint32_t c = next[w * n_experts + e];
            next[w * n_experts + e] = at;
            at += c;
        }
    }
    __syncthreads();
    // each wave places its run in order, 64 entries at a time: an entry goes behind the lower lanes of the same expert
    volatile uint32_t* const my_next = next + wave * n_experts;
    for (size_t i0 = w_lo; i0 < w_hi; i0 += kWave) {
        const size_t i = i0 + lane;
        const uint64_t e64 = i < w_hi ? experts[i] : ~(uint64_t)0;
        const bool held = e64 < (uint64_t)n_experts;
        const uint32_t e = held ? (uint32_t)e64 : 0u;
        uint64_t same = __ballot(held);
        for (int bit = 0; (1 << bit) < n_experts; bit++) {
            const uint64_t ones = __ballot((e >> bit) & 1u);
            same &= ((e >> bit) & 1u) ? ones : ~ones;
        }
        const uint32_t below = (uint32_t)__popcll(same & (((uint64_t)1 << lane) - 1));
        const uint32_t start = held ? my_next[e] : 0u;
        __builtin_amdgcn_wave_barrier();
        if (held && below + 1 == (uint32_t)__popcll(same)) my_next[e] = start + below + 1;
        __builtin_amdgcn_wave_barrier();
        if (i < w_hi) slots[i] = held ? (uint64_t)(start + below) : ~(uint64_t)0;
    }
}

// ------------------------------------------------------------------------------------------------
// Rows in the order of their experts, and back.  All are bound by memory: each row is read and written once, in pieces of four
// values at whatever 4-byte alignment the rows have (the memory system serves 16-byte accesses there; a row's last piece may
// hold fewer).  A thread owns a piece of a token's row and walks the token's k entries.
// ------------------------------------------------------------------------------------------------
typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));

template <bool ONCE = false>  // ONCE: past the memory-side cache
__device__ __forceinline__ float4u load_piece(const float* row, size_t c, size_t width) {
    if (ONCE && c + 4 <= width) return __builtin_nontemporal_load(reinterpret_cast<const float4u*>(row + c));
    if (c + 4 <= width) return *reinterpret_cast<const float4u*>(row + c);
    float4u v = {row[c], 0.f, 0.f, 0.f};
    if (c + 1 < width) v.y = row[c + 1];
    if (c + 2 < width) v.z = row[c + 2];
    return v;
}
template <bool ONCE = false>
__device__ __forceinline__ void store_piece(float* row, size_t c, size_t width, float4u v) {
    if (c + 4 <= width) {
        if (ONCE) __builtin_nontemporal_store(v, reinterpret_cast<float4u*>(row + c));
        else *reinterpret_cast<float4u*>(row + c) = v;
        return;
    }
    row[c] = v.x;
    if (c + 1 < width) row[c + 1] = v.y;
    if (c + 2 < width) row[c + 2] = v.z;
}
// Quotient and remainder; a 32-bit division where that does (a 64-bit one costs more than the rest of a piece).
__device__ __forceinline__ void split(size_t i, size_t by, size_t& q, size_t& rem) {
    if ((i | by) < ((size_t)1 << 32)) {
        const uint32_t d = (uint32_t)i / (uint32_t)by;
        q = d;
        rem = (uint32_t)i - d * (uint32_t)by;
    } else {
        q = i / by;
        rem = i - q * by;
    }
}

constexpr int kEntriesAtOnce = 4;  // of a token, whose loads are in flight together

template <bool ONCE>
__global__ __launch_bounds__(kBlock) void expert_spread_kernel(const float* x, const uint64_t* slots, float* y, size_t n_tokens,
                                                                size_t k, size_t width) {
    const size_t pieces = (width + 3) / 4, total = n_tokens * pieces, places = n_tokens * k;
    for (size_t i = (size_t)blockIdx.x * kBlock + threadIdx.x; i < total; i += (size_t)gridDim.x * kBlock) {
        size_t t, p;
        split(i, pieces, t, p);
        const float4u v = load_piece(x + t * width, 4 * p, width);
        for (size_t j0 = 0; j0 < k; j0 += kEntriesAtOnce) {
            uint64_t s[kEntriesAtOnce];
#pragma unroll
            for (int u = 0; u < kEntriesAtOnce; u++) s[u] = j0 + u < k ? slots[t * k + j0 + u] : ~(uint64_t)0;
#pragma unroll
            for (int u = 0; u < kEntriesAtOnce; u++)
                if (s[u] < places) store_piece<ONCE>(y + s[u] * width, 4 * p, width, v);
        }
    }
}

// SCALE: the weighted sum; else the plain one.  ACC: added to what is there.
template <bool SCALE, bool ACC, bool ONCE>
__global__ __launch_bounds__(kBlock) void expert_gather_kernel(const float* y, const uint64_t* slots, const float* weights,
                                                                float* out, size_t n_tokens, size_t k, size_t width) {
    const size_t pieces = (width + 3) / 4, total = n_tokens * pieces, places = n_tokens * k;
    for (size_t i = (size_t)blockIdx.x * kBlock + threadIdx.x; i < total; i += (size_t)gridDim.x * kBlock) {
        size_t t, p;
        split(i, pieces, t, p);
        float4u acc = {0.f, 0.f, 0.f, 0.f};
        if (ACC) acc = load_piece(out + t * width, 4 * p, width);
        for (size_t j0 = 0; j0 < k; j0 += kEntriesAtOnce) {
            bool held[kEntriesAtOnce];
            float w[kEntriesAtOnce];
            float4u v[kEntriesAtOnce];
#pragma unroll
            for (int u = 0; u < kEntriesAtOnce; u++) {
                const uint64_t s = j0 + u < k ? slots[t * k + j0 + u] : ~(uint64_t)0;
                held[u] = s < places;
                w[u] = SCALE && held[u] ? weights[t * k + j0 + u] : 1.f;
                v[u] = float4u{0.f, 0.f, 0.f, 0.f};
                if (held[u]) v[u] = load_piece<ONCE>(y + s * width, 4 * p, width);
            }
#pragma unroll
            for (int u = 0; u < kEntriesAtOnce; u++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float term = SCALE ? w[u] * v[u][e] : v[u][e];
                    acc[e] = held[u] ? acc[e] + term : acc[e];
                }
        }
        store_piece(out + t * width, 4 * p, width, acc);
    }
}

// The backward of the combination: L lanes take an entry, scale its token's gradient into its row and sum up the product of that gradient
// with the entry's output in the same pass.  ROWS / WEIGHTS: which of the two are wanted.
// ONCE_IN, ONCE_OUT: y and y_g pass by the memory-side cache.
template <int L, bool ROWS, bool WEIGHTS, bool ONCE_IN, bool ONCE_OUT>
__global__ __launch_bounds__(kBlock) void expert_combine_bwd_kernel(const float* out_g, const float* y, const uint64_t* slots,
                                                                     const float* weights, float* y_g, float* weights_g,
                                                                     size_t n_tokens, size_t k, size_t width) {
    constexpr int U = 4;
    const int lane = threadIdx.x % L;
    const size_t n = n_tokens * k, pieces = (width + 3) / 4;
    for (size_t i = (size_t)blockIdx.x * (kBlock / L) + threadIdx.x / L; i < n; i += (size_t)gridDim.x * (kBlock / L)) {
        const uint64_t s = slots[i];
        float sum = 0.f;
        if (s < n) {
            size_t t, j;
            split(i, k, t, j);
            const float w = ROWS ? weights[i] : 0.f;
            const float* g_row = out_g + t * width;
            const float* y_row = WEIGHTS ? y + s * width : nullptr;
            for (size_t p0 = lane; p0 < pieces; p0 += U * L) {
                float4u g[U], v[U];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const size_t p = p0 + (size_t)u * L;
                    g[u] = v[u] = float4u{0.f, 0.f, 0.f, 0.f};
                    if (p < pieces) {
                        g[u] = load_piece(g_row, 4 * p, width);
                        if (WEIGHTS) v[u] = load_piece<ONCE_IN>(y_row, 4 * p, width);
                    }
                }
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const size_t p = p0 + (size_t)u * L;
                    if (WEIGHTS) sum += (g[u].x * v[u].x + g[u].y * v[u].y) + (g[u].z * v[u].z + g[u].w * v[u].w);
                    if (ROWS && p < pieces)
                        store_piece<ONCE_OUT>(y_g + s * width, 4 * p, width, float4u{w * g[u].x, w * g[u].y, w * g[u].z, w * g[u].w});
                }
            }
        }
        if (WEIGHTS) {
#pragma unroll
            for (int m = L / 2; m >= 1; m >>= 1) sum += __shfl_xor(sum, m, kWave);
            if (lane == 0) weights_g[i] = sum;
        }
    }
}

static unsigned flat_grid(size_t items) {
    const size_t b = ceil_div_sz(items, kBlock);
    return (unsigned)(b < 1048576 ? b : 1048576);
}
// Whether so many floats pass a kernel once that the memory-side cache (256 MB) can not hold them.  Loads and stores that pass by it win
// then (8 entries of width 1024 for 16384 tokens: dispatch 110 -> 101 us, combine 117 -> 106, combine_bwd 217 -> 198; for 8192 tokens
// dispatch 58 -> 51 and combine_bwd, whose stores still go to the cache, 110 -> 98) and lose before (6 of 1030 for 4095: combine 21 -> 27,
// combine_bwd 39 -> 45).
static bool past_cache(size_t floats) { return floats > (size_t)64 << 20; }
static int experts_check(const char* op, const uint64_t* slots, size_t n_tokens, size_t k, size_t width) {
    ZG_REQUIRE(k >= 1 && k <= ZG_HIP_EXPERTS_MAX_K, "%s: k = %zu is not in 1 .. %d", op, k, (int)ZG_HIP_EXPERTS_MAX_K);
    ZG_REQUIRE(mul_sat(mul_sat(n_tokens, k), width) < ((size_t)1 << 60), "%s: %zu x %zu rows of %zu", op, n_tokens, k, width);
    ZG_REQUIRE(((uintptr_t)slots & 7u) == 0, "%s: slots are not on an 8-byte boundary", op);
    return ZG_HIP_OK;
}

}  // namespace zg

using namespace zg;

ZG_API int zg_hip_expert_sort(zg_hip_ctx* ctx, const uint64_t* experts, uint64_t* offsets, uint64_t* slots, size_t n_entries,
                              size_t n_experts) {
    ZG_CTX(ctx);
    ZG_REQUIRE(n_experts >= 1 && n_experts <= kMaxExperts, "expert_sort: %zu experts are not in 1 .. %d", n_experts, kMaxExperts);
    ZG_REQUIRE(n_entries < 0xffffffffull, "expert_sort: %zu entries", n_entries);
    ZG_REQUIRE(offsets && (n_entries == 0 || (experts && slots)), "expert_sort: null pointer");
    ZG_REQUIRE((((uintptr_t)experts | (uintptr_t)offsets | (uintptr_t)slots) & 7u) == 0,
               "expert_sort: an array is not on an 8-byte boundary");
    ZG_REQUIRE(!ranges_overlap(experts, n_entries * 8, slots, n_entries * 8) &&
                   !ranges_overlap(experts, n_entries * 8, offsets, (n_experts + 1) * 8) &&
                   !ranges_overlap(slots, n_entries * 8, offsets, (n_experts + 1) * 8),
               "expert_sort: two arrays overlap");
    DeviceGuard guard(ctx);
    // runs of 1024 entries or more; every workgroup reads all runs' counts, so many experts get fewer runs
    const size_t most = n_experts < 128 ? 256 : 32768 / n_experts;
    size_t blocks = n_entries <= kSortAlone ? 1 : ceil_div_sz(n_entries, 1024);
    if (blocks > most) blocks = most;
    const size_t per_block = ceil_div_sz(ceil_div_sz(n_entries, blocks), kSortThreads) * kSortThreads;
    blocks = n_entries ? ceil_div_sz(n_entries, per_block) : 1;
    uint32_t* counts = nullptr;
    if (blocks > 1) {
        counts = (uint32_t*)workspace(ctx, blocks * n_experts * sizeof(uint32_t));
        if (!counts) return ZG_HIP_EOOM;
        hipLaunchKernelGGL(expert_count_kernel, dim3((unsigned)blocks), dim3(kSortThreads), 0, ctx->stream, experts, counts,
                           n_entries, per_block, (int)n_experts);
        ZG_LAUNCH_CHECK();
    }
    const size_t lds = (kSortWaves + 2) * n_experts * sizeof(uint32_t);
    hipLaunchKernelGGL(expert_place_kernel, dim3((unsigned)blocks), dim3(kSortThreads), lds, ctx->stream, experts, counts, offsets,
                       slots, n_entries, per_block, (int)n_experts);
    ZG_LAUNCH_CHECK();
    return ZG_HIP_OK;
}

ZG_API int zg_hip_expert_dispatch(zg_hip_ctx* ctx, const float* x, const uint64_t* slots, float* y, size_t n_tokens, size_t k,
                                  size_t width) {
    ZG_CTX(ctx);
    if (int rc = experts_check("expert_dispatch", slots, n_tokens, k, width)) return rc;
    if (n_tokens == 0 || width == 0) return ZG_HIP_OK;
    ZG_REQUIRE(x && slots && y, "expert_dispatch: null pointer");
    const size_t bytes = n_tokens * k * width * 4;
    ZG_REQUIRE(!ranges_overlap(y, bytes, x, n_tokens * width * 4) && !ranges_overlap(y, bytes, slots, n_tokens * k * 8),
               "expert_dispatch: y overlaps an input");
    DeviceGuard guard(ctx);
    if (past_cache(n_tokens * width * k + n_tokens * width))
        hipLaunchKernelGGL(expert_spread_kernel<true>, dim3(flat_grid(n_tokens * ((width + 3) / 4))), dim3(kBlock), 0, ctx->stream, x, slots, y,
                       n_tokens, k, width);
    else
        hipLaunchKernelGGL(expert_spread_kernel<false>, dim3(flat_grid(n_tokens * ((width + 3) / 4))), dim3(kBlock), 0, ctx->stream, x, slots, y,
                       n_tokens, k, width);
    ZG_LAUNCH_CHECK();
    return ZG_HIP_OK;
}

namespace zg {
template <bool SCALE, bool ACC>
static int launch_gather(zg_hip_ctx* ctx, const float* y, const uint64_t* slots, const float* weights, float* out, size_t n_tokens,
                         size_t k, size_t width) {
    if (past_cache(n_tokens * width * k + n_tokens * width))
        hipLaunchKernelGGL((expert_gather_kernel<SCALE, ACC, true>), dim3(flat_grid(n_tokens * ((width + 3) / 4))), dim3(kBlock), 0, ctx->stream, y,
                       slots, weights, out, n_tokens, k, width);
    else
        hipLaunchKernelGGL((expert_gather_kernel<SCALE, ACC, false>), dim3(flat_grid(n_tokens * ((width + 3) / 4))), dim3(kBlock), 0, ctx->stream, y,
                       slots, weights, out, n_tokens, k, width);
    ZG_LAUNCH_CHECK();
    return ZG_HIP_OK;
}
}  // namespace zg

ZG_API int zg_hip_expert_dispatch_bwd(zg_hip_ctx* ctx, const float* y_g, const uint64_t* slots, float* x_g, size_t n_tokens,
                                      size_t k, size_t width, int accumulate) {
    ZG_CTX(ctx);
    if (int rc = experts_check("expert_dispatch_bwd", slots, n_tokens, k, width)) return rc;
    if (n_tokens == 0 || width == 0) return ZG_HIP_OK;
    ZG_REQUIRE(y_g && slots && x_g, "expert_dispatch_bwd: null pointer");
    const size_t bytes = n_tokens * width * 4;
    ZG_REQUIRE(!ranges_overlap(x_g, bytes, y_g, bytes * k) && !ranges_overlap(x_g, bytes, slots, n_tokens * k * 8),
               "expert_dispatch_bwd: x_g overlaps an input");
    DeviceGuard guard(ctx);
    return accumulate ? launch_gather<false, true>(ctx, y_g, slots, nullptr, x_g, n_tokens, k, width)
                      : launch_gather<false, false>(ctx, y_g, slots, nullptr, x_g, n_tokens, k, width);
}

ZG_API int zg_hip_expert_combine(zg_hip_ctx* ctx, const float* y, const uint64_t* slots, const float* weights, float* out,
                                 size_t n_tokens, size_t k, size_t width) {
    ZG_CTX(ctx);
    if (int rc = experts_check("expert_combine", slots, n_tokens, k, width)) return rc;
    if (n_tokens == 0 || width == 0) return ZG_HIP_OK;
    ZG_REQUIRE(y && slots && weights && out, "expert_combine: null pointer");
    const size_t bytes = n_tokens * width * 4;
    ZG_REQUIRE(!ranges_overlap(out, bytes, y, bytes * k) && !ranges_overlap(out, bytes, slots, n_tokens * k * 8) &&
                   !ranges_overlap(out, bytes, weights, n_tokens * k * 4),
               "expert_combine: out overlaps an input");
    DeviceGuard guard(ctx);
    return launch_gather<true, false>(ctx, y, slots, weights, out, n_tokens, k, width);
}

ZG_API int zg_hip_expert_combine_bwd(zg_hip_ctx* ctx, const float* out_g, const float* y, const uint64_t* slots,
                                     const float* weights, float* y_g, float* weights_g, size_t n_tokens, size_t k, size_t width) {
    ZG_CTX(ctx);
    if (int rc = experts_check("expert_combine_bwd", slots, n_tokens, k, width)) return rc;
    if (n_tokens == 0 || width == 0) return ZG_HIP_OK;
    ZG_REQUIRE(slots && out_g && (!y_g || weights) && (!weights_g || y), "expert_combine_bwd: null pointer");
    const size_t row_bytes = n_tokens * width * 4, n = n_tokens * k;
    ZG_REQUIRE(!ranges_overlap(y_g, row_bytes * k, out_g, row_bytes) && !ranges_overlap(y_g, row_bytes * k, y, row_bytes * k) &&
                   !ranges_overlap(y_g, row_bytes * k, slots, n * 8) && !ranges_overlap(y_g, row_bytes * k, weights, n * 4) &&
                   !ranges_overlap(y_g, row_bytes * k, weights_g, n * 4),
               "expert_combine_bwd: y_g overlaps another operand");
    ZG_REQUIRE(!ranges_overlap(weights_g, n * 4, out_g, row_bytes) && !ranges_overlap(weights_g, n * 4, y, row_bytes * k) &&
                   !ranges_overlap(weights_g, n * 4, slots, n * 8) && !ranges_overlap(weights_g, n * 4, weights, n * 4),
               "expert_combine_bwd: weights_g overlaps another operand");
    DeviceGuard guard(ctx);
    if (!y_g && !weights_g) return ZG_HIP_OK;
    // 16 lanes an entry for narrow rows, a wave else
    const bool once_in = past_cache(n * width * ((y_g ? 1 : 0) + (weights_g ? 1 : 0)) + n_tokens * width);
    const bool once_out = past_cache(n * width);
#define ZG_COMBINE_BWD_(L, ROWS, WEIGHTS, IN, OUT)                                                                                     \
    hipLaunchKernelGGL((expert_combine_bwd_kernel<L, ROWS, WEIGHTS, IN, OUT>), dim3(flat_grid(n * (L))), dim3(kBlock), 0, ctx->stream, \
                       out_g, y, slots, weights, y_g, weights_g, n_tokens, k, width)
#define ZG_COMBINE_BWD(L, ROWS, WEIGHTS)                                                       \
    do {                                                                                       \
        if (ROWS && once_out) ZG_COMBINE_BWD_(L, ROWS, WEIGHTS, WEIGHTS, ROWS);                \
        else if (WEIGHTS && once_in) ZG_COMBINE_BWD_(L, ROWS, WEIGHTS, WEIGHTS, false);        \
        else ZG_COMBINE_BWD_(L, ROWS, WEIGHTS, false, false);                                  \
    } while (0)
    if (width <= 128) {
        if (y_g && weights_g) ZG_COMBINE_BWD(16, true, true);
        else if (y_g) ZG_COMBINE_BWD(16, true, false);
        else ZG_COMBINE_BWD(16, false, true);
    } else {
        if (y_g && weights_g) ZG_COMBINE_BWD(64, true, true);
        else if (y_g) ZG_COMBINE_BWD(64, true, false);
        else ZG_COMBINE_BWD(64, false, true);
    }
#undef ZG_COMBINE_BWD
#undef ZG_COMBINE_BWD_
    ZG_LAUNCH_CHECK();
    return ZG_HIP_OK;
}
