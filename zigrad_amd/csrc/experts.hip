// Rows to experts and back: the order of the entries by expert, rows laid out in that order, their weighted sums.
#include "reduce_device.h"

namespace zg {

// ------------------------------------------------------------------------------------------------
// expert_sort: a stable counting sort.  A workgroup owns a run of entries, each of its waves a run of those; counters are
// integers in LDS, so their order of arrival changes nothing.
// ------------------------------------------------------------------------------------------------
constexpr int kSortThreads = 512;
constexpr int kSortWaves = kSortThreads / kWave;
constexpr size_t kSortAlone = 8192;  // entries one workgroup orders in one launch
constexpr size_t kSortMaxBlocks = 256;
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
    uint32_t* next = mem;                           // [wave][expert]: where the wave's next entry of the expert goes
    uint32_t* base = mem + kSortWaves * n_experts;  // [expert]: where the workgroup's entries of the expert begin
    uint32_t* scan = base + n_experts;              // one value per thread
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int i = threadIdx.x; i < kSortWaves * n_experts; i += kSortThreads) next[i] = 0;
    __syncthreads();
    const size_t lo = (size_t)blockIdx.x * per_block, hi = lo + per_block < n ? lo + per_block : n;
    const size_t per_wave = (per_block + kSortThreads - 1) / kSortThreads * kWave;
    const size_t w_lo = lo + wave * per_wave, w_hi = w_lo + per_wave < hi ? w_lo + per_wave : hi;
    for (size_t i = w_lo + lane; i < w_hi; i += kWave) {
        const uint64_t e = experts[i];
        if (e < (uint64_t)n_experts) atomicAdd(&next[wave * n_experts + e], 1u);
    }
    __syncthreads();
    // thread t sums up the experts [t * per, (t + 1) * per): all workgroups' counts, and those of the workgroups before
    const int per = (n_experts + kSortThreads - 1) / kSortThreads;
    const int e_lo = threadIdx.x * per, e_hi = e_lo + per < n_experts ? e_lo + per : n_experts;
    uint32_t mine = 0;
    for (int e = e_lo; e < e_hi; e++) {
        uint32_t all = 0, before = 0;
        if (counts) {
            for (unsigned b = 0; b < gridDim.x; b++) {
                const uint32_t c = counts[(size_t)b * n_experts + e];
                before += b < blockIdx.x ? c : 0u;
                all += c;
            }
        } else {
            for (int w = 0; w < kSortWaves; w++) all += next[w * n_experts + e];
        }
        base[e] = mine + before;
        mine += all;
    }
    scan[threadIdx.x] = mine;
    __syncthreads();
    for (int d = 1; d < kSortThreads; d <<= 1) {
        const uint32_t v = (int)threadIdx.x >= d ? scan[threadIdx.x - d] : 0u;
        __syncthreads();
        scan[threadIdx.x] += v;
        __syncthreads();
    }
    const uint32_t first = scan[threadIdx.x] - mine;  // entries of all experts before this thread's
    for (int e = e_lo; e < e_hi; e++) {
        uint32_t at = base[e] + first;
        base[e] = at;
        for (int w = 0; w < kSortWaves; w++) {
            const uint32_t c = next[w * n_experts + e];
            next[w * n_experts + e] = at;
            at += c;
        }
    }
    __syncthreads();
    if (blockIdx.x == 0) {  // its entries come first, so its bases are the experts' offsets
        for (int e = threadIdx.x; e < n_experts; e += kSortThreads) offsets[e] = base[e];
        if (threadIdx.x == kSortThreads - 1) offsets[n_experts] = scan[threadIdx.x];
    }
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
// rows in the order of their experts, and back
// ------------------------------------------------------------------------------------------------
// SCALE: the rows are multiplied by their weights (the backward of the combination)
template <int V, bool SCALE>
__global__ __launch_bounds__(kBlock) void expert_spread_kernel(const float* x, const uint64_t* slots, const float* weights,
                                                                float* y, size_t n_tokens, size_t k, size_t width) {
    typedef float vec __attribute__((ext_vector_type(V)));
    const size_t pieces = width / V, total = n_tokens * pieces, places = n_tokens * k;
    for (size_t i = (size_t)blockIdx.x * kBlock + threadIdx.x; i < total; i += (size_t)gridDim.x * kBlock) {
        const size_t t = i / pieces, p = i - t * pieces;
        const vec v = *reinterpret_cast<const vec*>(x + t * width + p * V);
        for (size_t j = 0; j < k; j++) {
            const uint64_t s = slots[t * k + j];
            if (s >= places) continue;
            vec o = v;
            if (SCALE) {
                const float w = weights[t * k + j];
                for (int u = 0; u < V; u++) o[u] = __fmul_rn(w, v[u]);
            }
            *reinterpret_cast<vec*>(y + s * width + p * V) = o;
        }
    }
}

// SCALE: the weighted sum; else the plain one.  ACC: added to what is there.
template <int V, bool SCALE, bool ACC>
__global__ __launch_bounds__(kBlock) void expert_gather_kernel(const float* y, const uint64_t* slots, const float* weights,
                                                                float* out, size_t n_tokens, size_t k, size_t width) {
    typedef float vec __attribute__((ext_vector_type(V)));
    const size_t pieces = width / V, total = n_tokens * pieces, places = n_tokens * k;
    for (size_t i = (size_t)blockIdx.x * kBlock + threadIdx.x; i < total; i += (size_t)gridDim.x * kBlock) {
        const size_t t = i / pieces, p = i - t * pieces;
        vec* const to = reinterpret_cast<vec*>(out + t * width + p * V);
        vec acc;
        for (int u = 0; u < V; u++) acc[u] = 0.f;
        if (ACC) acc = *to;
        for (size_t j = 0; j < k; j++) {
            const uint64_t s = slots[t * k + j];
            if (s >= places) continue;
            const vec v = *reinterpret_cast<const vec*>(y + s * width + p * V);
            const float w = SCALE ? weights[t * k + j] : 1.f;
            for (int u = 0; u < V; u++) acc[u] += SCALE ? w * v[u] : v[u];
        }
        *to = acc;
    }
}

// a wave per entry: the product of the row's gradient with the entry's output
__global__ __launch_bounds__(kBlock) void expert_weight_grad_kernel(const float* out_g, const float* y, const uint64_t* slots,
                                                                     float* weights_g, size_t n_tokens, size_t k, size_t width) {
    const int lane = threadIdx.x & 63;
    const size_t n = n_tokens * k;
    for (size_t i = (size_t)blockIdx.x * (kBlock / kWave) + (threadIdx.x >> 6); i < n; i += (size_t)gridDim.x * (kBlock / kWave)) {
        const uint64_t s = slots[i];
        float sum = 0.f;
        if (s < n)
            for (size_t c = lane; c < width; c += kWave) sum += out_g[i / k * width + c] * y[s * width + c];
        sum = group_reduce<SumAcc>(sum);
        if (lane == 0) weights_g[i] = sum;
    }
}

static unsigned flat_grid(size_t items) {
    const size_t b = ceil_div_sz(items, kBlock);
    return (unsigned)(b < 65536 ? b : 65536);
}
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
    size_t blocks = n_entries <= kSortAlone ? 1 : ceil_div_sz(n_entries, 1024);
    if (blocks > kSortMaxBlocks) blocks = kSortMaxBlocks;
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
    const size_t lds = ((kSortWaves + 1) * n_experts + kSortThreads) * sizeof(uint32_t);
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
    const bool vec = width % 4 == 0 && aligned16(x) && aligned16(y);
    if (vec) hipLaunchKernelGGL((expert_spread_kernel<4, false>), dim3(flat_grid(n_tokens * (width / 4))), dim3(kBlock), 0, ctx->stream,
                                x, slots, (const float*)nullptr, y, n_tokens, k, width);
    else hipLaunchKernelGGL((expert_spread_kernel<1, false>), dim3(flat_grid(n_tokens * width)), dim3(kBlock), 0, ctx->stream, x, slots,
                            (const float*)nullptr, y, n_tokens, k, width);
    ZG_LAUNCH_CHECK();
    return ZG_HIP_OK;
}

namespace zg {
template <bool SCALE, bool ACC>
static int launch_gather(zg_hip_ctx* ctx, const float* y, const uint64_t* slots, const float* weights, float* out, size_t n_tokens,
                         size_t k, size_t width) {
    const bool vec = width % 4 == 0 && aligned16(y) && aligned16(out);
    if (vec) hipLaunchKernelGGL((expert_gather_kernel<4, SCALE, ACC>), dim3(flat_grid(n_tokens * (width / 4))), dim3(kBlock), 0,
                                ctx->stream, y, slots, weights, out, n_tokens, k, width);
    else hipLaunchKernelGGL((expert_gather_kernel<1, SCALE, ACC>), dim3(flat_grid(n_tokens * width)), dim3(kBlock), 0, ctx->stream, y,
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
    if (y_g) {
        const bool vec = width % 4 == 0 && aligned16(out_g) && aligned16(y_g);
        if (vec) hipLaunchKernelGGL((expert_spread_kernel<4, true>), dim3(flat_grid(n_tokens * (width / 4))), dim3(kBlock), 0,
                                    ctx->stream, out_g, slots, weights, y_g, n_tokens, k, width);
        else hipLaunchKernelGGL((expert_spread_kernel<1, true>), dim3(flat_grid(n_tokens * width)), dim3(kBlock), 0, ctx->stream, out_g,
                                slots, weights, y_g, n_tokens, k, width);
        ZG_LAUNCH_CHECK();
    }
    if (weights_g) {
        hipLaunchKernelGGL(expert_weight_grad_kernel, dim3(flat_grid(n * kWave)), dim3(kBlock), 0, ctx->stream, out_g, y, slots,
                           weights_g, n_tokens, k, width);
        ZG_LAUNCH_CHECK();
    }
    return ZG_HIP_OK;
}
