// The k largest of a row, and the loss of a student against a teacher's k largest logits.
#include "reduce_device.h"

#include <type_traits>

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
//   * the first NT x 4 x VPT values are held in registers as groups, and the k-th largest of the groups' maxima is a lower
//     bound of the row's k-th largest value (k groups hold a value at least that large each).  It is found bit by
//     bit from the top, counting with ballots, and only to 16 bits: a bound that is a little low lets a few more through;
//   * values that reach the bound become candidates in LDS as 64-bit keys (value, then column), about k of them among the
//     first values and k / (4 NT VPT) of the rest of the row.  Each wave has a stretch of LDS and a counter in registers
//     for its own, so that a candidate costs a ballot and a store (a shared LDS counter, whose answer every store had to
//     wait for, took 332 us for 64 of 32000 in 8192 rows where this takes 182 us, 5.8 TB/s);
//   * with more than kRankMost candidates the k largest are cut out by a radix selection over their keys (eight bits at a
//     time, as many digits as it takes to tell them apart), which also raises the bound for the rest of the row;
//   * a candidate's place in the result is the number of larger keys, which every thread counts for its own candidates.
// Keys are unique, so neither the order in which candidates arrive nor the variant taken changes the result.
// When a stretch of the row brings more candidates than LDS has room for (rows in rising order, rows of few different values)
// the row is read again in pieces that fit whatever they hold (select_slowly).
// ------------------------------------------------------------------------------------------------
typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));  // 16 bytes at any 4-byte alignment

constexpr int kSegment = 1024;       // candidates a wave has room for, or fewer (SEG)
constexpr uint32_t kRankMost = 384;
constexpr int kThin = 6;             // times 64: candidates of a wave that are thinned out with ballots

template <int NT, int SEG = kSegment>
struct Select {
    static constexpr int kWaves = NT / kWave;
    uint64_t key[kWaves][SEG + 2];
    uint32_t hist[256];
    uint32_t low[kWaves];       // the waves' bounds
    uint32_t n[kWaves];         // candidates, written down where other waves need them
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

// What a value has to reach, as a key and as that key's number (NaN where there is none: every value passes).
struct Bound {
    uint32_t key;
    float low;
};
__device__ __forceinline__ Bound bound_of(uint32_t key) { return {key, key_value(key)}; }

// The thread's place: its number among the NT, its wave, its lane; n: the wave's candidates, the same in all its lanes, of which
// the first `keyed` are in LDS as keys and the rest as they came, (bits of the value, column).
struct Place {
    int tid, wave, lane;
    uint32_t n, keyed;
};

// Whole pieces of four values of a row, from `base` (the same in all lanes) on; `bytes`: how far the row's whole pieces reach from
// there.  Pieces behind that are -inf, which loses to every value of the row: a buffer load takes any 4-byte alignment and
// reads nothing behind the end.
typedef unsigned uint4v __attribute__((ext_vector_type(4)));
template <bool ONCE = false>  // ONCE: past the memory-side cache
__device__ __forceinline__ float4u row_piece(const float* base, uint32_t bytes, uint32_t off) {
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(base), 0, (int)bytes, 0x00020000);
    const float4u v = __builtin_bit_cast(float4u, (uint4v)__builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)off, 0, ONCE ? 2 : 0));
    const bool in = off < bytes;
    return float4u{in ? v.x : -INFINITY, in ? v.y : -INFINITY, in ? v.z : -INFINITY, in ? v.w : -INFINITY};
}
// N pieces of a row, `by` bytes apart; all loads before the first is waited for
template <int N>
__device__ __forceinline__ void row_pieces(float4u* v, const float* base, uint32_t bytes, uint32_t off, uint32_t by, bool once) {
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(base), 0, (int)bytes, 0x00020000);
    uint4v raw[N];
    if (once) {
#pragma unroll
        for (int u = 0; u < N; u++) raw[u] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)(off + u * by), 0, 2);
    } else {
#pragma unroll
        for (int u = 0; u < N; u++) raw[u] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)(off + u * by), 0, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < N; u++) {
        const float4u p = __builtin_bit_cast(float4u, raw[u]);
        const bool in = off + u * by < bytes;
        v[u] = float4u{in ? p.x : -INFINITY, in ? p.y : -INFINITY, in ? p.z : -INFINITY, in ? p.w : -INFINITY};
    }
}
__device__ __forceinline__ uint32_t bytes_from(uint32_t c0, uint32_t whole) {  // whole: columns in whole pieces
    const uint32_t left = c0 < whole ? whole - c0 : 0u;
    return left < (1u << 28) ? left * 4u : 1u << 30;
}
__device__ __forceinline__ uint32_t lanes_below(uint64_t lanes) {  // how many of `lanes` are below this one
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(lanes >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)lanes, 0u));
}

// Those of the four values that reach the bound become candidates of the wave, all of whose lanes call this.  Candidates past
// SEG are counted and find no room.  CHECK: columns from `cols` on are none.
template <int NT, bool CHECK, int SEG>
__device__ __forceinline__ void push_piece(Select<NT, SEG>& s, Place& at, float4u v, uint32_t col, uint32_t cols, float low) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const bool in = !(v[e] < low) && (!CHECK || col + e < cols);
        const uint64_t ins = __ballot(in);
        if (!ins) continue;
        const uint32_t to = at.n + lanes_below(ins);
        if (in && to < SEG) s.key[at.wave][to] = ((uint64_t)__float_as_uint(v[e]) << 32) | (col + e);
        at.n += (uint32_t)__popcll(ins);
    }
    __builtin_amdgcn_sched_barrier(0);  // a piece at a time: done side by side they cost the registers of half the waves
}
// The up to three values behind the row's whole pieces.
template <int NT, int SEG>
__device__ __forceinline__ void push_tail(Select<NT, SEG>& s, Place& at, const float* row, uint32_t whole, uint32_t cols, float low) {
    if (whole == cols || at.wave != 0) return;
    const uint32_t col = whole + at.lane;
    const float x = col < cols ? row[col] : -INFINITY;
    push_piece<NT, true>(s, at, float4u{x, -INFINITY, -INFINITY, -INFINITY}, col, col < cols ? col + 1 : 0u, low);
}
// The candidates that came since are turned into keys.
template <int NT, int SEG>
__device__ __forceinline__ void key_candidates(Select<NT, SEG>& s, Place& at) {
    select_sync<kWave>();
    for (uint32_t i = at.keyed + at.lane; i < at.n; i += kWave) {
        const uint64_t c = s.key[at.wave][i];
        s.key[at.wave][i] = element_key(order_key(__uint_as_float((uint32_t)(c >> 32))), (uint32_t)c);
    }
    at.keyed = at.n;
}

// The most candidates any wave has; a sync.
template <int NT, int SEG>
__device__ __forceinline__ uint32_t select_most(Select<NT, SEG>& s, const Place& at) {
    if constexpr (NT == kWave) {
        select_sync<NT>();
        return at.n;
    } else {
        if (at.lane == 0) s.n[at.wave] = at.n;
        __syncthreads();
        uint32_t most = 0;
#pragma unroll
        for (int w = 0; w < Select<NT>::kWaves; w++) most = s.n[w] > most ? s.n[w] : most;
        return most;
    }
}

// Leaves the k largest of the candidates (none lost, at least k) and returns the bound for values of later columns.  All threads
// call it after select_most.
template <int NT, int SEG>
__device__ Bound select_cut(Select<NT, SEG>& s, Place& at, uint32_t k) {
    const int lane = at.lane;
    key_candidates<NT>(s, at);
    uint64_t prefix = 0, mask = 0;
    uint32_t need = k;
    for (int shift = 56; shift >= 0; shift -= 8) {
        for (int i = at.tid; i < 256; i += NT) s.hist[i] = 0;
        select_sync<NT>();
        for (uint32_t i = lane; i < at.n; i += kWave) {
            const uint64_t key = s.key[at.wave][i];
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
    // each wave moves its own down: what is kept lands where keys have been read already
    uint32_t kept = 0;
    for (uint32_t i0 = 0; i0 < at.n; i0 += kWave) {
        const uint64_t mine = i0 + lane < at.n ? s.key[at.wave][i0 + lane] : 0;
        const bool in = mine >= prefix && mine != 0;
        const uint64_t ins = __ballot(in);
        select_sync<kWave>();
        if (in) s.key[at.wave][kept + lanes_below(ins)] = mine;
        select_sync<kWave>();
        kept += (uint32_t)__popcll(ins);
    }
    at.n = at.keyed = kept;
    // with the whole value told apart, later columns of the same value lose
    const uint32_t top = (uint32_t)(prefix >> 32);
    return bound_of((uint32_t)mask ? top + 1 : top);
}

// The largest number t of 16 bits, then zeros, that at least `share` of the wave's keys reach; 0 when it has fewer.  KEYS keys a lane.
template <int KEYS>
__device__ __forceinline__ uint32_t wave_bound(const uint32_t (&key)[KEYS], uint32_t share) {
    uint32_t t = 0;
#pragma unroll
    for (int bit = 31; bit >= 16; bit--) {
        const uint32_t c = t | (1u << bit);
        uint32_t reach = 0;
#pragma unroll
        for (int e = 0; e < KEYS; e++) reach += (uint32_t)__popcll(__ballot(key[e] >= c));
        if (reach >= share) t = c;
        if (reach == share) break;  // no need to know the bound better
    }
    return t;
}
// The lowest of the waves' bounds: k values of the row reach it when each wave bounds its share of k.
template <int NT, int SEG>
__device__ __forceinline__ uint32_t lowest_bound(Select<NT, SEG>& s, const Place& at, uint32_t t) {
    if constexpr (NT != kWave) {
        if (at.lane == 0) s.low[at.wave] = t;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < Select<NT>::kWaves; w++) t = s.low[w] < t ? s.low[w] : t;
    }
    return t;
}

// Drops candidates that a bound from the candidates themselves excludes (a few hundred come down to little more than k; ranking is
// quadratic in what is left) and returns that bound.  No wave has more than 64 KEYS; all threads call it after a sync.
template <int NT, int KEYS, int SEG>
__device__ __forceinline__ uint32_t select_thin(Select<NT, SEG>& s, Place& at, uint32_t share) {
    key_candidates<NT>(s, at);
    select_sync<kWave>();
    uint32_t key[KEYS];
#pragma unroll
    for (int e = 0; e < KEYS; e++) {
        const uint32_t i = at.lane + e * kWave;
        key[e] = i < at.n ? (uint32_t)(s.key[at.wave][i] >> 32) : 0u;
    }
    const uint32_t t = lowest_bound<NT>(s, at, wave_bound<KEYS>(key, share));
    uint32_t kept = 0;
#pragma unroll
    for (int e = 0; e < KEYS; e++) {
        const uint32_t i = at.lane + e * kWave;
        const bool in = i < at.n && key[e] >= t;
        const uint64_t ins = __ballot(in);
        if (!ins) continue;
        const uint32_t low = (uint32_t)s.key[at.wave][i < at.n ? i : 0];
        select_sync<kWave>();
        if (in) s.key[at.wave][kept + lanes_below(ins)] = ((uint64_t)key[e] << 32) | low;
        select_sync<kWave>();
        kept += (uint32_t)__popcll(ins);
    }
    at.n = at.keyed = kept;
    return t;
}

// The row again, NT x 4 values at a time, with room made before each.  (64 of 32000 in 8192 rows, 179 us where this is not needed: rows in
// rising order 2150 us, one number in a hundred among zeros 370, four different values 273.)
template <int NT, int SEG>
__device__ void select_slowly(Select<NT, SEG>& s, Place& at, const float* row, uint32_t cols, uint32_t k) {
    const uint32_t whole = cols & ~3u;
    Bound bound = bound_of(0u);
    at.n = at.keyed = 0;
    for (uint32_t c0 = 0; c0 < cols; c0 += 4 * NT) {  // (the last round may hold nothing but the tail)
        if (select_most<NT>(s, at) > SEG - 5 * kWave) bound = select_cut<NT>(s, at, k);
        push_piece<NT, true>(s, at, row_piece(row + c0, bytes_from(c0, whole), 16 * at.tid), c0 + 4 * at.tid, whole, bound.low);
        if (cols - c0 <= 4 * NT) push_tail<NT>(s, at, row, whole, cols, bound.low);
        select_sync<NT>();
    }
}

// The candidates of a row, at least k of them, its k largest among them.
// BEYOND: rows may be longer than the tile.
// v: the row's tile (load_tile); `next` (null: none): the row whose tile takes its place while this row's candidates are sorted out.
template <int NT, int VPT, bool BEYOND>
__device__ __forceinline__ void load_tile(float4u (&v)[VPT], const Place& at, const float* row, uint32_t cols) {
#pragma unroll
    for (int u = 0; u < VPT; u++)
        v[u] = BEYOND ? __builtin_nontemporal_load(reinterpret_cast<const float4u*>(row) + at.tid + u * NT)
                      : row_piece(row, bytes_from(0, cols & ~3u), 16 * (at.tid + u * NT));
}
template <int NT, int VPT, int U, bool BEYOND, int SEG>
__device__ __forceinline__ void select_row(Select<NT, SEG>& s, Place& at, float4u (&v)[VPT], const float* row, const float* next,
                                           uint32_t cols, uint32_t k) {
    constexpr uint32_t kTile = 4 * NT * VPT;
    constexpr uint32_t kStep = 4 * NT * U;  // columns of the pieces that are looked through or on their way at a time
    const uint32_t whole = cols & ~3u;
    // behind the tile a step of pieces is looked through while the next one is on its way
    float4u w[2][U];
    auto load = [&](float4u (&to)[U], uint32_t c0) {
#pragma unroll
        for (int u = 0; u < U; u++)
            to[u] = __builtin_nontemporal_load(reinterpret_cast<const float4u*>(row + c0) + at.tid + u * NT);
    };
    float4u top = v[0];
#pragma unroll
    for (int u = 1; u < VPT; u++)
#pragma unroll
        for (int e = 0; e < 4; e++) top[e] = larger(top[e], v[u][e]);
    // each wave bounds its share of k by its own groups, without waiting for the others
    const uint32_t share = (k + Select<NT>::kWaves - 1) / Select<NT>::kWaves;
    uint32_t t;
    if (share <= 32) {  // 64 groups do for a small share, a quarter of the counting
        const uint32_t one[1] = {order_key(larger(larger(top[0], top[1]), larger(top[2], top[3])))};
        t = wave_bound<1>(one, share);
    } else {
        const uint32_t four[4] = {order_key(top[0]), order_key(top[1]), order_key(top[2]), order_key(top[3])};
        t = wave_bound<4>(four, share);
    }
    Bound bound = bound_of(lowest_bound<NT>(s, at, t));
    at.n = at.keyed = 0;
#pragma unroll
    for (int u = 0; u < VPT; u++) push_piece<NT, !BEYOND>(s, at, v[u], 4 * (at.tid + u * NT), whole, bound.low);
    push_tail<NT>(s, at, row, whole, cols, bound.low);
    if constexpr (BEYOND) {
        bool room = true;
        uint32_t c0 = kTile;
        // A look at the number of candidates: a wave by itself raises its bound whenever they are twice k, a workgroup, whose waves
        // have to meet for it, every four steps when LDS fills up.
        auto look = [&]() {
            if constexpr (NT == kWave) {
                if (at.n <= 2 * k + kWave) return;
                room = at.n <= SEG;
                if (!room) return;
                Bound b;
                if (at.n <= kThin * kWave) b = bound_of(select_thin<NT, kThin>(s, at, k));
                else b = select_cut<NT>(s, at, k);
                if (b.key > bound.key) bound = b;
            } else if ((c0 - kTile) % (4 * kStep) == 0) {
                const uint32_t most = select_most<NT>(s, at);
                room = most <= SEG;
                if (!room) return;
                if (most > SEG / 2) {
                    const Bound b = select_cut<NT>(s, at, k);
                    if (b.key > bound.key) bound = b;
                }
                select_sync<NT>();
            }
        };
        if (kTile + kStep <= whole) load(w[0], kTile);
        while (c0 + kStep <= whole) {
            look();
            if (!room) break;
            const bool more = c0 + 2 * kStep <= whole;
            if (more) load(w[1], c0 + kStep);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int u = 0; u < U; u++) push_piece<NT, false>(s, at, w[0][u], c0 + 4 * (at.tid + u * NT), whole, bound.low);
            c0 += kStep;
            if (!more) break;
            if constexpr (NT == kWave) {
                look();
                if (!room) break;
            }
            if (c0 + 2 * kStep <= whole) load(w[0], c0 + kStep);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int u = 0; u < U; u++) push_piece<NT, false>(s, at, w[1][u], c0 + 4 * (at.tid + u * NT), whole, bound.low);
            c0 += kStep;
        }
        if (room && c0 < whole) {  // less than a step
#pragma unroll
            for (int u = 0; u < U; u++)
                push_piece<NT, true>(s, at, row_piece(row + c0, bytes_from(c0, whole), 16 * (at.tid + u * NT)), c0 + 4 * (at.tid + u * NT),
                                     whole, bound.low);
        }
    }
    if (next) load_tile<NT, VPT, BEYOND>(v, at, next, cols);
    if (select_most<NT>(s, at) > SEG) {
        select_sync<NT>();
        select_slowly<NT>(s, at, row, cols, k);
    }
    key_candidates<NT>(s, at);
}

// The value of the lane whose number differs in the bits of M.
template <int M>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v) {
    if constexpr (M == 1) return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xb1, 0xf, 0xf, true);        // quad_perm 1 0 3 2
    else if constexpr (M == 2) return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4e, 0xf, 0xf, true);   // quad_perm 2 3 0 1
    else if constexpr (M == 8) return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, true);  // row_ror 8
    else if constexpr (M == 32) return (uint32_t)__shfl_xor((int)v, 32, kWave);
    else return (uint32_t)__builtin_amdgcn_ds_swizzle((int)v, M << 10 | 0x1f);
}
// Bit l: whether element BASE + l keeps the larger of the two that meet in this step of a bitonic network for descending order.
constexpr uint64_t keeps_larger(int base, int size, int stride) {
    uint64_t m = 0;
    for (int l = 0; l < 64; l++)
        if ((((base + l) & stride) == 0) == (((base + l) & size) == 0)) m |= (uint64_t)1 << l;
    return m;
}
template <int KEYS, int SIZE, int STRIDE>
__device__ __forceinline__ void sort_step(uint64_t (&key)[KEYS]) {
    if constexpr (STRIDE >= kWave) {  // (of two keys a lane, the last merge)
        const uint64_t a = key[0], b = key[1];
        key[0] = a > b ? a : b;
        key[1] = a > b ? b : a;
    } else {
        auto step = [&](auto e_tag) {
            constexpr int e = decltype(e_tag)::value;
            constexpr uint64_t larger_mask = keeps_larger(e * kWave, SIZE, STRIDE);
            const uint64_t other = (uint64_t)lane_xor<STRIDE>((uint32_t)(key[e] >> 32)) << 32 | lane_xor<STRIDE>((uint32_t)key[e]);
            const bool keep = __builtin_amdgcn_inverse_ballot_w64(__ballot(key[e] > other) ^ ~larger_mask);
            key[e] = keep ? key[e] : other;
        };
        step(std::integral_constant<int, 0>{});
        if constexpr (KEYS == 2) step(std::integral_constant<int, 1>{});
    }
    if constexpr (STRIDE > 1) sort_step<KEYS, SIZE, STRIDE / 2>(key);
    else if constexpr (SIZE < KEYS * kWave) sort_step<KEYS, SIZE * 2, SIZE>(key);
}
// A wave's candidates sorted in registers, KEYS of them a lane (of 64 keys 21 steps of six instructions; a rank costs four instructions
// and a read of LDS for every two keys).
template <int KEYS, int SEG, class Emit>
__device__ __forceinline__ void emit_sorted(const Select<kWave, SEG>& s, const Place& at, uint32_t k, Emit emit) {
    uint64_t key[KEYS];
#pragma unroll
    for (int e = 0; e < KEYS; e++) {
        const uint32_t i = at.lane + e * kWave;
        key[e] = i < at.n ? s.key[0][i] : 0;
    }
    sort_step<KEYS, 2, 1>(key);
#pragma unroll
    for (int e = 0; e < KEYS; e++)
        if ((uint32_t)(at.lane + e * kWave) < k) emit((uint32_t)(at.lane + e * kWave), key[e]);
}

// The k largest candidates in order: emit(rank, key).
// SORT: for k beyond 16 (the sort's registers slow the rest down: 8 of 600 in 60000 rows 42 us with it in the kernel, 37 without; 64 of
// 1000 in 16384 rows 29 with it, 33 by ranks).
template <int NT, bool SORT, int SEG, class Emit>
__device__ __forceinline__ void select_emit(Select<NT, SEG>& s, Place& at, uint32_t k, Emit emit) {
    constexpr int kWaves = Select<NT>::kWaves;
    uint32_t all = 0;
    auto total = [&]() {
        select_sync<NT>();
        select_most<NT>(s, at);
        all = 0;
        if constexpr (NT == kWave) {
            all = at.n;
        } else {
#pragma unroll
            for (int w = 0; w < kWaves; w++) all += s.n[w];
        }
    };
    total();
    if (SORT && NT == kWave ? all > 2 * kWave : all > k + k / 2 + 16) {
        constexpr int kKeys = NT == kWave ? kThin : 2;
        if (select_most<NT>(s, at) <= kKeys * kWave) {
            select_thin<NT, kKeys>(s, at, (k + kWaves - 1) / kWaves);
            total();
        }
    }
    if constexpr (NT == kWave && SORT) {
        if (all <= kWave) return emit_sorted<1>(s, at, k, emit);
        if (all <= 2 * kWave) return emit_sorted<2>(s, at, k, emit);
    }
    if (all > kRankMost && all > k) {
        select_cut<NT>(s, at, k);
        total();
    }
    if (at.lane < 2) s.key[at.wave][at.n + at.lane] = 0;
    select_sync<NT>();
    // the threads take the candidates of all waves in turn
    for (uint32_t i = at.tid; i < all; i += NT) {
        uint64_t mine;
        if constexpr (NT == kWave) {
            mine = s.key[0][i];
        } else {
            uint32_t j = i;
            int w = 0;
            while (j >= s.n[w]) j -= s.n[w++];
            mine = s.key[w][j];
        }
        uint32_t rank = 0;
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
            const uint32_t n = NT == kWave ? at.n : s.n[w];
#pragma unroll 8
            for (uint32_t j = 0; j < n; j += 2) rank += (uint32_t)(s.key[w][j] > mine) + (uint32_t)(s.key[w][j + 1] > mine);
        }
        if (rank < k) emit(rank, mine);
    }
}

template <int NT, int VPT, int U, bool BEYOND, bool SORT, int SEG, int PER_CU>
__global__ __launch_bounds__(256, PER_CU) void topk_kernel(const float* x, float* values, uint64_t* indices, size_t rows, uint32_t cols,
                                                      uint32_t k) {
    constexpr int kRows = 256 / NT;
    __shared__ Select<NT, SEG> mem[kRows];
    const int w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x / kWave));  // scalars: the row and its pieces' base are then too
    Place at{(int)(threadIdx.x % NT), NT == kWave ? 0 : w, (int)(threadIdx.x % kWave), 0u, 0u};
    const int sub = NT == kWave ? w : 0;
    Select<NT, SEG>& s = mem[sub];
    const size_t step = (size_t)gridDim.x * kRows;
    size_t r = (size_t)blockIdx.x * kRows + sub;
    if (r >= rows) return;  // (only waves that own a row of their own: no barrier is missed)
    float4u v[VPT];
    load_tile<NT, VPT, BEYOND>(v, at, x + r * cols, cols);
    for (; r < rows; r += step) {
        const float* row = x + r * cols;
        select_row<NT, VPT, U, BEYOND>(s, at, v, row, r + step < rows ? x + (r + step) * cols : nullptr, cols, k);
        select_emit<NT, SORT>(s, at, k, [&](uint32_t rank, uint64_t key) {
            const uint32_t c = ~(uint32_t)key;
            float v = key_value((uint32_t)(key >> 32));
            if (v == 0.f || v != v) v = row[c];  // the key knows neither the sign of a zero nor which NaN it was
            values[r * k + rank] = v;
            indices[r * k + rank] = c;
        });
        select_sync<NT>();
    }
}

// A few long rows: a workgroup per segment of a row leaves the segment's k largest, in order, as keys with the row's columns ...
constexpr uint32_t kTopkSegment = 4096;
__global__ __launch_bounds__(256, 4) void topk_segments_kernel(const float* x, uint64_t* keys, uint32_t cols, uint32_t k, uint32_t len,
                                                               uint32_t n_seg) {
    __shared__ Select<256> s;
    Place at{(int)threadIdx.x, __builtin_amdgcn_readfirstlane((int)(threadIdx.x / kWave)), (int)(threadIdx.x % kWave), 0u, 0u};
    const size_t r = blockIdx.x / n_seg;
    const uint32_t seg = blockIdx.x % n_seg, c0 = seg * len, n = cols - c0 < len ? cols - c0 : len;
    const float* part = x + r * cols + c0;
    float4u v[4];
    load_tile<256, 4, false>(v, at, part, n);
    select_row<256, 4, 4, false>(s, at, v, part, nullptr, n, k);
    select_emit<256, true>(s, at, k, [&](uint32_t rank, uint64_t key) {
        keys[((size_t)blockIdx.x) * k + rank] = (key & ~(uint64_t)0xffffffffu) | (uint32_t)~(~(uint32_t)key + c0);
    });
}
// ... and a workgroup per row takes the k largest of those.  Each segment's share-th key is known, and the lowest of them is a bound.
__global__ __launch_bounds__(256, 4) void topk_join_kernel(const float* x, const uint64_t* keys, float* values, uint64_t* indices,
                                                           uint32_t cols, uint32_t k, uint32_t n_seg) {
    __shared__ Select<256> s;
    __shared__ uint64_t bounds[4];
    Place at{(int)threadIdx.x, __builtin_amdgcn_readfirstlane((int)(threadIdx.x / kWave)), (int)(threadIdx.x % kWave), 0u, 0u};
    const size_t r = blockIdx.x;
    const uint64_t* list = keys + r * n_seg * k;
    const uint32_t share = (k + n_seg - 1) / n_seg, total = n_seg * k;
    uint64_t low = ~(uint64_t)0;
    for (uint32_t i = threadIdx.x; i < n_seg; i += 256) {
        const uint64_t b = list[(size_t)i * k + share - 1];
        low = b < low ? b : low;
    }
#pragma unroll
    for (int m = kWave / 2; m >= 1; m >>= 1) {
        const uint64_t o = (uint64_t)__shfl_xor((unsigned long long)low, m, kWave);
        low = o < low ? o : low;
    }
    if (at.lane == 0) bounds[at.wave] = low;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; w++) low = bounds[w] < low ? bounds[w] : low;
    for (uint32_t i0 = 0; i0 < total; i0 += 256) {
        if (i0 % (256 * 8) == 0 && i0 && select_most<256>(s, at) > kSegment - 8 * kWave) select_cut<256>(s, at, k);
        const uint64_t key = i0 + threadIdx.x < total ? list[i0 + threadIdx.x] : 0;
        const uint64_t ins = __ballot(key >= low && key != 0);
        if (key >= low && key != 0) s.key[at.wave][at.n + lanes_below(ins)] = key;
        at.n += (uint32_t)__popcll(ins);
        at.keyed = at.n;
        if (i0 % (256 * 8) == 0) __syncthreads();
    }
    select_emit<256, true>(s, at, k, [&](uint32_t rank, uint64_t key) {
        const uint32_t c = ~(uint32_t)key;
        float v = key_value((uint32_t)(key >> 32));
        if (v == 0.f || v != v) v = x[r * cols + c];
        values[r * k + rank] = v;
        indices[r * k + rank] = c;
    });
}

// Short rows and few of their values chosen (a router's scores): L lanes share a row, each holding KPL adjacent columns as keys in
// registers, and the largest is taken out k times (8 of 128 in 65536 rows: 15 us, a wave per row with a bound and candidates 29 us).
// A round is a handful of maxima across the lanes; a tie goes to the lowest lane and there to the lowest column, which is the lowest
// column of the row.
template <int L>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
    auto step = [&](auto ctrl) {
        const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(ctrl)::value, 0xf, 0xf, false);
        v = o > v ? o : v;
    };
    step(std::integral_constant<int, 0xB1>{});  // neighbours in pairs
    step(std::integral_constant<int, 0x4E>{});  // pairs in quads
    if (L == 16) {
        step(std::integral_constant<int, 0x124>{});  // rotations of the 16 by a quad and by two
        step(std::integral_constant<int, 0x128>{});
    }
    return v;
}
template <int L, int KPL>
__global__ __launch_bounds__(256) void topk_short_kernel(const float* x, float* values, uint64_t* indices, size_t rows, uint32_t cols,
                                                         uint32_t k) {
    const size_t r = (size_t)blockIdx.x * (256 / L) + threadIdx.x / L;
    const uint32_t lane = threadIdx.x % L, first = lane * KPL;
    const bool live = r < rows;
    const float* row = x + (live ? r : 0) * cols;
    uint32_t key[KPL];
#pragma unroll
    for (int p = 0; p < KPL; p += 4) {
        const uint32_t c = first + p;
        if (live && c + 4 <= cols) {
            const float4u v = __builtin_nontemporal_load(reinterpret_cast<const float4u*>(row + c));
#pragma unroll
            for (int e = 0; e < 4; e++) key[p + e] = order_key(v[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) key[p + e] = live && c + e < cols ? order_key(row[c + e]) : 0u;
        }
    }
    for (uint32_t j = 0; j < k; j++) {
        uint32_t mine = key[0];
#pragma unroll
        for (int e = 1; e < KPL; e++) mine = key[e] > mine ? key[e] : mine;
        const uint32_t top = lanes_max<L>(mine);
        const uint32_t shift = threadIdx.x & (kWave - 1) & ~(L - 1);
        const uint32_t holders = (uint32_t)(__ballot(mine == top) >> shift) & ((1u << L) - 1);
        if ((uint32_t)__builtin_ctz(holders) == lane) {
            uint32_t at = 0;
            bool found = false;
#pragma unroll
            for (int e = 0; e < KPL; e++) {
                const bool hit = !found && key[e] == top;
                at = hit ? (uint32_t)e : at;
                key[e] = hit ? 0u : key[e];
                found = found || hit;
            }
            if (live) {
                float v = key_value(top);
                if (v == 0.f || v != v) v = row[first + at];  // the key knows neither the sign of a zero nor which NaN it was
                values[r * k + j] = v;
                indices[r * k + j] = first + at;
            }
        }
    }
}

// A row's chosen places in LDS: entry j holds its column (kNoCol: none), and only the first of the entries that name a
// column speaks for it.
constexpr uint32_t kNoCol = 0xffffffffu;
// The gradient of a selection, dense, for short rows and few places: 16 lanes share a row, every lane compares its columns with each
// chosen one (the gradients of a repeated index are added in the order of j by themselves).
template <int P>  // pieces of four columns a lane has: 64 P columns at most
__global__ __launch_bounds__(256) void topk_bwd_short_kernel(const uint64_t* indices, const float* y_g, float* x_g, size_t rows,
                                                             uint32_t cols, uint32_t k) {
    const size_t r = (size_t)blockIdx.x * 16 + threadIdx.x / 16;
    if (r >= rows) return;
    const uint64_t* idx = indices + r * k;
    const float* g = y_g + r * k;
    float* row = x_g + r * cols;
    const uint32_t first = threadIdx.x % 16 * 4;
    float4u v[P];
#pragma unroll
    for (int p = 0; p < P; p++) v[p] = float4u{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (uint32_t j = 0; j < k; j++) {
        const uint64_t c = idx[j];
        const uint32_t at = c < cols ? (uint32_t)c - first : ~0u - 255u;  // no lane's column
        const float a = g[j];
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int e = 0; e < 4; e++) v[p][e] = at == (uint32_t)(64 * p + e) ? __fadd_rn(v[p][e], a) : v[p][e];
    }
#pragma unroll
    for (int p = 0; p < P; p++) {
        const uint32_t c = first + 64 * p;
        if (c + 4 <= cols) {
            __builtin_nontemporal_store(v[p], reinterpret_cast<float4u*>(row + c));
        } else {
#pragma unroll
            for (int e = 0; e < 3; e++)
                if (c + e < cols) row[c + e] = v[p][e];
        }
    }
}

// The lanes of `among` that hold the same number of `bits` bits as this one.
__device__ __forceinline__ uint64_t same_lanes(uint32_t v, int bits, uint64_t among) {
    for (int b = 0; b < bits; b++) {
        const bool one = (v >> b) & 1u;
        const uint64_t ones = __ballot(one);
        among &= one ? ones : ~ones;
    }
    return among;
}
// Adds the entries of a wave to a row, one a lane: `same`, the lanes that name this lane's column (none: no entry); the lowest of them
// writes, the gradients in the order of the lanes.
__device__ __forceinline__ void add_entries(float* at, float g, uint64_t same, int lane) {
    const bool writes = same != 0 && (same & (((uint64_t)1 << lane) - 1)) == 0;
    float v = writes ? __fadd_rn(*at, g) : g;
    uint64_t rest = writes ? same & (same - 1) : 0;
    while (__any(rest != 0)) {
        const int l = rest ? __builtin_ctzll(rest) : lane;
        const float a = __shfl(g, l, kWave);
        if (rest) v = __fadd_rn(v, a);
        rest &= rest - 1;
    }
    if (writes) *at = v;
}

// The same for any row: NT threads (a wave up to 1024 columns, else a workgroup for each of even spans) put together up to 16 NT columns in
// LDS: zeros, then the entries, which one wave adds 64 at a time, then whole pieces to memory.  (64 of 32000 in 8192 rows: 202 us, 5.2
// TB/s; clearing the span in memory and writing the entries after it, each a part of a line, 241.  Stores past the cache take 23
// us for 583 rows of 41270, these 15.  65536 rows of 300 by workgroups: 54 us, by waves 19.)
__device__ __forceinline__ void stores_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
template <int NT>
__global__ __launch_bounds__(256) void topk_bwd_kernel(const uint64_t* indices, const float* y_g, float* x_g, size_t rows,
                                                       uint32_t cols, uint32_t k, uint32_t spans, uint32_t span_cols, int bits) {
    constexpr uint32_t kSpan = 16 * NT;
    __shared__ __attribute__((aligned(16))) float span_mem[256 / NT * kSpan];
    const int lane = threadIdx.x % kWave, tid = threadIdx.x % NT;
    const int sub = __builtin_amdgcn_readfirstlane((int)(threadIdx.x / NT));
    float* const span = span_mem + sub * kSpan;
    const size_t job = (size_t)blockIdx.x * (256 / NT) + sub, r = job / spans;
    if (r >= rows) return;  // (only waves with rows of their own: no barrier is missed)
    const uint32_t c0 = (uint32_t)(job - r * spans) * span_cols, n = cols - c0 < span_cols ? cols - c0 : span_cols;
    float* row = x_g + r * cols + c0;
    uint64_t idx = ~(uint64_t)0;
    float g = 0.f;
    if (tid < kWave && (uint32_t)lane < k) {
        idx = indices[r * k + lane];
        g = y_g[r * k + lane];
    }
    for (uint32_t c = 4 * tid; c < n; c += 4 * NT) *reinterpret_cast<float4*>(span + c) = make_float4(0.f, 0.f, 0.f, 0.f);
    select_sync<NT>();
    if (tid < kWave) {
        for (uint32_t j0 = 0;;) {
            const uint64_t at = idx - c0;
            const bool here = at < n;
            const uint64_t heres = __ballot(here);
            if (heres) {
                const uint32_t col = here ? (uint32_t)at : 0u;
                uint64_t same = same_lanes(col, bits, heres);
                if (!here) same = 0;
                add_entries(span + col, here ? g : 0.f, same, lane);
                select_sync<kWave>();
            }
            j0 += kWave;
            if (j0 >= k) break;
            const bool live = j0 + lane < k;
            idx = live ? indices[r * k + j0 + lane] : ~(uint64_t)0;
            g = live ? y_g[r * k + j0 + lane] : 0.f;
        }
    }
    select_sync<NT>();
    uint32_t c = 4 * tid;
    for (; c + 4 <= n; c += 4 * NT) *reinterpret_cast<float4u*>(row + c) = *reinterpret_cast<const float4u*>(span + c);
    for (; c < n; c++) row[c] = span[c];
}
// Adding to what is there: a wave takes as many rows as it has lanes for, or one of more than 64 places.
__global__ __launch_bounds__(256) void topk_bwd_add_kernel(const uint64_t* indices, const float* y_g, float* x_g, size_t rows,
                                                           uint32_t cols, uint32_t k, int bits) {
    const int lane = threadIdx.x % kWave;
    const uint32_t wide = k < kWave ? k : kWave;  // entries of a row the wave takes at a time
    const uint32_t per_wave = kWave / wide, mine = lane / wide, j_lane = lane % wide;
    const uint64_t row_lanes = wide == kWave ? ~(uint64_t)0 : (((uint64_t)1 << wide) - 1) << (mine * wide % kWave);
    for (size_t r0 = ((size_t)blockIdx.x * 4 + threadIdx.x / kWave) * per_wave; r0 < rows; r0 += (size_t)gridDim.x * 4 * per_wave) {
        const size_t r = r0 + mine;
        for (uint32_t j0 = 0; j0 < k; j0 += wide) {
            if (j0) stores_done();
            const bool live = mine < per_wave && r < rows && j0 + j_lane < k;
            const size_t i = r * k + j0 + j_lane;
            const uint64_t idx = live ? indices[i] : ~(uint64_t)0;
            const bool here = idx < cols;
            const uint32_t col = here ? (uint32_t)idx : 0u;
            uint64_t same = same_lanes(col, bits, __ballot(here) & row_lanes);
            if (!here) same = 0;
            add_entries(x_g + (here ? r : 0) * cols + col, here ? y_g[i] : 0.f, same, lane);
        }
    }
}

// ------------------------------------------------------------------------------------------------
// Distillation.  With c = log2(e) / T and m, tm the largest logit of the student and the teacher:
//   e_c = 2^((x_c - m) c), s = sum e_c, p_c = e_c / s      f_j = 2^((t_j - tm) c), S = sum f_j, q_j = f_j / S
//   row_loss = T^2 (sum_j f_j ((t_j - tm) - (x_{i_j} - m)) / T / S - log S + log s)
// A row's logits are read once, into registers, by 16 lanes, a wave, or a workgroup of 256, 512 or 1024, by its length (the loss alone
// reads rows of more than 32768 columns with a running maximum; for more than 65536 the gradient reads them again); the maxima, then
// all sums, take one reduction each.  Bound by memory: 8192 x 32000 forward 159 us, 6.6 TB/s.  In the gradient of rows of up to 2048
// columns the q_j go into a stretch of LDS laid out like the row, from where every thread takes what belongs to its columns; of longer
// rows the few classes that have a share are written a second time.  Either way a class that is named twice gets both shares,
// added in the order of j.
// ------------------------------------------------------------------------------------------------
struct DistillArgs {
    const float* x;
    const float* t;
    const uint64_t* idx;
    const float* w;
    float* stats;
    float* row_loss;
    float* grad;
    size_t rows;
    uint32_t cols, k;
    float temp, inv_temp, scale, mean;  // scale = log2(e) / temp
    uint32_t segments, segment;         // the gradient alone: parts of a row, and their columns
    bool once;                          // more is read than the memory-side cache holds: loads leave nothing there

    DistillArgs part(size_t first, size_t n) const {  // n rows from `first` on
        DistillArgs a = *this;
        a.x += first * cols;
        a.t += first * k;
        a.idx += first * k;
        if (w) a.w += first;
        a.stats += 2 * first;
        if (row_loss) a.row_loss += first;
        if (grad) a.grad += first * cols;
        a.rows = n;
        return a;
    }
};

// Loads that pass by the memory-side cache (256 MB) win as soon as it can not hold what is read (logits, an old gradient: 16384 x
// 10001 forward 171 -> 109 us, 8192 x 32000 168 -> 159; 8000 x 8000 added to the gradient 149 -> 131) and lose before (1000 x
// 50257 step 71 -> 85 us, 5000 x 10000 70 -> 77); in between both take the same (1500 x 50257: step 118 and 124, forward 61 and 60).
constexpr size_t kCachedFloats = (size_t)80 << 20;

// the hardware's 2^x: off by a step at most, which with the roundings of its argument is what exp(x) of a library has lost as well
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// The largest of `top` and the sum of each of `sum` over the NT threads of a row, in all of them.  `smem`: 4 (NT / 64) floats.
template <int NT, int N>
__device__ __forceinline__ void row_sums(float (&sum)[N], float* smem) {
    constexpr int W = NT < kWave ? NT : kWave;
#pragma unroll
    for (int m = W / 2; m >= 1; m >>= 1)
#pragma unroll
        for (int i = 0; i < N; i++) sum[i] += __shfl_xor(sum[i], m, kWave);
    if constexpr (NT > kWave) {
        const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
        __syncthreads();
        if (lane == 0)
#pragma unroll
            for (int i = 0; i < N; i++) smem[i * (NT / kWave) + wave] = sum[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; i++) {
            float all = smem[i * (NT / kWave)];
            for (int w = 1; w < NT / kWave; w++) all += smem[i * (NT / kWave) + w];
            sum[i] = all;
        }
    }
}
template <int NT, int N>
__device__ __forceinline__ void row_maxima(float (&top)[N], float* smem) {
    constexpr int W = NT < kWave ? NT : kWave;
#pragma unroll
    for (int m = W / 2; m >= 1; m >>= 1)
#pragma unroll
        for (int i = 0; i < N; i++) top[i] = fmaxf(top[i], __shfl_xor(top[i], m, kWave));
    if constexpr (NT > kWave) {
        const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
        __syncthreads();
        if (lane == 0)
#pragma unroll
            for (int i = 0; i < N; i++) smem[i * (NT / kWave) + wave] = top[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; i++) {
            float all = smem[i * (NT / kWave)];
            for (int w = 1; w < NT / kWave; w++) all = fmaxf(all, smem[i * (NT / kWave) + w]);
            top[i] = all;
        }
    }
}

// What the row's numbers come to once they are known: the statistics, the loss and the factors of the gradient.
struct RowResult {
    float m, ls, loss;      // stats and row_loss
    float inv_s, inv_S, f;  // p = e inv_s, q = f_j inv_S, gradient = f (p - q)
    bool empty;
};
// m, tm: the maxima as found (-inf: nothing above); s, S, W: the sums, taken from 0 where a maximum is -inf.  With FWD false m and ls
// are the row's statistics and s, W are not looked at.
template <bool FWD>
__device__ __forceinline__ RowResult row_result(const DistillArgs& a, float w, float m, float ls, float s, float S, float W) {
    RowResult r;
    r.m = m;
    r.ls = ls;
    if (FWD) {
        r.ls = logf(s);
        if (m == -INFINITY) {
            if (s != 0.f) r.m = NAN;  // NaNs among logits of -inf
            else r.ls = 0.f;
        }
        r.inv_s = __fdiv_rn(1.f, s);
    } else {
        r.inv_s = expf(-ls);
    }
    r.empty = S == 0.f || r.m == -INFINITY;
    r.loss = r.empty ? 0.f : (W / S - logf(S) + r.ls) * (a.temp * a.temp);
    r.inv_S = __fdiv_rn(1.f, S);
    r.f = w * a.temp;
    return r;
}

// An entry of the teacher: its column (kNoCol: padding) and its logit.
__device__ __forceinline__ void teacher_entry(const DistillArgs& a, size_t r, uint32_t j, uint32_t& col, float& t) {
    const bool live = j < a.k;
    const uint64_t c = live ? a.idx[r * a.k + j] : ~(uint64_t)0;
    col = c < a.cols ? (uint32_t)c : kNoCol;
    t = col != kNoCol ? a.t[r * a.k + j] : -INFINITY;
}
// f_j and its part of W: x is the student's logit of the entry's class
__device__ __forceinline__ void teacher_terms(const DistillArgs& a, float t, float x, float from_t, float from_x, float& f, float& part) {
    f = exp2_fast((t - from_t) * a.scale);
    part = f != 0.f ? f * (((t - from_t) - (x - from_x)) * a.inv_temp) : 0.f;
}

// Short rows with at most 16 entries: 16 lanes a row, P pieces of four columns and an entry each.  ONE: the only workgroup, which also
// adds up the loss.
template <int NTB, int P, bool FWD, bool BWD, bool ACC, bool ONE>
__global__ __launch_bounds__(NTB) void distill_short_kernel(DistillArgs a, float* loss) {
    const int lane = threadIdx.x % 16, group = threadIdx.x / 16;
    float total = 0.f;
    for (size_t r0 = (size_t)blockIdx.x * (NTB / 16); r0 < a.rows; r0 += (size_t)gridDim.x * (NTB / 16)) {
        const size_t r = r0 + group;
        const bool live = r < a.rows;
        const float w = live ? (a.w ? a.w[r] : a.mean) : 0.f;
        const bool real = live && w != 0.f;
        const float* x = a.x + (real ? r : 0) * a.cols;
        float* grad = BWD ? a.grad + (real ? r : 0) * a.cols : nullptr;
        float v[4 * P], old[4 * P];
#pragma unroll
        for (int p = 0; p < P; p++) {
            const uint32_t c = 64 * p + 4 * lane;
            if (real && c + 4 <= a.cols) {
                const float4u xs = *reinterpret_cast<const float4u*>(x + c);
                float4u gs = {0.f, 0.f, 0.f, 0.f};
                if (ACC) gs = *reinterpret_cast<const float4u*>(grad + c);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    v[4 * p + e] = xs[e];
                    old[4 * p + e] = gs[e];
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    v[4 * p + e] = real && c + e < a.cols ? x[c + e] : -INFINITY;
                    old[4 * p + e] = ACC && real && c + e < a.cols ? grad[c + e] : 0.f;
                }
            }
        }
        uint32_t col = kNoCol;
        float t = -INFINITY;
        if (real) teacher_entry(a, r, lane, col, t);
        const float xe = FWD && col != kNoCol ? x[col] : 0.f;
        float top[2] = {t, -INFINITY};
        if (FWD) {
#pragma unroll
            for (int i = 0; i < 4 * P; i++) top[1] = fmaxf(top[1], v[i]);
        }
        row_maxima<16, 2>(top, nullptr);
        const float m = FWD ? top[1] : (real ? a.stats[2 * r] : 0.f), ls = FWD ? 0.f : (real ? a.stats[2 * r + 1] : 0.f);
        const float from_x = m == -INFINITY ? 0.f : m, from_t = top[0] == -INFINITY ? 0.f : top[0];
        float sum[3] = {0.f, 0.f, 0.f};  // s, S, W
#pragma unroll
        for (int i = 0; i < 4 * P; i++) {
            v[i] = exp2_fast((v[i] - from_x) * a.scale);
            sum[0] += v[i];
        }
        float f, part;
        teacher_terms(a, t, xe, from_t, from_x, f, part);
        sum[1] = f;
        sum[2] = part;
        row_sums<16, 3>(sum, nullptr);
        const RowResult res = row_result<FWD>(a, w, m, ls, sum[0], sum[1], sum[2]);
        if (FWD && live && lane == 0) {
            a.stats[2 * r] = real ? res.m : 0.f;
            a.stats[2 * r + 1] = real ? res.ls : 0.f;
            const float l = real ? res.loss : 0.f;
            a.row_loss[r] = l;
            if (ONE && real) total += a.w ? w * l : l;
        }
        if (BWD) {
            const bool zero = !real || res.empty;
            float share[4 * P];
#pragma unroll
            for (int i = 0; i < 4 * P; i++) share[i] = 0.f;
            const float q = f * res.inv_S;
            for (uint32_t j = 0; j < a.k; j++) {
                const uint32_t at = (uint32_t)__shfl((int)col, j, 16) - 4 * lane;
                const float qj = __shfl(q, j, 16);
#pragma unroll
                for (int i = 0; i < 4 * P; i++) share[i] = at == (uint32_t)((i / 4) * 64 + i % 4) ? share[i] + qj : share[i];
            }
            if (live && !(ACC && zero)) {
                float* g = a.grad + r * a.cols;
#pragma unroll
                for (int p = 0; p < P; p++) {
                    const uint32_t c = 64 * p + 4 * lane;
                    float4u d;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int i = 4 * p + e;
                        d[e] = zero ? 0.f : res.f * (v[i] * res.inv_s - share[i]);
                        if (ACC) d[e] = old[i] + d[e];
                    }
                    if (c + 4 <= a.cols) {
                        *reinterpret_cast<float4u*>(g + c) = d;
                    } else {
#pragma unroll
                        for (int e = 0; e < 3; e++)
                            if (c + e < a.cols) g[c + e] = d[e];
                    }
                }
            }
        }
    }
    if constexpr (ONE) {
        __shared__ float smem[NTB / kWave];
        total = block_reduce<SumAcc>(total, smem);
        if (threadIdx.x == 0) *loss = a.w ? total : __fdiv_rn(total, (float)a.rows);
    }
}

// The q_j into the stretch of n zeros `span`, by one wave, in the order of j.
__device__ __forceinline__ void span_shares(float* span, const uint32_t* col, const float* q, uint32_t k, uint32_t n, int bits, int lane) {
    for (uint32_t j0 = 0; j0 < k; j0 += kWave) {
        const uint32_t at = j0 + lane < k ? col[j0 + lane] : kNoCol;
        const bool here = at < n;
        const uint64_t heres = __ballot(here);
        if (!heres) continue;
        uint64_t same = same_lanes(here ? at : 0u, bits, heres);
        if (!here) same = 0;
        add_entries(span + (here ? at : 0u), here ? q[j0 + lane] : 0.f, same, lane);
        select_sync<kWave>();
    }
}

// NT threads a row (a wave: four rows a workgroup), which they hold in VPT pieces of four columns each.  The gradient (of rows of a wave
// only) takes its shares from a stretch of LDS.  ENTRIES: the teacher's that a thread has, at most.
template <int NT, int VPT, int ENTRIES, bool FWD, bool BWD, bool ACC>
__global__ __launch_bounds__(NT < 256 ? 256 : NT, NT == 1024 ? 8 : 1) void distill_row_kernel(DistillArgs a) {
    static_assert(!BWD || NT == kWave, "one wave fills the stretch and reads it");
    constexpr int kRows = NT < 256 ? 256 / NT : 1;
    constexpr uint32_t kSpan = 4 * NT * VPT;
    constexpr int kBits = VPT == 2 ? 9 : VPT == 4 ? 10 : 11;
    static_assert(!BWD || kSpan == 1u << kBits, "bits of a column");
    __shared__ __attribute__((aligned(16))) float span_mem[BWD ? kRows * kSpan : 4];
    __shared__ uint32_t col_mem[BWD ? kRows * ENTRIES * NT : 1];
    __shared__ float q_mem[BWD ? kRows * ENTRIES * NT : 1];
    __shared__ float smem[NT > kWave ? 3 * (NT / kWave) : 1];
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x / kWave));
    const int sub = NT == kWave ? wave : 0, tid = threadIdx.x % NT;
    float* const span = span_mem + (BWD ? sub * kSpan : 0);
    uint32_t* const col_of = col_mem + (BWD ? sub * ENTRIES * NT : 0);
    float* const q_of = q_mem + (BWD ? sub * ENTRIES * NT : 0);
    const size_t r = (size_t)blockIdx.x * kRows + sub;
    if (r >= a.rows) return;  // only waves that own a row of their own: no barrier is missed
    const uint32_t cols = a.cols, whole = cols & ~3u;
    const float* x = a.x + r * cols;
    float* grad = BWD ? a.grad + r * cols : nullptr;
    const float w = a.w ? a.w[r] : a.mean;
    if (w == 0.f) {
        if (FWD && tid == 0) {
            a.stats[2 * r] = a.stats[2 * r + 1] = 0.f;
            a.row_loss[r] = 0.f;
        }
        if (BWD && !ACC) {
            for (uint32_t c = 4 * tid; c < whole; c += 4 * NT) *reinterpret_cast<float4u*>(grad + c) = float4u{0.f, 0.f, 0.f, 0.f};
            if (whole + tid < cols) grad[whole + tid] = 0.f;
        }
        return;
    }
    float4u v[VPT];
    row_pieces<VPT>(v, x, bytes_from(0, whole), 16 * tid, 16 * NT, a.once);
    const float tail = whole + tid < cols ? x[whole + tid] : -INFINITY;  // of the first threads
    uint32_t col[ENTRIES];
    float t[ENTRIES], xe[ENTRIES];
    float top[2] = {-INFINITY, tail};
#pragma unroll
    for (int i = 0; i < ENTRIES; i++) {
        if (i == 0 || i * NT < (int)a.k) {
            teacher_entry(a, r, tid + i * NT, col[i], t[i]);
            xe[i] = FWD && col[i] != kNoCol ? x[col[i]] : 0.f;
            top[0] = fmaxf(top[0], t[i]);
        } else {
            col[i] = kNoCol;
            t[i] = -INFINITY;
            xe[i] = 0.f;
        }
    }
    if (BWD) {
#pragma unroll
        for (int u = 0; u < VPT; u++) *reinterpret_cast<float4*>(span + 4 * (tid + u * NT)) = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float m, ls;
    if (FWD) {
#pragma unroll
        for (int u = 0; u < VPT; u++)
#pragma unroll
            for (int e = 0; e < 4; e++) top[1] = fmaxf(top[1], v[u][e]);
        row_maxima<NT, 2>(top, smem);
        m = top[1];
        ls = 0.f;
    } else {
        float one[1] = {top[0]};
        row_maxima<NT, 1>(one, smem);
        top[0] = one[0];
        m = a.stats[2 * r];
        ls = a.stats[2 * r + 1];
    }
    const float from_x = m == -INFINITY ? 0.f : m, from_t = top[0] == -INFINITY ? 0.f : top[0];
    float sum[3] = {0.f, 0.f, 0.f};
    float f[ENTRIES];
#pragma unroll
    for (int i = 0; i < ENTRIES; i++) {
        float part;
        teacher_terms(a, t[i], xe[i], from_t, from_x, f[i], part);
        sum[0] += f[i];
        sum[1] += part;
    }
#pragma unroll
    for (int u = 0; u < VPT; u++) {
#pragma unroll
        for (int e = 0; e < 4; e++) v[u][e] = exp2_fast((v[u][e] - from_x) * a.scale);
        sum[2] += (v[u][0] + v[u][1]) + (v[u][2] + v[u][3]);
    }
    const float tail_e = exp2_fast((tail - from_x) * a.scale);
    sum[2] += tail_e;
    if (FWD) {
        row_sums<NT, 3>(sum, smem);
    } else {
        float one[1] = {sum[0]};
        row_sums<NT, 1>(one, smem);
        sum[0] = one[0];
    }
    const RowResult res = row_result<FWD>(a, w, m, ls, sum[2], sum[0], sum[1]);
    if (FWD && tid == 0) {
        a.stats[2 * r] = res.m;
        a.stats[2 * r + 1] = res.ls;
        a.row_loss[r] = res.loss;
    }
    if constexpr (BWD) {
        if (ACC && res.empty) return;
#pragma unroll
        for (int i = 0; i < ENTRIES; i++) {
            col_of[tid + i * NT] = col[i];
            q_of[tid + i * NT] = f[i] * res.inv_S;
        }
        const float fac = res.empty ? 0.f : res.f, inv_s = res.inv_s;
        float4u old[VPT];
        if (ACC) {
#pragma unroll
            for (int u = 0; u < VPT; u++) old[u] = row_piece(grad, bytes_from(0, whole), 16 * (tid + u * NT));
        }
        select_sync<NT>();
        span_shares(span, col_of, q_of, a.k, kSpan, kBits, tid);
        select_sync<NT>();
#pragma unroll
        for (int u = 0; u < VPT; u++) {
            const uint32_t c = 4 * (tid + u * NT);
            if (c >= whole) continue;
            const float4 q = *reinterpret_cast<const float4*>(span + c);
            const float4u share = {q.x, q.y, q.z, q.w};
            float4u g;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float d = res.empty ? 0.f : fac * (v[u][e] * inv_s - share[e]);
                g[e] = ACC ? old[u][e] + d : d;
            }
            __builtin_nontemporal_store(g, reinterpret_cast<float4u*>(grad + c));
        }
        if (whole + tid < cols) {
            const float d = res.empty ? 0.f : fac * (tail_e * inv_s - span[whole + tid]);
            grad[whole + tid] = ACC ? grad[whole + tid] + d : d;
        }
    }
}

// The gradient of rows of more than 2048 columns, with the loss (FWD) by a workgroup for the whole row, without it (the statistics are
// known) by one for each segment of a row.  R pieces of four columns a thread are held in registers and L in LDS.  A stretch of
// shares would cost a barrier for every part of the row it covers: the gradient is written without them, and once that is done the thread
// of the first of a class's entries writes the class's gradient again, from the logit that it read.
// Rows of 32769 to 53248 columns fit twice on a compute unit that way, so that one is read or written while the other is summed
// up.  (2048 x 50257, k = 100: 165 us against 189 with the row in registers and shares from LDS; 8192 x 32000: 355 against 394; added
// to an old gradient, whose pieces take the registers: 221 against 250 and 496 against 581.)
template <int NT, int R, int L, bool FWD, bool ACC, bool ONCE>
__global__ __launch_bounds__(NT, R <= (ACC ? 4 : 9) ? 8 : 4) void distill_grad_kernel(DistillArgs a) {
    static_assert(!ACC || L == 0, "old pieces of those in LDS");
    constexpr uint32_t kCols = 4 * NT * (R + L);
    constexpr int kEntries = (kMaxK + NT - 1) / NT;
    constexpr int kBatch = ACC ? (R < 8 ? R : 8) : 1;  // old pieces on their way at a time, the first before the sums
    __shared__ float4 held[L ? L * NT : 1];
    __shared__ uint32_t col_of[kMaxK];
    __shared__ float q_of[kMaxK];
    __shared__ float smem[3 * (NT / kWave)];
    __shared__ uint32_t named[kCols / 32];  // a bit for each class
    __shared__ uint32_t twice;              // whether one is named twice
    const int tid = threadIdx.x;
    const size_t r = FWD ? blockIdx.x : blockIdx.x / a.segments;
    const uint32_t first = FWD ? 0u : (uint32_t)(blockIdx.x - r * a.segments) * a.segment;
    const uint32_t cols = FWD || a.cols - first < a.segment ? a.cols - first : a.segment;
    const float* x = a.x + r * a.cols + first;
    float* grad = a.grad + r * a.cols + first;
    // The pieces begin where 128-byte lines do in a gradient that starts on one, so that no line is written in parts (2048 x 50257: 151
    // against 166 us).  What a row adds up to does not depend on where the arrays lie.  The first threads have a column each of those
    // before and behind the pieces.
    const uint32_t to_line = (uint32_t)(-(r * a.cols + first) & 31), head = to_line < cols ? to_line : cols, whole = (cols - head) & ~3u;
    const uint32_t edge = (uint32_t)threadIdx.x < head ? (uint32_t)threadIdx.x : whole + threadIdx.x;
    const float w = a.w ? a.w[r] : a.mean;
    auto zeros = [&] {
        for (uint32_t c = 4 * tid; c < whole; c += 4 * NT) *reinterpret_cast<float4u*>(grad + head + c) = float4u{0.f, 0.f, 0.f, 0.f};
        if (edge < cols) grad[edge] = 0.f;
    };
    if (w == 0.f) {
        if (FWD && tid == 0) a.stats[2 * r] = a.stats[2 * r + 1] = a.row_loss[r] = 0.f;
        if (!ACC) zeros();
        return;
    }
    for (int i = tid; i < (int)(kCols / 32); i += NT) named[i] = 0;
    if (tid == 0) twice = 0;
    float4u v[R], low[L ? L : 1];  // the first L pieces go to LDS
#pragma unroll
    for (int u = 0; u < L; u++) low[u] = row_piece<ONCE>(x + head, bytes_from(0, whole), 16 * (tid + u * NT));
#pragma unroll
    for (int u = 0; u < R; u++) v[u] = row_piece<ONCE>(x + head, bytes_from(0, whole), 16 * (tid + (L + u) * NT));
    float mx = -INFINITY;
#pragma unroll
    for (int u = 0; u < L; u++) {
#pragma unroll
        for (int e = 0; e < 4; e++) mx = fmaxf(mx, low[u][e]);
        held[tid + u * NT] = make_float4(low[u].x, low[u].y, low[u].z, low[u].w);
    }
    __builtin_amdgcn_sched_barrier(0);  // (nothing else finds room in registers before)
    const float tail = edge < cols ? x[edge] : -INFINITY;
    // entries tid, tid + NT, ... of the teacher; their columns are counted from the segment's first (others lie behind its end)
    uint32_t col[kEntries];
    float t[kEntries], xe[kEntries], f[kEntries], old_e[kEntries];
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < kEntries; i++) {
        teacher_entry(a, r, tid + i * NT, col[i], t[i]);
        col[i] = col[i] == kNoCol ? kNoCol : col[i] - first;
        xe[i] = col[i] < cols ? x[col[i]] : 0.f;
        top[0] = fmaxf(top[0], t[i]);
    }
    float m, ls;
    if (FWD) {
#pragma unroll
        for (int u = 0; u < R; u++)
#pragma unroll
            for (int e = 0; e < 4; e++) mx = fmaxf(mx, v[u][e]);
        top[1] = fmaxf(tail, mx);
        row_maxima<NT, 2>(top, smem);
        m = top[1];
        ls = 0.f;
    } else {
        float one[1] = {top[0]};
        row_maxima<NT, 1>(one, smem);
        top[0] = one[0];
        m = a.stats[2 * r];
        ls = a.stats[2 * r + 1];
    }
    const float from_x = m == -INFINITY ? 0.f : m, from_t = top[0] == -INFINITY ? 0.f : top[0];
    auto power = [&](float value) { return exp2_fast((value - from_x) * a.scale); };
    float sum[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kEntries; i++) {
        float part;
        teacher_terms(a, t[i], xe[i], from_t, from_x, f[i], part);
        sum[0] += f[i];
        sum[1] += part;
    }
#pragma unroll
    for (int u = 0; u < R; u++) {
#pragma unroll
        for (int e = 0; e < 4; e++) v[u][e] = power(v[u][e]);
        sum[2] += (v[u][0] + v[u][1]) + (v[u][2] + v[u][3]);
    }
#pragma unroll
    for (int u = 0; u < L; u++) {
        float4 h = held[tid + u * NT];
        h = make_float4(power(h.x), power(h.y), power(h.z), power(h.w));
        held[tid + u * NT] = h;
        sum[2] += (h.x + h.y) + (h.z + h.w);
    }
    const float tail_e = power(tail);
    sum[2] += tail_e;
    float4u old[kBatch];
    auto load_old = [&](int u0) {
#pragma unroll
        for (int u = u0; u < u0 + kBatch && u < R; u++) old[u - u0] = row_piece<ONCE>(grad + head, bytes_from(0, whole), 16 * (tid + u * NT));
    };
    if (ACC) load_old(0);
    if (FWD) {
        row_sums<NT, 3>(sum, smem);
    } else {
        float one[1] = {sum[0]};
        row_sums<NT, 1>(one, smem);
        sum[0] = one[0];
    }
    const RowResult res = row_result<FWD>(a, w, m, ls, sum[2], sum[0], sum[1]);
    if (FWD && tid == 0) {
        a.stats[2 * r] = res.m;
        a.stats[2 * r + 1] = res.ls;
        a.row_loss[r] = res.loss;
    }
    if (res.empty) {
        if (!ACC) zeros();
        return;
    }
#pragma unroll
    for (int i = 0; i < kEntries; i++) {
        const bool here = col[i] < cols;
        old_e[i] = ACC && here ? grad[col[i]] : 0.f;
        if (tid + i * NT < kMaxK) {
            col_of[tid + i * NT] = col[i];
            q_of[tid + i * NT] = f[i] * res.inv_S;
        }
        if (here && (atomicOr(&named[col[i] / 32], 1u << col[i] % 32) >> col[i] % 32 & 1u)) twice = 1;
    }
    __syncthreads();  // what is added to has been read where entries stand
    const float fac = res.f * res.inv_s;  // of a class without a share
    auto put = [&](uint32_t c, float4u e, float4u add_to) {
        if (c >= whole) return;
        float4u g;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float d = e[i] * fac;
            g[i] = ACC ? add_to[i] + d : d;
        }
        __builtin_nontemporal_store(g, reinterpret_cast<float4u*>(grad + head + c));
    };
    if constexpr (ACC) {
#pragma unroll
        for (int u0 = 0; u0 < R; u0 += kBatch) {
            if (u0) load_old(u0);
#pragma unroll
            for (int u = u0; u < u0 + kBatch && u < R; u++) put(4 * (tid + u * NT), v[u], old[u - u0]);
        }
    } else {
#pragma unroll
        for (int u = 0; u < R; u++) put(4 * (tid + (L + u) * NT), v[u], v[u]);
#pragma unroll
        for (int u = 0; u < L; u++) {
            const float4 h = held[tid + u * NT];
            const float4u e = {h.x, h.y, h.z, h.w};
            put(4 * (tid + u * NT), e, e);
        }
    }
    if (edge < cols) {
        const float d = tail_e * fac;
        grad[edge] = ACC ? grad[edge] + d : d;
    }
    // the classes that the teacher names: their shares in the order of j
    float share[kEntries];
    bool mine[kEntries];
#pragma unroll
    for (int i = 0; i < kEntries; i++) {
        share[i] = f[i] * res.inv_S;
        mine[i] = col[i] < cols;
        if (twice && mine[i]) {
            share[i] = 0.f;
            for (uint32_t j = 0; j < a.k; j++) {
                const bool same = col_of[j] == col[i];
                if (same && j < (uint32_t)(tid + i * NT)) mine[i] = false;
                share[i] = same ? share[i] + q_of[j] : share[i];
            }
        }
    }
    __syncthreads();  // the gradient without shares is written
#pragma unroll
    for (int i = 0; i < kEntries; i++)
        if (mine[i]) {
            const float d = res.f * (power(xe[i]) * res.inv_s - share[i]);
            grad[col[i]] = ACC ? old_e[i] + d : d;
        }
}

// The loss of rows of any length: a workgroup reads the row with a running maximum per thread, whose sum is rescaled when it grows.
constexpr int kStreamNT = 1024;
__global__ __launch_bounds__(kStreamNT, 8) void distill_stream_kernel(DistillArgs a) {
    constexpr int NT = kStreamNT, U = 4;
    __shared__ float smem[3 * (NT / kWave)];
    const int tid = threadIdx.x;
    const uint32_t cols = a.cols, whole = cols & ~3u;
    for (size_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const float* x = a.x + r * cols;
        const float w = a.w ? a.w[r] : a.mean;
        if (w == 0.f) {
            if (tid == 0) a.stats[2 * r] = a.stats[2 * r + 1] = a.row_loss[r] = 0.f;
            continue;
        }
        uint32_t col;
        float t;
        teacher_entry(a, r, tid, col, t);
        const float xe = col != kNoCol ? x[col] : 0.f;
        const float tail = whole + tid < cols ? x[whole + tid] : -INFINITY;
        float mine = -INFINITY, s = 0.f;  // this thread's maximum, and its sum from there
        for (uint32_t c0 = 0; c0 < whole; c0 += 4 * NT * U) {
            float4u v[U];
            row_pieces<U>(v, x + c0, bytes_from(c0, whole), 16 * tid, 16 * NT, a.once);
            float mx = v[0][0];
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int e = 0; e < 4; e++) mx = fmaxf(mx, v[u][e]);
            if (mx > mine) {
                s = mine == -INFINITY ? s : s * exp2_fast((mine - mx) * a.scale);
                mine = mx;
            }
            const float from = mine == -INFINITY ? 0.f : mine;
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int e = 0; e < 4; e++) s += exp2_fast((v[u][e] - from) * a.scale);
        }
        float top[2] = {t, fmaxf(tail, mine)};
        row_maxima<NT, 2>(top, smem);
        const float m = top[1];
        if (mine != -INFINITY) s *= exp2_fast((mine - m) * a.scale);
        const float from_x = m == -INFINITY ? 0.f : m, from_t = top[0] == -INFINITY ? 0.f : top[0];
        float f, part;
        teacher_terms(a, t, xe, from_t, from_x, f, part);
        float sum[3] = {f, part, s + exp2_fast((tail - from_x) * a.scale)};
        row_sums<NT, 3>(sum, smem);
        const RowResult res = row_result<true>(a, w, m, 0.f, sum[2], sum[0], sum[1]);
        if (tid == 0) {
            a.stats[2 * r] = res.m;
            a.stats[2 * r + 1] = res.ls;
            a.row_loss[r] = res.loss;
        }
    }
}

static unsigned row_grid(size_t rows) { return (unsigned)(rows < 65536 ? rows : 65536); }

template <bool FWD, bool BWD, bool ACC>
static int distill_launch(zg_hip_ctx* ctx, DistillArgs a, float* loss, bool* summed) {
    *summed = false;
    if (a.cols <= 256 && a.k <= 16) {
        const size_t blocks = ceil_div_sz(a.rows, 16);
        const dim3 grid((unsigned)(blocks < 65536 ? blocks : 65536));
        // a workgroup of its own for a small batch adds up the loss in the same launch
        const bool one = FWD && a.rows <= 256;
        *summed = one;
#define ZG_SHORT(P)                                                                                                                  \
    do {                                                                                                                             \
        if (one) hipLaunchKernelGGL((distill_short_kernel<1024, P, FWD, BWD, ACC, FWD>), dim3(1), dim3(1024), 0, ctx->stream, a, loss); \
        else hipLaunchKernelGGL((distill_short_kernel<256, P, FWD, BWD, ACC, false>), grid, dim3(256), 0, ctx->stream, a, loss);        \
    } while (0)
        if (a.cols <= 64) ZG_SHORT(1);
        else if (a.cols <= 128) ZG_SHORT(2);
        else ZG_SHORT(4);
#undef ZG_SHORT
        ZG_LAUNCH_CHECK();
        return ZG_HIP_OK;
    }
    // The rows of a launch but the last are a multiple of 32 (a segment has 8192 columns of fewer than 2^31): the gradient's pieces begin
    // where they would in one launch.
#define ZG_ROWS_(NT, VPT, ENTRIES)                                                                                                        \
    do {                                                                                                                                  \
        constexpr size_t threads = NT < 256 ? 256 : NT, per = threads / NT;                                                               \
        in_launches(a.rows, most_groups(threads) * per, [&](size_t first, size_t n) {                                                     \
            hipLaunchKernelGGL((distill_row_kernel<NT, VPT, ENTRIES, FWD, BWD, ACC>), dim3((unsigned)ceil_div_sz(n, per)), dim3(threads), \
                               0, ctx->stream, a.part(first, n));                                                                         \
        });                                                                                                                               \
    } while (0)
#define ZG_ROWS(NT, VPT)                                       \
    do {                                                       \
        if (a.k <= NT && few) ZG_ROWS_(NT, VPT, 1);            \
        else ZG_ROWS_(NT, VPT, (kMaxK + NT - 1) / NT);         \
    } while (0)
#define ZG_GRAD(NT, R, L)                                                                                                              \
    in_launches(a.rows, most_groups(NT) / a.segments / 32 * 32, [&](size_t first, size_t n) {                                          \
        const dim3 grid((unsigned)(n * a.segments));                                                                                   \
        const DistillArgs part = a.part(first, n);                                                                                     \
        if (a.once) hipLaunchKernelGGL((distill_grad_kernel<NT, R, L, FWD, ACC, true>), grid, dim3(NT), 0, ctx->stream, part);         \
        else hipLaunchKernelGGL((distill_grad_kernel<NT, R, L, FWD, ACC, false>), grid, dim3(NT), 0, ctx->stream, part);               \
    })
    // One entry of the teacher a thread where that does (65536 rows of 600, k = 8: step 55 us against 78 with room for 512), but for the
    // gradient that is added to in rows of more than 1024 columns (2000, k = 64: 300 us against 285).
    const bool few = !ACC || a.cols <= 1024;
    // (the gradient alone: even segments)
    a.segments = FWD || a.cols <= 8192 ? 1u : (a.cols - 1) / 8192 + 1;
    a.segment = ((a.cols - 1) / a.segments + 4) & ~3u;
    a.segments = (a.cols - 1) / a.segment + 1;  // as many as have columns
    if (a.cols <= 512) {
        ZG_ROWS(64, 2);
    } else if (a.cols <= 1024) {
        ZG_ROWS(64, 4);
    } else if (a.cols <= 2048) {
        ZG_ROWS(64, 8);
    } else if constexpr (!BWD) {
        if (a.cols <= 4096) ZG_ROWS(64, 16);
        else if (a.cols <= 8192) ZG_ROWS(256, 8);
        else if (a.cols <= 16384) ZG_ROWS(512, 8);
        else if (a.cols <= 32768) ZG_ROWS(1024, 8);
        else hipLaunchKernelGGL(distill_stream_kernel, dim3(row_grid(a.rows)), dim3(kStreamNT), 0, ctx->stream, a);
    } else if (a.segment <= 4096) {
        ZG_GRAD(256, 4, 0);
    } else if (a.segment <= 8192) {
        ZG_GRAD(256, 8, 0);
    } else if constexpr (FWD) {
        if (a.cols <= 16384) {
            ZG_GRAD(1024, 4, 0);
        } else if (a.cols <= 32768) {
            ZG_GRAD(1024, 8, 0);
        } else if (a.cols <= 53248) {
            if constexpr (ACC) ZG_GRAD(1024, 13, 0);
            else ZG_GRAD(1024, 9, 4);
        } else if (a.cols <= 65536) {
            ZG_GRAD(1024, 16, 0);
        } else {
            // Rows that no workgroup holds: the loss, then the gradient.  (2048 x 128000: 514 us, 16 x 128000: 18 us; one kernel that read
            // each row twice took 526 and 36.  Some rows at a time, for the second pass to find them in the memory-side cache,
            // costs more in half-empty launches than it saves: 619 us.)
            bool unused;
            if (int rc = distill_launch<true, false, false>(ctx, a, loss, &unused)) return rc;
            return distill_launch<false, true, ACC>(ctx, a, loss, &unused);
        }
    }
#undef ZG_GRAD
#undef ZG_ROWS
#undef ZG_ROWS_
    ZG_LAUNCH_CHECK();
    return ZG_HIP_OK;
}


static int distill_check(const char* op, const float* logits, const float* teacher, const uint64_t* indices,
                         const float* row_weights, size_t rows, size_t cols, size_t k, float temperature) {
    ZG_REQUIRE(logits && teacher && indices, "%s: null pointer", op);
    ZG_REQUIRE(((uintptr_t)indices & 7u) == 0, "%s: indices are not on an 8-byte boundary", op);
    ZG_REQUIRE(cols < ((size_t)1 << 31), "%s: %zu columns", op, cols);
    ZG_REQUIRE(mul_sat(rows, cols) < ((size_t)1 << 60) && mul_sat(rows, k) < ((size_t)1 << 60), "%s: %zu rows", op, rows);
    ZG_REQUIRE(k >= 1 && k <= kMaxK, "%s: k = %zu is not in 1 .. %d", op, k, kMaxK);
    // its square and its inverse are normal numbers
    ZG_REQUIRE(temperature >= 1e-18f && temperature <= 1e18f, "%s: temperature %g is not in 1e-18 .. 1e18", op, temperature);
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
#define ZG_TOPK_(NT, VPT, U, BEYOND, SORT, SEG, PER_CU)                                                                                \
    hipLaunchKernelGGL((topk_kernel<NT, VPT, U, BEYOND, SORT, SEG, PER_CU>), dim3(grid(256 / (NT), PER_CU)), dim3(256), 0, ctx->stream, \
                       x, values, indices, rows, c32, k32)
#define ZG_TOPK_WAVE(VPT, SEG, PER_CU)                                \
    do {                                                              \
        if (k > 16) ZG_TOPK_(64, VPT, 4, false, true, SEG, PER_CU);   \
        else ZG_TOPK_(64, VPT, 4, false, false, SEG, PER_CU);         \
    } while (0)
#define ZG_TOPK(NT, VPT, U, BEYOND) ZG_TOPK_(NT, VPT, U, BEYOND, true, kSegment, (U > 4 ? 3 : 4))
    // as many workgroups as the compute units hold, with the same number of rows each
    auto grid = [&](size_t per_block, size_t per_cu) {
        const size_t blocks = ceil_div_sz(rows, per_block), most = ctx->n_cu * per_cu;
        return (unsigned)ceil_div_sz(blocks, ceil_div_sz(blocks, most));
    };
    // A few long rows are cut into segments, which takes two launches (64 of 128000: 1 row 16 us against 39 us with a workgroup per
    // row, 64 rows 26 against 43).  Up to 32000 columns both take the same time, and from k = 256 on the second launch has too much
    // to sort (256 of 128000 in 64 rows: 66 against 53 us).
    if (rows <= 64 && k <= 128 && cols >= 8 * (size_t)kTopkSegment) {
        uint32_t n_seg = (uint32_t)ceil_div_sz(cols, kTopkSegment);
        const uint32_t len = (uint32_t)((ceil_div_sz(cols, n_seg) + 3) & ~(size_t)3);  // at most kTopkSegment, as n_seg segments reach
        n_seg = (uint32_t)ceil_div_sz(cols, len);
        if (cols - (size_t)(n_seg - 1) * len >= k && rows * n_seg <= most_groups(256)) {
            uint64_t* keys = (uint64_t*)workspace(ctx, rows * n_seg * k * sizeof(uint64_t));
            if (!keys) return ZG_HIP_EOOM;
            hipLaunchKernelGGL(topk_segments_kernel, dim3((unsigned)(rows * n_seg)), dim3(256), 0, ctx->stream, x, keys, c32, k32, len, n_seg);
            ZG_LAUNCH_CHECK();
            hipLaunchKernelGGL(topk_join_kernel, dim3((unsigned)rows), dim3(256), 0, ctx->stream, x, keys, values, indices, c32, k32, n_seg);
            ZG_LAUNCH_CHECK();
            return ZG_HIP_OK;
        }
    }
    // A wave per row as far as its 256 groups can bound k and there are rows enough to fill the compute units (or the row is
    // short): its waves never wait for each other (64 of 8192 in 8192 rows: 64 us against 97 us with a workgroup per row).  A
    // workgroup per row else.
#define ZG_TOPK_SHORT(L, KPL)                                                                                                       \
    in_launches(rows, most_groups(256) * (256 / (L)), [&](size_t first, size_t n) {                                                 \
        hipLaunchKernelGGL((topk_short_kernel<L, KPL>), dim3((unsigned)ceil_div_sz(n, 256 / (L))), dim3(256), 0, ctx->stream,       \
                           x + first * cols, values + first * k, indices + first * k, n, c32, k32);                                 \
    })
    // (8 of 128 in 65536 rows 15 us against 29 by a wave per row, 4 of 200 25 against 26, 8 of 256 34 against 29, 16 of 256 48 against 30)
    if (cols <= 256 && k <= (cols <= 128 ? 16u : 4u)) {
        if (cols <= 16) ZG_TOPK_SHORT(4, 4);
        else if (cols <= 64) ZG_TOPK_SHORT(16, 4);
        else if (cols <= 128) ZG_TOPK_SHORT(16, 8);
        else ZG_TOPK_SHORT(16, 16);
    } else if (k <= 128 && (cols <= 2048 || rows >= (size_t)ctx->n_cu * 8)) {
        if (cols <= 256) ZG_TOPK_WAVE(1, 256, 8);
        else if (cols <= 512) ZG_TOPK_WAVE(2, 512, 7);
        else if (cols <= 1024) ZG_TOPK_WAVE(4, 512, 6);
        else if (cols <= 2048) ZG_TOPK_WAVE(8, 512, 4);
        else if (cols <= 8192) ZG_TOPK(64, 8, 4, true);
        else ZG_TOPK(64, 4, 6, true);  // fewer waves with more on its way each (64 of 32000 in 8192 rows: 182 us against 202)
    } else if (cols <= 2048) {
        ZG_TOPK(256, 2, 4, false);
    } else if (cols <= 4096) {
        ZG_TOPK(256, 4, 4, false);
    } else if (cols <= 8192) {
        ZG_TOPK(256, 8, 4, false);
    } else {
        ZG_TOPK(256, 8, 4, true);
    }
#undef ZG_TOPK_SHORT
#undef ZG_TOPK
#undef ZG_TOPK_WAVE
#undef ZG_TOPK_
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
    const uint32_t c32 = (uint32_t)cols, k32 = (uint32_t)k;
    int bits = 1;  // of a column
    while (((size_t)1 << bits) < cols) bits++;
    if (accumulate) {
        const size_t per_wave = k < kWave ? kWave / k : 1;
        hipLaunchKernelGGL(topk_bwd_add_kernel, dim3(row_grid(ceil_div_sz(rows, 4 * per_wave))), dim3(256), 0, ctx->stream, indices, y_g,
                           x_g, rows, c32, k32, bits);
    } else if (cols <= 256 && k <= 16) {
        in_launches(rows, most_groups(256) * 16, [&](size_t first, size_t n) {
            auto launch = [&](auto* kernel) {
                hipLaunchKernelGGL(kernel, dim3((unsigned)ceil_div_sz(n, 16)), dim3(256), 0, ctx->stream, indices + first * k, y_g + first * k,
                                   x_g + first * cols, n, c32, k32);
            };
            if (cols <= 64) launch(topk_bwd_short_kernel<1>);
            else if (cols <= 128) launch(topk_bwd_short_kernel<2>);
            else launch(topk_bwd_short_kernel<4>);
        });
    } else {
        // even spans of whole 128-byte lines
        const size_t span = cols <= 1024 ? cols : (ceil_div_sz(cols, ceil_div_sz(cols, 4096)) + 31) / 32 * 32;
        const size_t spans = ceil_div_sz(cols, span), most = most_groups(256);
        in_launches(rows, cols <= 1024 ? most * 4 : most / spans, [&](size_t first, size_t n) {
            const uint64_t* idx = indices + first * k;
            const float* g = y_g + first * k;
            float* out = x_g + first * cols;
            if (cols <= 1024)
                hipLaunchKernelGGL(topk_bwd_kernel<64>, dim3((unsigned)ceil_div_sz(n, 4)), dim3(256), 0, ctx->stream, idx, g, out, n, c32, k32,
                                   (uint32_t)spans, (uint32_t)span, bits);
            else
                hipLaunchKernelGGL(topk_bwd_kernel<256>, dim3((unsigned)(n * spans)), dim3(256), 0, ctx->stream, idx, g, out, n, c32, k32,
                                   (uint32_t)spans, (uint32_t)span, bits < 12 ? bits : 12);
        });
    }
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
    const float inv_temp = 1.f / temperature;
    DistillArgs a{logits, teacher, indices, row_weights, stats, row_loss, grad, rows, (uint32_t)cols, (uint32_t)k, temperature, inv_temp,
                  inv_temp * 1.44269504088896340736f, 1.f / (float)rows, 1, (uint32_t)cols,
                  rows * cols * (accumulate ? 2 : 1) > kCachedFloats};
    bool summed = false;
    int rc;
    if (fwd && !bwd) rc = distill_launch<true, false, false>(ctx, a, loss, &summed);
    else if (!fwd && !accumulate) rc = distill_launch<false, true, false>(ctx, a, loss, &summed);
    else if (!fwd) rc = distill_launch<false, true, true>(ctx, a, loss, &summed);
    else if (!accumulate) rc = distill_launch<true, true, false>(ctx, a, loss, &summed);
    else rc = distill_launch<true, true, true>(ctx, a, loss, &summed);
    if (rc || !fwd || summed) return rc;
    return distill_total(ctx, row_loss, row_weights, loss, rows);
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
