// A cache cut to a budget: which cells keep their place, and the rows brought to the front.
//
// The `keep` cells that stay are the guarded ones first, then those of the largest mass, the lower index on a tie.  A cell that stays and lies in front keeps its place; the others that stay go, in their order, to the places that became free
// there: source[i] = the cell whose rows stand at i afterwards, and no more rows move than have to.
#include "ops_common.h"
#include "kernel_timing.h"

#include <algorithm>

#define CC_THREADS 1024
#define CC_BINS 2048
#define CC_WINDOW 32768      /* cells that move, a window of LDS at a time */

// order of the cells: guarded, then by mass (-0 like 0), what is no number last
static __device__ __forceinline__ uint32_t cc_key(float x, bool guarded) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    const uint32_t k = b & 0x80000000u ? ~b : b | 0x80000000u;
    return guarded ? 0xffffffffu : x != x ? 0u : k;
}

// inclusive sum over the workgroup's threads before this one in order, and over all (sixteen waves; two barriers)
static __device__ __forceinline__ uint32_t cc_before(uint32_t v, uint32_t * waves, int lane, int wave, uint32_t & all) {
    uint32_t x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) { const uint32_t y = __shfl_up(x, o, 64); if (lane >= o) x += y; }
    __syncthreads();
    if (lane == 63) waves[wave] = x;
    __syncthreads();
    uint32_t base = 0; all = 0;
#pragma unroll
    for (int i = 0; i < CC_THREADS / 64; i++) { const uint32_t w = waves[i]; if (i < wave) base += w; all += w; }
    return base + x - v;
}

// One workgroup; a wave owns a run of cells, 64 of them a step.  The boundary's key by its digits of 11, 11 and 10 bits from the counts of what is left.  VPT > 0: the keys of up to 1024 VPT cells stay in registers
template <int VPT> __global__ void __launch_bounds__(CC_THREADS) k_cache_choose(const float * __restrict__ mass, const uint32_t * __restrict__ guard, int cells, int keep, int32_t * __restrict__ source, const int32_t * __restrict__ abort_w) {
    if (pi_aborted(abort_w)) return;
    __shared__ uint32_t bins[CC_BINS];
    __shared__ int32_t movers[CC_WINDOW];
    __shared__ uint32_t waves[CC_THREADS / 64], found[3];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, steps = (cells + CC_THREADS - 1) / CC_THREADS;
    const int64_t first = (int64_t) wave * steps * 64 + lane;
    uint32_t keys[VPT > 0 ? VPT : 1];
    auto load = [&](int j) __attribute__((always_inline)) -> uint32_t {
        const int64_t c = first + (int64_t) j * 64;
        return c < cells ? cc_key(mass[c], guard && (guard[c >> 5] >> (c & 31) & 1)) : 0u;
    };
    if constexpr (VPT > 0) {
#pragma unroll
        for (int j = 0; j < VPT; j++) keys[j] = j < steps ? load(j) : 0u;
    }
    // f(cell, is one, key) for the wave's cells in their order
    auto each = [&](auto && f) __attribute__((always_inline)) {
        if constexpr (VPT > 0) {
#pragma unroll
            for (int j = 0; j < VPT; j++) if (j < steps) { const int64_t c = first + (int64_t) j * 64; f((int) c, c < cells, keys[j]); }
        } else for (int j = 0; j < steps; j++) { const int64_t c = first + (int64_t) j * 64; f((int) c, c < cells, load(j)); }
    };
    uint32_t prefix = 0, left = (uint32_t) keep;               // `left` of the cells whose key begins like `prefix` stay; those above stay, those below do not
    int shift = 32;
    for (int pass = 0; pass < 3 && left > 0; pass++) {
        const int width = pass == 2 ? 10 : 11, from = shift - width;
        for (int i = tid; i < CC_BINS; i += CC_THREADS) bins[i] = 0;
        __syncthreads();
        each([&](int, bool is, uint32_t key) __attribute__((always_inline)) {
            const bool in = is && (pass == 0 || key >> shift == prefix);
            const uint32_t bin = key >> from & ((1u << width) - 1);
            const unsigned long long who = __ballot(in);
            if (who == 0) return;
            const int lead = __builtin_ctzll(who);
            const uint32_t b0 = (uint32_t) __builtin_amdgcn_readlane((int) bin, lead);
            if (__ballot(in && bin == b0) == who) { if (lane == lead) atomicAdd(&bins[b0], (uint32_t) __popcll(who)); }          // (equal masses: one address)
            else if (in) atomicAdd(&bins[bin], 1u);
        });
        __syncthreads();
        // from the top bin down, two to a thread
        const int top = (1 << width) - 1 - 2 * tid;
        const uint32_t a = top >= 0 ? bins[top] : 0, b = top >= 1 ? bins[top - 1] : 0;
        uint32_t all, before = cc_before(a + b, waves, lane, wave, all);
        if (a + b > 0 && before < left && before + a + b >= left) {
            const bool second = before + a < left;
            found[0] = (uint32_t) (second ? top - 1 : top); found[1] = left - before - (second ? a : 0); found[2] = second ? b : a;
        }
        __syncthreads();
        prefix = prefix << width | found[0]; left = found[1]; shift = from;
        if (found[2] == left) break;                         // all of the bin stay
    }
    __syncthreads();
    // key >> shift > prefix stays; == prefix: the first `left` (all, where the passes ended early)
    uint32_t equal = 0;
    auto above = [&](bool is, uint32_t key) __attribute__((always_inline)) { return is && keep > 0 && (shift < 32 ? key >> shift : 0) > prefix; };
    auto same = [&](bool is, uint32_t key) __attribute__((always_inline)) { return is && keep > 0 && (shift < 32 ? key >> shift : 0) == prefix; };
    each([&](int, bool is, uint32_t key) __attribute__((always_inline)) { equal += (uint32_t) __popcll(__ballot(same(is, key))); });
    uint32_t all;
    const uint32_t equal_before = cc_before(lane == 0 ? equal : 0, waves, lane, wave, all);
    const uint32_t equal0 = (uint32_t) __builtin_amdgcn_readfirstlane((int) equal_before);
    auto stays = [&](bool is, uint32_t key, uint32_t & seen) __attribute__((always_inline)) {
        const unsigned long long who = __ballot(same(is, key));
        const bool mine = same(is, key) && seen + (uint32_t) __popcll(who & ((1ull << lane) - 1)) < left;
        seen += (uint32_t) __popcll(who);
        return mine || above(is, key);
    };
    uint32_t holes = 0, moves = 0, seen = equal0;
    each([&](int c, bool is, uint32_t key) __attribute__((always_inline)) {
        const bool s = stays(is, key, seen);
        holes += (uint32_t) __popcll(__ballot(is && c < keep && !s)); moves += (uint32_t) __popcll(__ballot(is && c >= keep && s));
    });
    uint32_t total;
    const uint32_t hole0 = (uint32_t) __builtin_amdgcn_readfirstlane((int) cc_before(lane == 0 ? holes : 0, waves, lane, wave, total));
    const uint32_t move0 = (uint32_t) __builtin_amdgcn_readfirstlane((int) cc_before(lane == 0 ? moves : 0, waves, lane, wave, total));
    for (uint32_t w = 0; w == 0 || w < total; w += CC_WINDOW) {
        uint32_t at = move0;
        seen = equal0;
        __syncthreads();
        each([&](int c, bool is, uint32_t key) __attribute__((always_inline)) {
            const bool m = stays(is, key, seen) && c >= keep;
            const unsigned long long who = __ballot(m);
            const uint32_t r = at + (uint32_t) __popcll(who & ((1ull << lane) - 1)) - w;
            if (m && r < CC_WINDOW) movers[r] = c;           // (r wraps far above for those of earlier windows)
            at += (uint32_t) __popcll(who);
        });
        __syncthreads();
        at = hole0; seen = equal0;
        each([&](int c, bool is, uint32_t key) __attribute__((always_inline)) {
            const bool s = stays(is, key, seen), h = is && c < keep && !s;
            const unsigned long long who = __ballot(h);
            const uint32_t r = at + (uint32_t) __popcll(who & ((1ull << lane) - 1)) - w;
            if (h && r < CC_WINDOW) source[c] = movers[r];
            if (w == 0 && is && c < keep && s) source[c] = c;
            at += (uint32_t) __popcll(who);
        });
    }
}

extern "C" int pi_op_cache_choose(const float * mass, const uint32_t * guard, int cells, int keep, int32_t * source, void * stream) {
    if (cells < 0 || keep < 0 || keep > cells || cells > 0x7ffff000) { pi_set_error("pi_op_cache_choose: %d of %d cells", keep, cells); return -1; }
    if (keep == 0) return 0;
    if (!mass || !source) { pi_set_error("pi_op_cache_choose: mass or source is NULL"); return -1; }
#define CC_GO(V) PI_KT_LAUNCH(PI_KT_OTHER, 0, 1, 4.0 * cells + 4.0 * keep, (k_cache_choose<V>), dim3(1), dim3(CC_THREADS), 0, (hipStream_t) stream, mass, guard, cells, keep, source, pi_abort_word())
    if (cells <= CC_THREADS * 4) CC_GO(4); else if (cells <= CC_THREADS * 16) CC_GO(16); else if (cells <= CC_THREADS * 32) CC_GO(32); else CC_GO(0);
#undef CC_GO
    PI_CHECK_LAUNCH();
    return 0;
}

// ---- the rows -----------------------------------------------------------------------------------------------------------------------------------------------------------------------
#define CM_ARRAYS 120        /* of one launch: their addresses are the kernel's arguments */
struct cm_arrays { uint8_t * at[CM_ARRAYS]; uint64_t bytes[CM_ARRAYS]; };

// row i <- row source[i] of one array's 64 rows a wave: the moves are listed in LDS, and as many lanes as a row has units take one.  Rows come from behind `keep` and go in front of it: nothing is read that another thread writes
template <class T> static __device__ __forceinline__ void cm_rows(uint8_t * base, uint64_t bytes, const int2 * list, int n, int lane) {
    const uint32_t units = (uint32_t) (bytes / sizeof(T));
    int per = 64;
    while (per > 1 && (uint32_t) per / 2 >= units) per >>= 1;
    const int sub = lane & (per - 1), rows = 64 / per;
    for (int i = lane / per; i < n; i += 4 * rows) {
        T * to[4]; const T * from[4];
#pragma unroll
        for (int k = 0; k < 4; k++) { const int2 m = list[min(i + k * rows, n - 1)]; to[k] = (T *) (base + (uint64_t) m.x * bytes); from[k] = (const T *) (base + (uint64_t) m.y * bytes); }
        for (uint32_t u = sub; u < units; u += per) {
            T x[4];
#pragma unroll
            for (int k = 0; k < 4; k++) x[k] = from[k][u];
#pragma unroll
            for (int k = 0; k < 4; k++) if (i + k * rows < n) to[k][u] = x[k];
        }
    }
}

__global__ void __launch_bounds__(256) k_cache_move(const cm_arrays A, const int32_t * __restrict__ source, int keep, int cells, const int32_t * __restrict__ abort_w) {
    if (pi_aborted(abort_w)) return;
    __shared__ int2 lists[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = (blockIdx.x * 4 + wave) * 64 + lane;
    const int from = row < keep ? source[row] : -1;
    const bool moves = from >= keep && from < cells;
    const unsigned long long who = __ballot(moves);
    if (moves) lists[wave][__popcll(who & ((1ull << lane) - 1))] = make_int2(row, from);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    uint8_t * base = A.at[blockIdx.y];
    const uint64_t bytes = A.bytes[blockIdx.y];
    const int n = __popcll(who);
    if ((((uintptr_t) base | bytes) & 15) == 0) cm_rows<uint4>(base, bytes, lists[wave], n, lane);
    else if ((((uintptr_t) base | bytes) & 3) == 0) cm_rows<uint32_t>(base, bytes, lists[wave], n, lane);
    else cm_rows<uint8_t>(base, bytes, lists[wave], n, lane);
}

extern "C" int pi_op_cache_move(void * const * arrays, const int64_t * row_bytes, int n_arrays, const int32_t * source, int keep, int cells, void * stream) {
    if (n_arrays < 0 || keep < 0 || keep > cells) { pi_set_error("pi_op_cache_move: %d arrays, %d of %d cells", n_arrays, keep, cells); return -1; }
    if (n_arrays == 0 || keep == 0 || keep == cells) return 0;
    if (!arrays || !row_bytes || !source) { pi_set_error("pi_op_cache_move: arrays, their rows' bytes or source is NULL"); return -1; }
    for (int i = 0; i < n_arrays; i++) if (!arrays[i] || row_bytes[i] < 1 || row_bytes[i] > 0x7fffffff) { pi_set_error("pi_op_cache_move: array %d is NULL or has rows of %lld bytes", i, (long long) row_bytes[i]); return -1; }
    for (int i0 = 0; i0 < n_arrays; i0 += CM_ARRAYS) {
        cm_arrays A{};
        const int n = std::min(CM_ARRAYS, n_arrays - i0);
        double bytes = 0;
        for (int i = 0; i < n; i++) { A.at[i] = (uint8_t *) arrays[i0 + i]; A.bytes[i] = (uint64_t) row_bytes[i0 + i]; bytes += 2.0 * std::min(keep, cells - keep) * row_bytes[i0 + i]; }
        PI_KT_LAUNCH(PI_KT_OTHER, 0, 1, bytes, k_cache_move, dim3((unsigned) ((keep + 255) / 256), (unsigned) n), dim3(256), 0, (hipStream_t) stream, A, source, keep, cells, pi_abort_word());
        PI_CHECK_LAUNCH();
    }
    return 0;
}
