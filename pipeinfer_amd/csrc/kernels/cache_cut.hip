// A cache cut to a budget: which cells keep their place, and the rows brought to the front.
//
// The `keep` cells that stay are the guarded ones first, then those of the largest mass, the lower index on a tie.  A cell that stays and lies in front keeps its place; the others that stay go, in their order, to the places that became free
// there: source[i] = the cell whose rows stand at i afterwards, and no more rows move than have to.
#include "ops_common.h"
#include "kernel_timing.h"
#include "wave_scan.h"

#include <algorithm>

#define CC_THREADS 1024
#define CC_BINS 2048
#define CC_KEYS 28672        /* keys in LDS (112 KB); cells that move, as many at a time */
#define CC_CELLS 131072      /* cells of the bitmap */

// order of the cells: guarded, then by mass (-0 like 0), what is no number last; 0 is no cell's
static __device__ __forceinline__ uint32_t cc_key(float x, bool guarded) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    const uint32_t k = b & 0x80000000u ? ~b : b | 0x80000000u;
    return guarded ? 0xffffffffu : x != x ? 1u : k;
}

// the sum over the workgroup's threads ahead of this one, and over all of them (sixteen waves; two barriers)
static __device__ __forceinline__ uint32_t cc_before(uint32_t v, uint32_t * waves, int lane, int wave, uint32_t & all) {
    const uint32_t x = pi_wave_scan(v);
    __syncthreads();
    if (lane == 63) waves[wave] = x;
    __syncthreads();
    uint32_t base = 0; all = 0;
#pragma unroll
    for (int i = 0; i < CC_THREADS / 64; i++) { const uint32_t w = waves[i]; if (i < wave) base += w; all += w; }
    return base + x - v;
}

// One workgroup.  The boundary's key: its first 11 bits from the counts of all keys, the rest by digits of 11 and 10 bits of those that share them, listed in LDS (of all keys where the list does not hold them).  What stays is then a bit of
// a bitmap in LDS, and where a cell goes follows from the bits ahead of it: no pass walks the cells in their order.  Bound by the instructions of one compute unit, a handful per pass and 64 cells: keys of CC_KEYS cells stay in LDS, of
// 4096 more in registers, the others' are made again from the masses.  (32768 cells: 25 us, 19 of them the keys, their counts and the passes over them; with loops over cells, tests in every lane, 31.)
struct cc_shared {
    __attribute__((aligned(16))) uint32_t bins[CC_BINS], words[2 * CC_CELLS / 32], waves[CC_THREADS / 64], found[4];
    __attribute__((aligned(16))) uint32_t keys[CC_KEYS];       // then the cells that move
};
__global__ void __launch_bounds__(CC_THREADS) k_cache_choose(const float * __restrict__ mass, const uint32_t * __restrict__ guard, int cells, int keep, int32_t * __restrict__ source, const int32_t * __restrict__ abort_w) {
    const int gone = pi_abort_peek(abort_w);
    __shared__ cc_shared L;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    for (int i = tid; i < CC_BINS; i += CC_THREADS) L.bins[i] = 0;
    if (tid == 0) L.found[3] = 0;
    if (pi_aborted_together(gone, abort_w)) return;
    auto count = [&](bool in, uint32_t bin) __attribute__((always_inline)) {
        const uint32_t b0 = (uint32_t) __builtin_amdgcn_readfirstlane((int) bin);
        if (__all(in && bin == b0)) { if (lane == 0) atomicAdd(&L.bins[b0], 64u); }              // (equal masses: one address)
        else if (in) atomicAdd(&L.bins[bin], 1u);
    };
    // the keys, eight cells a thread on their way at a time; in LDS zeros behind the last of them, to the end of a round of four steps
    const int steps = (cells + CC_THREADS - 1) / CC_THREADS;
    constexpr int HELD = CC_KEYS / CC_THREADS;
    uint32_t behind[4] = {};                                   // the four steps behind those in LDS
    for (int i0 = 0; i0 < steps; i0 += 8) {
        float m[8]; uint32_t g[8] = {};
#pragma unroll
        for (int j = 0; j < 8; j++) m[j] = mass[min((i0 + j) * CC_THREADS + tid, cells - 1)];
        if (guard)
#pragma unroll
            for (int j = 0; j < 8; j++) g[j] = guard[min((i0 + j) * CC_THREADS + tid, cells - 1) >> 5];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int c = (i0 + j) * CC_THREADS + tid;
            if (i0 + j >= (steps + 3 & ~3)) break;
            const uint32_t key = c < cells ? cc_key(m[j], g[j] >> (tid & 31) & 1) : 0u;
            if (i0 + j < HELD) L.keys[c] = key;
            if (j >= HELD % 8 && j < HELD % 8 + 4 && i0 == HELD / 8 * 8) behind[j & 3] = key;
            if (i0 + j < steps) count(key != 0, key >> 21);
        }
    }
    // f(step, key) for every CC_THREADS-th cell, four keys on their way; 0 where there is no cell
    auto each = [&](auto && f) __attribute__((always_inline)) {
        static_assert(HELD % 4 == 0 && CC_CELLS % (32 * CC_THREADS) == 0, "");
        int i = 0;
#pragma unroll 1
        for (; i < min(steps, HELD); i += 4) {
            uint32_t key[4];
#pragma unroll
            for (int j = 0; j < 4; j++) key[j] = L.keys[(i + j) * CC_THREADS + tid];
#pragma unroll
            for (int j = 0; j < 4; j++) f(i + j, key[j]);
        }
        if (i < steps) {
#pragma unroll
            for (int j = 0; j < 4; j++) f(i + j, behind[j]);
            i += 4;
        }
#pragma unroll 1
        for (; i < steps; i += 4) {                          // (from memory, where one at a time is a microsecond a step)
            float m[4]; uint32_t g[4] = {};
#pragma unroll
            for (int j = 0; j < 4; j++) m[j] = mass[min((i + j) * CC_THREADS + tid, cells - 1)];
            if (guard)
#pragma unroll
                for (int j = 0; j < 4; j++) g[j] = guard[min((i + j) * CC_THREADS + tid, cells - 1) >> 5];
#pragma unroll
            for (int j = 0; j < 4; j++) f(i + j, (i + j) * CC_THREADS + tid < cells ? cc_key(m[j], g[j] >> (tid & 31) & 1) : 0u);
        }
    };
    uint32_t prefix = 0, left = (uint32_t) keep, same = 0;     // of the `same` cells whose key begins like `prefix` `left` stay, the lowest; all above stay, none below
    // from the top bin down, two to a thread
    auto border = [&](int width) __attribute__((always_inline)) {
        __syncthreads();
        const int top = (1 << width) - 1 - 2 * tid;
        const uint32_t a = top >= 0 ? L.bins[top] : 0, b = top >= 1 ? L.bins[top - 1] : 0;
        uint32_t all;
        const uint32_t before = cc_before(a + b, L.waves, lane, wave, all);
        if (before < left && before + a + b >= left) {
            const bool second = before + a < left;
            L.found[0] = (uint32_t) (second ? top - 1 : top); L.found[1] = left - before - (second ? a : 0); L.found[2] = second ? b : a;
        }
        __syncthreads();
        prefix = prefix << width | L.found[0]; left = L.found[1]; same = L.found[2];
    };
    border(11);
    int shift = 21;
    const bool listed = same <= 2 * (CC_CELLS / 32);             // (bitmap and sums are not in use yet)
    uint32_t * const list = L.words, * const bitmap = L.words, * const ahead = L.words + CC_CELLS / 32;
    const uint32_t in_list = same;
    if (same != left && listed) {
        uint32_t mine = 0;                                   // (counted first: no store waits for an atomic)
        const uint32_t least = max(prefix << 21, 1u), span = ((prefix + 1) << 21) - least;
        each([&](int, uint32_t key) __attribute__((always_inline)) { mine += key - least < span; });
        if (__any(mine > 0)) {
            uint32_t at = mine > 0 ? atomicAdd(&L.found[3], mine) : 0;
            each([&](int, uint32_t key) __attribute__((always_inline)) { if (key - least < span) list[at++] = key; });
        }
        __syncthreads();
    }
    for (int pass = 0; pass < 2 && same != left; pass++) {
        const int width = 11 - pass, from = shift - width;
        for (int i = tid; i < CC_BINS; i += CC_THREADS) L.bins[i] = 0;
        __syncthreads();
        auto digit = [&](int, uint32_t key) __attribute__((always_inline)) { count(key != 0 && key >> shift == prefix, key >> from & ((1u << width) - 1)); };
        if (listed) for (uint32_t i = tid; i - lane < in_list; i += CC_THREADS) digit(0, i < in_list ? list[i] : 0u);
        else each(digit);
        border(width);
        shift = from;
    }
    __syncthreads();
    // the bitmap of what stays; where not all of the boundary's key do, the first of them
    const uint32_t bound = max(prefix << shift, 1u);
    const bool some = same != left;                            // (then `bound` is the boundary's whole key)
    const int words = (cells + 31) / 32;
    uint32_t stay = 0, equal = 0;                              // lane l: half l & 1 of step l / 2, of 32 steps
    auto leave = [&](int step) __attribute__((always_inline)) {
        const int at = ((step & ~31) + lane / 2) * (CC_THREADS / 32) + 2 * wave + (lane & 1);
        bitmap[at] = stay;
        if (some) ahead[at] = equal;
        stay = equal = 0;
    };
    each([&](int i, uint32_t key) __attribute__((always_inline)) {
        const bool mine = lane >> 1 == (i & 31);
        const unsigned long long who = __ballot(key >= bound);
        stay = mine ? lane & 1 ? (uint32_t) (who >> 32) : (uint32_t) who : stay;
        if (some) {
            const unsigned long long eq = __ballot(key == bound);
            equal = mine ? lane & 1 ? (uint32_t) (eq >> 32) : (uint32_t) eq : equal;
        }
        if ((i & 31) == 31) leave(i);
    });
    if ((steps + 3 & ~3) & 31) leave(steps - 1);
    __syncthreads();
    uint32_t all;
    if (some) {
        // of the words' equal ones (in `ahead`) those past the first `left` go
        for (uint32_t w0 = 0, seen = 0; w0 < (uint32_t) words; w0 += CC_THREADS) {
            const uint32_t w = w0 + tid;
            uint32_t eq = w < (uint32_t) words ? ahead[w] : 0, n = seen + cc_before((uint32_t) __popc(eq), L.waves, lane, wave, all);
            uint32_t go = 0;
            for (; eq; eq &= eq - 1, n++) if (n >= left) go |= eq & -eq;
            if (go) bitmap[w] &= ~go;
            seen += all;
        }
        __syncthreads();
    }
    // ahead of a word in front of the budget: the places that become free; behind it: the cells that stay (both in the word where it ends)
    const uint32_t edge = (uint32_t) keep / 32, in_front = (1u << (keep & 31)) - 1;          // of the edge's word
    uint32_t total = 0, edge_free = 0;
    for (int part = 0; part < 2; part++) {
        uint32_t seen = 0;
        for (uint32_t w0 = part == 0 ? 0 : edge / CC_THREADS * CC_THREADS; w0 < (part == 0 ? edge + 1 : (uint32_t) words); w0 += CC_THREADS) {
            const uint32_t w = w0 + tid, b = w < (uint32_t) words ? bitmap[w] : 0;
            const uint32_t mine = part == 0 ? (w < edge ? ~b : w == edge ? ~b & in_front : 0) : (w > edge ? b : w == edge ? b & ~in_front : 0);
            const uint32_t n = seen + cc_before((uint32_t) __popc(mine), L.waves, lane, wave, all);
            if (w < (uint32_t) words && (part == 0 ? w < edge : w > edge)) ahead[w] = n;
            if (part == 0 && w == edge) L.found[0] = n;          // (there the cells that stay begin with none ahead)
            seen += all;
        }
        total = seen;
        __syncthreads();
        if (part == 0) edge_free = L.found[0];
    }
    for (uint32_t w0 = 0; w0 == 0 || w0 < total; w0 += CC_KEYS) {
#pragma unroll 1
        for (int i = keep / (4 * CC_THREADS) * 4; i < steps; i += 4) {
            uint32_t b[4], r[4];
#pragma unroll
            for (int j = 0; j < 4; j++) { const int w = (i + j) * (CC_THREADS / 32) + tid / 32; b[j] = bitmap[w]; r[j] = ahead[w]; }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int c = (i + j) * CC_THREADS + tid;
                if ((uint32_t) c / 32 == edge) { b[j] &= ~in_front; r[j] = 0; }
                r[j] += (uint32_t) __popc(b[j] & ((1u << (tid & 31)) - 1)) - w0;               // (wraps far above for those of earlier windows)
                if (c >= keep && (b[j] >> (tid & 31) & 1) && r[j] < CC_KEYS) L.keys[r[j]] = (uint32_t) c;
            }
        }
        __syncthreads();
#pragma unroll 1
        for (int i = 0; i * CC_THREADS < keep; i += 4) {
            uint32_t b[4], r[4], k[4];
#pragma unroll
            for (int j = 0; j < 4; j++) { const int w = (i + j) * (CC_THREADS / 32) + tid / 32; b[j] = bitmap[w]; r[j] = (uint32_t) w == edge ? edge_free : ahead[w]; }
#pragma unroll
            for (int j = 0; j < 4; j++) { r[j] += (uint32_t) __popc(~b[j] & ((1u << (tid & 31)) - 1)) - w0; k[j] = L.keys[min(r[j], (uint32_t) CC_KEYS - 1)]; }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int c = (i + j) * CC_THREADS + tid;
                const bool stays = b[j] >> (tid & 31) & 1;
                if (c < keep && (stays ? w0 == 0 : r[j] < CC_KEYS)) source[c] = stays ? c : (int32_t) k[j];
            }
        }
        __syncthreads();
    }
}

// Caches of more cells than the bitmap holds: the same border, then the cells in their order, a wave's run of them 64 a step
static __device__ __forceinline__ uint32_t cc_rank(unsigned long long who) { return __builtin_amdgcn_mbcnt_hi((uint32_t) (who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t) who, 0u)); }

__global__ void __launch_bounds__(CC_THREADS) k_cache_choose_long(const float * __restrict__ mass, const uint32_t * __restrict__ guard, int cells, int keep, int32_t * __restrict__ source, const int32_t * __restrict__ abort_w) {
    const int gone = pi_abort_peek(abort_w);
    __shared__ uint32_t bins[CC_BINS], waves[CC_THREADS / 64], found[3], list[CC_KEYS];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), steps = (cells + CC_THREADS - 1) / CC_THREADS;
    const int64_t first = (int64_t) wave * steps * 64;
    if (pi_aborted_together(gone, abort_w)) return;
    // f(first cell of the step, is this lane's one, key) for the wave's cells in their order
    auto each = [&](auto && f) __attribute__((always_inline)) {
        for (int j = 0; j < steps; j++) {
            const int64_t c = first + (int64_t) j * 64, mine = c + lane;
            if (c >= cells) break;
            f((int) c, mine < cells, mine < cells ? cc_key(mass[mine], guard && (guard[mine >> 5] >> (mine & 31) & 1)) : 0u);
        }
    };
    uint32_t prefix = 0, left = (uint32_t) keep, same = 0, all;
    int shift = 32;
    for (int pass = 0; pass < 3 && same != left; pass++) {
        const int width = pass == 2 ? 10 : 11, from = shift - width;
        for (int i = tid; i < CC_BINS; i += CC_THREADS) bins[i] = 0;
        __syncthreads();
        each([&](int, bool is, uint32_t key) __attribute__((always_inline)) {
            const bool in = is && (pass == 0 || key >> shift == prefix);
            const uint32_t bin = key >> from & ((1u << width) - 1), b0 = (uint32_t) __builtin_amdgcn_readfirstlane((int) bin);
            if (__all(in && bin == b0)) { if (lane == 0) atomicAdd(&bins[b0], 64u); }
            else if (in) atomicAdd(&bins[bin], 1u);
        });
        __syncthreads();
        const int top = (1 << width) - 1 - 2 * tid;
        const uint32_t a = top >= 0 ? bins[top] : 0, b = top >= 1 ? bins[top - 1] : 0, before = cc_before(a + b, waves, lane, wave, all);
        if (a + b > 0 && before < left && before + a + b >= left) {
            const bool second = before + a < left;
            found[0] = (uint32_t) (second ? top - 1 : top); found[1] = left - before - (second ? a : 0); found[2] = second ? b : a;
        }
        __syncthreads();
        prefix = prefix << width | found[0]; left = found[1]; same = found[2]; shift = from;
    }
    const uint32_t bound = prefix << shift;
    uint32_t equal = 0;
    each([&](int, bool is, uint32_t key) __attribute__((always_inline)) { equal += (uint32_t) __popcll(__ballot(is && key >> shift == prefix)); });
    const uint32_t equal0 = (uint32_t) __builtin_amdgcn_readfirstlane((int) cc_before(lane == 0 ? equal : 0, waves, lane, wave, all));
    auto stays = [&](bool is, uint32_t key, uint32_t & seen) __attribute__((always_inline)) {
        const bool eq = is && key >> shift == prefix;
        const unsigned long long who = __ballot(eq);
        const bool mine = eq ? seen + cc_rank(who) < left : is && key >= bound;
        seen += (uint32_t) __popcll(who);
        return mine;
    };
    uint32_t holes = 0, moves = 0, seen = equal0, total;
    each([&](int c, bool is, uint32_t key) __attribute__((always_inline)) {
        const bool s = stays(is, key, seen);
        holes += (uint32_t) __popcll(__ballot(c + lane < keep && !s)); moves += (uint32_t) __popcll(__ballot(c + lane >= keep && s));
    });
    const uint32_t hole0 = (uint32_t) __builtin_amdgcn_readfirstlane((int) cc_before(lane == 0 ? holes : 0, waves, lane, wave, total));
    const uint32_t move0 = (uint32_t) __builtin_amdgcn_readfirstlane((int) cc_before(lane == 0 ? moves : 0, waves, lane, wave, total));
    for (uint32_t w = 0; w == 0 || w < total; w += CC_KEYS) {
        uint32_t at = move0;
        seen = equal0;
        __syncthreads();
        each([&](int c, bool is, uint32_t key) __attribute__((always_inline)) {
            const bool m = stays(is, key, seen) && c + lane >= keep;
            const unsigned long long who = __ballot(m);
            const uint32_t r = at + cc_rank(who) - w;
            if (m && r < CC_KEYS) list[r] = (uint32_t) (c + lane);
            at += (uint32_t) __popcll(who);
        });
        __syncthreads();
        at = hole0; seen = equal0;
        each([&](int c, bool is, uint32_t key) __attribute__((always_inline)) {
            const bool s = stays(is, key, seen), in = c + lane < keep, h = in && !s;
            const unsigned long long who = __ballot(h);
            const uint32_t r = at + cc_rank(who) - w;
            if (h && r < CC_KEYS) source[c + lane] = (int32_t) list[r];
            if (w == 0 && in && s) source[c + lane] = c + lane;
            at += (uint32_t) __popcll(who);
        });
    }
}

extern "C" int pi_op_cache_choose(const float * mass, const uint32_t * guard, int cells, int keep, int32_t * source, void * stream) {
    if (cells < 0 || keep < 0 || keep > cells || cells > 0x7ffff000) { pi_set_error("pi_op_cache_choose: %d of %d cells", keep, cells); return -1; }
    if (keep == 0) return 0;
    if (!mass || !source) { pi_set_error("pi_op_cache_choose: mass or source is NULL"); return -1; }
    if (cells <= CC_CELLS) PI_KT_LAUNCH(PI_KT_OTHER, 0, 1, 4.0 * cells + 4.0 * keep, k_cache_choose, dim3(1), dim3(CC_THREADS), 0, (hipStream_t) stream, mass, guard, cells, keep, source, pi_abort_word());
    else PI_KT_LAUNCH(PI_KT_OTHER, 0, 1, 4.0 * cells + 4.0 * keep, k_cache_choose_long, dim3(1), dim3(CC_THREADS), 0, (hipStream_t) stream, mass, guard, cells, keep, source, pi_abort_word());
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

// An array's address stands in the kernel's arguments, in host memory: that read is most of a short move, 3 us for one workgroup's, and the reads of all of them queue (45 arrays of 1000 rows, 331 moving: 1440 workgroups of 256 threads 18 us,
// 45 of 1024 9).  So a workgroup takes 1024 rows of one array, or fewer, down to 64, while they
// hold more than a megabyte and there are fewer than two workgroups a compute unit (80 arrays of 1000 rows of 8 KB, half of them moving: 164 us, of 1024 rows 248; 4 of 2500 such rows 25 and 95).  Long moves are bound by memory (32 arrays, half of 32768 rows of 2 KB kept: 229 us, 1.07 GB at 4.7 TB/s)
__global__ void __launch_bounds__(1024) k_cache_move(const cm_arrays A, const int32_t * __restrict__ source, int blocks, int of_wave, int keep, int cells, const int32_t * __restrict__ abort_w) {
    if (pi_aborted(abort_w)) return;
    __shared__ int2 lists[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, array = (int) blockIdx.x / blocks, block = (int) blockIdx.x % blocks;
    uint8_t * base = A.at[array];
    const uint64_t bytes = A.bytes[array];
    const int64_t row64 = ((int64_t) block * 16 + wave) * of_wave + lane;
    const int row = (int) min(row64, (int64_t) keep), from = lane < of_wave && row < keep ? source[row] : -1;
    const bool moves = from >= keep && from < cells;
    const unsigned long long who = __ballot(moves);
    if (moves) lists[wave][__popcll(who & ((1ull << lane) - 1))] = make_int2(row, from);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const int n = __popcll(who);
    if ((((uintptr_t) base | bytes) & 15) == 0) cm_rows<uint4>(base, bytes, lists[wave], n, lane);
    else if ((((uintptr_t) base | bytes) & 3) == 0) cm_rows<uint32_t>(base, bytes, lists[wave], n, lane);
    else cm_rows<uint8_t>(base, bytes, lists[wave], n, lane);
}

extern "C" int pi_op_cache_move(void * const * arrays, const int64_t * row_bytes, int n_arrays, const int32_t * source, int keep, int cells, void * stream) {
    if (n_arrays < 0 || keep < 0 || keep > cells || cells > 0x7ffff000) { pi_set_error("pi_op_cache_move: %d arrays, %d of %d cells", n_arrays, keep, cells); return -1; }
    if (n_arrays == 0 || keep == 0 || keep == cells) return 0;
    if (!arrays || !row_bytes || !source) { pi_set_error("pi_op_cache_move: arrays, their rows' bytes or source is NULL"); return -1; }
    for (int i = 0; i < n_arrays; i++) if (!arrays[i] || row_bytes[i] < 1 || row_bytes[i] > 0x7fffffff) { pi_set_error("pi_op_cache_move: array %d is NULL or has rows of %lld bytes", i, (long long) row_bytes[i]); return -1; }
    for (int i0 = 0; i0 < n_arrays; i0 += CM_ARRAYS) {
        cm_arrays A{};
        const int n = std::min(CM_ARRAYS, n_arrays - i0);
        double bytes = 0;
        int64_t largest = 0;
        for (int i = 0; i < n; i++) { A.at[i] = (uint8_t *) arrays[i0 + i]; A.bytes[i] = (uint64_t) row_bytes[i0 + i]; largest = std::max(largest, row_bytes[i0 + i]); bytes += 2.0 * std::min(keep, cells - keep) * row_bytes[i0 + i]; }
        int of_wave = 64;                                    // rows
        while (of_wave > 4 && (int64_t) n * ((keep + 16 * of_wave - 1) / (16 * of_wave)) < 2 * pi_cu_count() && largest * 16 * of_wave > 1 << 20) of_wave /= 2;
        const int blocks = (keep + 16 * of_wave - 1) / (16 * of_wave);
        if ((int64_t) n * blocks > 0x7fffffff) { pi_set_error("pi_op_cache_move: %d rows of %d arrays", keep, n); return -1; }
        PI_KT_LAUNCH(PI_KT_OTHER, 0, 1, bytes, k_cache_move, dim3((unsigned) (n * blocks)), dim3(1024), 0, (hipStream_t) stream, A, source, blocks, of_wave, keep, cells, pi_abort_word());
        PI_CHECK_LAUNCH();
    }
    return 0;
}
