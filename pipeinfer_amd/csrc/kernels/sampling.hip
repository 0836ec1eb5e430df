// A token for every row of logits, from a given random number.
//
//   order: larger logits first, the lower id on a tie; minus infinity and what is no number are not there
//   top-k: the first top_k (0 or less: all)                                          w = exp(x - max)
//   top-p: of those, the ones whose weights ahead of them add up to less than top_p * (the weights of all of them), and the first       (1 or more: all)
//   min-p: of those, the ones with w >= min_p, and the first
//   e = exp((x - max) / temperature) of what stays (temperature 0 or less: of the first alone);  the token: in the order of the ids the first whose running sum of e exceeds u * (the sum of all), its probability e / sum
//
// Sums are whole numbers, weights in steps of 2^-44 (a row of 2^19 of the largest weight fits 64 bits): the order of additions, and with it of atomics, is without effect, and a sum is off by less than the number of its terms x 2^-45
// of a total of at least 1.  Exponentials are fp64, within 1.5e-13: with fp32's the borders of thousands of candidates would move by whole tokens.
// Rows of up to 32768 logits: a workgroup each, the values in registers (k_sample).  Bound by the steps one after the other, code that runs once for the most part (1 row of 32000, top-k 40: 11 us; 64 of 32768, top-p 0.95: 39).
//   few of the best (top_k up to 128): what every wave has its sixteenth of top_k lanes above bounds the top_k-th from below; what reaches the bound - a few times top_k values - is listed in LDS, ranked there, and one wave does the rest
//   any number: the weights are added up in bins of equal width below the maximum, the bin that holds the border is listed and ranked
// Longer rows in slices of 8192, so that a few of them fill the chip, in four launches (4 rows of 32768 by a workgroup each: top-k 20 10.9 us, top-p 0.95 36; of 50000 in slices 15.3 and 32):
//   k_sample_slice   few of the best: the slice's list; otherwise the slice's largest value, and of every bin the count or the sum of the weights, 16 bits of each
//   k_sample_border  a workgroup per row: few of the best to the end; otherwise the bins in which the border lies (one, or two where it is too near the edge for sums of 16 bits)
//   k_sample_exact   the exact sums of what lies above those bins, the list of what lies in them (top_k up to 1024: of all from there up)
//   k_sample_join    a workgroup per row: the border's rank, and the token from the slices' sums.  A row whose lists are too long, whose bins begin too low, or with a top_k above 1024: the whole row from memory, as k_sample does
// A list that does not fit gives way to the digits of (value, id), eight bits a pass.
#include "ops_common.h"
#include "kernel_timing.h"
#include "wave_scan.h"

#include <algorithm>

#define SP_THREADS 1024
#define SP_WAVES (SP_THREADS / 64)
#define SP_BINS 4096
#define SP_PER_UNIT 128.0f   /* bins to a unit of logits: 32 below the maximum; 330 values in the fullest where 2^18 are spread by 2.5 */
#define SP_RANKED 512        /* entries that are ranked by counting, a thread each */
#define SP_LIST 2048
#define SP_BEST 1024
#define SP_SLICE 8192        /* values of a slice, 32 to a thread */
#define SP_RUN 512           /* values whose chances are added up by themselves */
#define SP_RUNS (SP_SLICE / SP_RUN)
#define SP_COARSE 2048       /* a slice's bins */
#define SP_COARSE_UNIT 64.0f /* of them to a unit of logits, or twice to sixteen times as many (sp_unit) */
#define SP_AHEAD 512.0f      /* how many lie above the largest of the row's first 1024 values: 24 units below it are left at 64 to a unit */
#define SP_POOL 8192         /* entries of a row's lists of few */
#define SP_SLICE_LIST 512
#define SP_REGISTERS 32768   /* longest row whose values stay in a workgroup's registers */
#define SP_ONE 17592186044416.0    /* 2^44 */
#define SP_HALF 0x1p-45      /* half a step: a weight up to here is none (sp_steps) */
#define SP_MAX_VOCAB (1 << 19)

typedef unsigned long long sp_u64;
// e^x, x <= 0 (or a little above): x = n ln 2 / 256 + r, 2^(n / 256) from a table (sp_table) and the exponent, e^r by its series up to r^3 / 6, |r| <= 0.00136 (the next term: 1.4e-13)
#define SP_TABLE 256
static __device__ __forceinline__ double sp_scaled(double s, double p, int n) {      // s 2^(n / 256): the table's value p with another exponent
    return s * __builtin_bit_cast(double, __builtin_bit_cast(sp_u64, p) + ((sp_u64) (uint32_t) ((n >> 8) << 20) << 32));
}
static __device__ __forceinline__ double sp_exp(double x, const double * table) {
    x = fmax(x, -600.0);                                     // (1e-260 for nothing: a choice of 0 instead would be a branch, and every exponential would wait for the one before)
    const double t = fma(x, 369.32993046757462871, 0x1.8p52), r = fma(t - 0x1.8p52, -0.0027076061740622863649, x);          // (n: the low bits of t)
    const int n = (int) (uint32_t) __builtin_bit_cast(sp_u64, t);
    return sp_scaled(fma(fma(fma(1.0 / 6.0, r, 0.5), r, 1.0), r, 1.0), table[n & 255], n);
}
// four of them (x >= -600) side by side: one by one their latency - a dozen dependent fp64 instructions and the table, 350 clocks - is all the time
static __device__ __forceinline__ void sp_exp4(const double (&x)[4], double (&y)[4], const double * table) {
    double t[4], r[4], p[4], s[4];
    int n[4];
#pragma unroll
    for (int e = 0; e < 4; e++) t[e] = fma(x[e], 369.32993046757462871, 0x1.8p52);
#pragma unroll
    for (int e = 0; e < 4; e++) { n[e] = (int) (uint32_t) __builtin_bit_cast(sp_u64, t[e]); p[e] = table[n[e] & 255]; r[e] = fma(t[e] - 0x1.8p52, -0.0027076061740622863649, x[e]); }
#pragma unroll
    for (int e = 0; e < 4; e++) s[e] = fma(1.0 / 6.0, r[e], 0.5);
#pragma unroll
    for (int e = 0; e < 4; e++) s[e] = fma(s[e], r[e], 1.0);
#pragma unroll
    for (int e = 0; e < 4; e++) s[e] = fma(s[e], r[e], 1.0);
#pragma unroll
    for (int e = 0; e < 4; e++) y[e] = sp_scaled(s[e], p[e], n[e]);
}
// 2^(i / 256) by the series of e^(i ln 2 / 256 - ln 2 / 2) up to its 15th power, times the root of two (by the first 256 threads)
static __device__ __forceinline__ void sp_table(double * table) {
    const int i = threadIdx.x;
    if (i >= SP_TABLE) return;
    const double x = (double) (i - 128) * 0.0027076061740622863649;
    double s = 1.0;
#pragma unroll
    for (int k = 15; k > 0; k--) s = fma(s * x, 1.0 / (double) k, 1.0);
    table[i] = s * 1.4142135623730950488;
}
// in steps: a weight, as the fraction of a double of 2^52; a sum of weights
static __device__ __forceinline__ sp_u64 sp_steps(double w) { return __builtin_bit_cast(sp_u64, fma(w, SP_ONE, 0x1p52)) & 0xfffffffffffffull; }
static __device__ __forceinline__ sp_u64 sp_sum_steps(double sum) { return (sp_u64) (sum * SP_ONE + 0.5); }

// larger value first, then the lower id; 0: not there
static __device__ __forceinline__ sp_u64 sp_rank(float x, int id) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return (sp_u64) (b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (uint32_t) ~id;
}
static __device__ __forceinline__ float sp_value(sp_u64 r) { const uint32_t k = (uint32_t) (r >> 32); return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
static __device__ __forceinline__ int sp_id(sp_u64 r) { return (int) ~(uint32_t) r; }

static __device__ __forceinline__ sp_u64 sp_wave_sum(sp_u64 v) { pi_butterfly<32>([&](auto o) { v += pi_partner<decltype(o)::value>(v); }); return v; }
static __device__ __forceinline__ sp_u64 sp_wave_top(sp_u64 v) { pi_butterfly<32>([&](auto o) { const sp_u64 x = pi_partner<decltype(o)::value>(v); v = x > v ? x : v; }); return v; }

static __device__ __forceinline__ int sp_lane(int v, int l) { return __builtin_amdgcn_readlane(v, l); }
static __device__ __forceinline__ sp_u64 sp_lane(sp_u64 v, int l) { return (sp_u64) (uint32_t) __builtin_amdgcn_readlane((int) (v >> 32), l) << 32 | (uint32_t) __builtin_amdgcn_readlane((int) v, l); }

// how many of the wave's lanes ahead of this one say so
static __device__ __forceinline__ int sp_rank_in(unsigned long long who) { return (int) __builtin_amdgcn_mbcnt_hi((uint32_t) (who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t) who, 0u)); }

struct sp_args {
    const float * logits; int64_t stride; int vocab;
    const float * temp; const int32_t * top_k; const float * top_p, * min_p, * u;
    int32_t * id; float * prob; int32_t * kept;
};

// what the launches over slices hand on: values above `above` are added up, those above `listed` listed; joined 0: left to one workgroup
struct sp_slice { sp_u64 best, listed, weights, above, kept, chances[SP_RUNS]; double over; };
struct sp_rest { sp_u64 best; float zero, above, listed; int32_t open, joined; float unit; };
static int sp_slices(int vocab) { return (vocab + SP_SLICE - 1) / SP_SLICE; }
struct sp_scratch { sp_rest * rest; sp_slice * slices; sp_u64 * lists; uint32_t * bins; };          // [row], [row][slice], [row][slice][SP_SLICE_LIST], [row][slice][SP_COARSE]

struct __attribute__((aligned(16))) sp_shared {
    sp_u64 weight[SP_BINS]; uint32_t count[SP_BINS];         // bins; digits
    double table[SP_TABLE];
    sp_u64 list[SP_LIST], chance[SP_BEST], waves[SP_WAVES]; int n, hit; sp_u64 before, answer;
};

static __device__ __forceinline__ sp_u64 sp_all_sum(sp_u64 v, sp_shared & L, int lane, int wave) {
    v = sp_wave_sum(v);
    __syncthreads();
    if (lane == 0) L.waves[wave] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int i = 0; i < SP_WAVES; i++) v += L.waves[i];
    return v;
}
// this thread's share of a running sum: what the threads ahead of it have; `all`: everybody's
static __device__ __forceinline__ sp_u64 sp_before(sp_u64 v, sp_shared & L, int lane, int wave, sp_u64 & all) {
    const sp_u64 x = pi_wave_scan(v);
    __syncthreads();
    if (lane == 63) L.waves[wave] = x;
    __syncthreads();
    sp_u64 base = 0; all = 0;
#pragma unroll
    for (int i = 0; i < SP_WAVES; i++) { const sp_u64 w = L.waves[i]; if (i < wave) base += w; all += w; }
    return base + x - v;
}


// a row's settings, and what is known of it so far
struct sp_row {
    const float * x; int V; float top_p, min_p; double cooled; bool greedy; int k; const double * table;
    float top, zero, unit; sp_u64 best, last;                // the first of the order; where the bins begin; the slices' bins to a unit; nothing below the rank `last` stays
    __device__ __forceinline__ sp_row(const sp_args & A, int row, const double * t) : table(t) {
        x = A.logits + (int64_t) row * A.stride; V = A.vocab;
        const float temp = A.temp ? A.temp[row] : 1.0f;
        top_p = A.top_p ? A.top_p[row] : 1.0f; min_p = A.min_p ? A.min_p[row] : 0.0f; k = A.top_k ? A.top_k[row] : 0;
        greedy = !(temp > 0.0f); cooled = greedy ? 1.0 : 1.0 / (double) temp;
        top = zero = 0.0f; unit = SP_COARSE_UNIT; best = last = 0;
        if (k < 0 || k >= V) k = 0;
        if (min_p > 1.0f) k = 1;                             // (nothing reaches it: the first alone)
    }
    __device__ __forceinline__ void known(sp_u64 b) { best = b; top = zero = sp_value(b); }
    __device__ __forceinline__ bool nucleus() const { return top_p < 1.0f; }
    __device__ __forceinline__ double below(float v) const { return v == top ? 0.0 : (double) v - (double) top; }        // (an infinite maximum: 0 of itself)
    __device__ __forceinline__ double weight(float v) const { return sp_exp(below(v), table); }
    __device__ __forceinline__ double chance(float v) const { return sp_exp(below(v) * cooled, table); }
    __device__ __forceinline__ bool enough(double w) const { return !(min_p > 0.0f) || w >= (double) min_p; }
    __device__ __forceinline__ int bin(float v) const { return (int) fminf(v >= zero ? 0.0f : (zero - v) * SP_PER_UNIT, (float) (SP_BINS - 1)); }
    // the slices' bins, from `zero` on, a value's place in its bin in `rest`; what is no number or not there: the last
    __device__ __forceinline__ int coarse(float v, float & rest) const {
        const float d = __builtin_amdgcn_fmed3f((zero - v) * unit, 0.0f, (float) SP_COARSE - 0.5f), f = floorf(d);
        rest = d - f;
        return (int) f;
    }
    __device__ __forceinline__ bool stays(float v, int id) const {
        if (!(v > -INFINITY)) return false;
        const sp_u64 r = sp_rank(v, id);
        return r >= last && (r == best || !(min_p > 0.0f) || enough(weight(v)));
    }
    __device__ __forceinline__ sp_u64 share(float v, int id) const { return greedy ? (sp_rank(v, id) == best ? sp_steps(1.0) : 0) : sp_steps(chance(v)); }
    __device__ __forceinline__ float part(float v, sp_u64 sum) const { return (float) ((greedy ? 1.0 : chance(v)) * SP_ONE / (double) sum); }
};
// Bins to a unit where the first 1024 values lie `spread` apart: the bins below the largest of them reach one and a half times that.  (64 rows of 250000 of deviation 1, top-p 0.95: of 64 bins to a unit one holds 1600, the lists are full and
// the rows go to a workgroup each, 754 us; of 128 to a unit 76)
static __device__ __forceinline__ float sp_unit(float spread) { return SP_COARSE_UNIT * (spread <= 1.0f ? 16.0f : spread <= 2.0f ? 8.0f : spread <= 4.0f ? 4.0f : spread <= 8.0f ? 2.0f : 1.0f); }
// the step of the sum that u falls on
static __device__ __forceinline__ sp_u64 sp_drawn(float u, sp_u64 sum) {
    const double want = (double) u * (double) sum;
    return want >= (double) sum ? sum - 1 : want > 0.0 ? min((sp_u64) want, sum - 1) : 0;
}
static __device__ __forceinline__ void sp_leave(const sp_args & A, int row, int id, float prob, int kept) {
    A.id[row] = id;
    if (A.prob) A.prob[row] = prob;
    if (A.kept) A.kept[row] = kept;
}

// bins from the top down, four to a thread: the bin in which a sum of `target` is reached, and what the bins ahead of it hold
template <class F> static __device__ __forceinline__ int sp_reach(sp_shared & L, sp_u64 target, F && bin, sp_u64 & ahead) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    sp_u64 v[4], s = 0, all;
#pragma unroll
    for (int e = 0; e < 4; e++) { v[e] = bin(4 * tid + e); s += v[e]; }
    sp_u64 b = sp_before(s, L, lane, wave, all);
    if (tid == 0) { L.hit = SP_BINS - 1; L.before = 0; }
    __syncthreads();
    if (b < target && b + s >= target) {
#pragma unroll
        for (int e = 0; e < 4; e++) { if (b < target && b + v[e] >= target) { L.hit = 4 * tid + e; L.before = b; } b += v[e]; }
    }
    __syncthreads();
    ahead = L.before;
    return L.hit;
}

// the token in the values [from, to), of which `t` of the sum is left.  (A run's sum may be above its values', which are rounded one by one: then it is the last of them.  What is no step by itself is not in the sum either, so one of them has a share)
static __device__ __forceinline__ void sp_pick(const sp_args & A, const sp_row & R, int row, int from, int to, sp_u64 t, sp_u64 sum, int kept) {
    const int lane = threadIdx.x & 63;
    int last = -1;
    for (int i0 = from; i0 < to; i0 += 64) {
        const int i = i0 + lane;
        const float v = i < to ? R.x[i] : -INFINITY;
        const sp_u64 mine = i < to && R.stays(v, i) ? R.share(v, i) : 0;
        const sp_u64 run = pi_wave_scan(mine), all = sp_lane(run, 63);
        if (t < all) {
            if (run > t && run - mine <= t) sp_leave(A, row, i, R.part(v, sum), kept);
            return;
        }
        t -= all;
        const unsigned long long who = __ballot(mine > 0);
        if (who) last = i0 + 63 - __builtin_clzll(who);
    }
    if (lane == 0 && last >= 0) sp_leave(A, row, last, R.part(R.x[last], sum), kept);
}
// the same for a run of values whose sum is held: the workgroup's waves take a sixteenth each
static __device__ __forceinline__ void sp_pick_run(const sp_args & A, const sp_row & R, sp_shared & L, int row, int from, int to, sp_u64 t, sp_u64 sum, int kept) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int part = 64 * ((to - from + SP_THREADS - 1) / SP_THREADS), a = min(from + wave * part, to), b = min(a + part, to);
    sp_u64 e = 0;
    for (int i = a + lane; i < b; i += 64) { const float v = R.x[i]; if (R.stays(v, i)) e += R.share(v, i); }
    e = sp_wave_sum(e);
    __syncthreads();
    if (lane == 0) L.waves[wave] = e;
    __syncthreads();
    int sub = 0, last = 0;
    for (int i = 0; i < SP_WAVES; i++) if (L.waves[i] > 0) last = i;
    while (sub < last && t >= L.waves[sub]) t -= L.waves[sub++];
    if (wave == sub) sp_pick(A, R, row, a, b, t, sum, kept);
}

// the rank at which `target` is reached by its digits, over the values at or above R.last; measure(v): 1 or a weight
template <class F> static __device__ __forceinline__ sp_u64 sp_digits(const sp_row & R, sp_shared & L, sp_u64 target, F && measure) {
    sp_u64 prefix = 0;
    for (int p = 7; p >= 0; p--) {
        __syncthreads();
        for (int i = threadIdx.x; i < 256; i += SP_THREADS) L.weight[i] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < R.V; i += SP_THREADS) {
            const float v = R.x[i];
            if (!(v > -INFINITY)) continue;
            const sp_u64 r = sp_rank(v, i);
            if (r >= R.last && (p == 7 || r >> (8 * p + 8) == prefix)) atomicAdd(&L.weight[r >> (8 * p) & 255], measure(v));
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            int d = 255;
            sp_u64 left = target;
            for (; d > 0 && L.weight[d] < left; d--) left -= L.weight[d];
            L.hit = d; L.before = target - left;
        }
        __syncthreads();
        prefix = prefix << 8 | (sp_u64) L.hit; target -= L.before;
    }
    return prefix;
}
// the same from a list of n up to SP_RANKED whose measures stand in L.weight (~0: not reached)
static __device__ __forceinline__ sp_u64 sp_ranked(const sp_row & R, sp_shared & L, int n, sp_u64 target) {
    __syncthreads();
    if (threadIdx.x == 0) L.answer = ~0ull;
    __syncthreads();
    if ((int) threadIdx.x < n) {
        const sp_u64 r = L.list[threadIdx.x];
        sp_u64 ahead = 0;
#pragma unroll 8
        for (int i = 0; i < n; i++) { const sp_u64 o = L.list[i], m = L.weight[i]; ahead += o > r && o >= R.last ? m : 0; }
        if (r >= R.last && ahead < target) atomicMin(&L.answer, r);          // (the last that is not behind the target)
    }
    __syncthreads();
    return L.answer;
}
// list[0 .. n) in falling order; n <= SP_LIST, behind it zeros up to the power of two
static __device__ __forceinline__ void sp_sort(sp_u64 * list, int n) {
    int m = 2;
    while (m < n) m <<= 1;
    for (int i = n + threadIdx.x; i < m; i += SP_THREADS) list[i] = 0;
    for (int size = 2; size <= m; size <<= 1)
        for (int d = size >> 1; d > 0; d >>= 1) {
            __syncthreads();
            for (int p = threadIdx.x; p < m / 2; p += SP_THREADS) {
                const int i = 2 * p - (p & (d - 1)), j = i + d;
                const sp_u64 a = list[i], b = list[j];
                if ((a < b) == ((i & size) == 0)) { list[i] = b; list[j] = a; }
            }
        }
    __syncthreads();
}

// a key that at least r of the wave's lanes reach (0: fewer have one), 16 bits of it
static __device__ __forceinline__ uint32_t sp_bound(uint32_t key, int r) {
    uint32_t t = 0;
#pragma unroll 1
    for (int b = 31; b >= 16; b--) { const uint32_t c = t | 1u << b; if (__popcll(__ballot(key >= c)) >= r) t = c; }
    return t;
}
static __device__ __forceinline__ uint32_t sp_key(float v) { return v > -INFINITY ? (uint32_t) (sp_rank(v, 0) >> 32) : 0u; }
// The waves with a value, `mine` the largest, in enough of their lanes for twice their share of the first k (and in a quarter of them) bound it: each a share of all k; without one there is little to list.  (A wave with few has a
// low bound: where all took part, a row of 31000 whose last wave had 280 values took 26 us, one of 32000 12; where only those with something in every lane did, 4 masked rows of 8000 took 20 instead of 9)
template <int WAVES> static __device__ __forceinline__ uint32_t sp_wave_bound(uint32_t * bounds, float mine, int k) {
    const int wave = threadIdx.x >> 6, have = __popcll(__ballot(mine > -INFINITY));
    const bool joins = have >= max(16, 2 * ((k + WAVES - 1) / WAVES));
    if ((threadIdx.x & 63) == 0) bounds[WAVES + wave] = joins;
    __syncthreads();
    uint32_t waves = 0, bound = ~0u;
#pragma unroll
    for (int i = 0; i < WAVES; i++) waves += bounds[WAVES + i];
    if (waves == 0) return 0;
    const uint32_t b = joins ? sp_bound(sp_key(mine), (k + (int) waves - 1) / (int) waves) : ~0u;
    if ((threadIdx.x & 63) == 0) bounds[wave] = b;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WAVES; i++) bound = min(bound, bounds[i]);
    return bound;
}
static __device__ __forceinline__ float sp_at_least(uint32_t key) { return key == 0 ? -INFINITY : sp_value((sp_u64) key << 32); }

// The first k of the order are among the n <= 128 of L.list: the rest of the way by one wave.  A lane has the places `lane` and, where there are more than 64, lane + 64 of the order
static __device__ __forceinline__ void sp_of_few(const sp_args & A, sp_row & R, sp_shared & L, int row, int n) {
    const int lane = threadIdx.x & 63, k = min(R.k, n);
    {
        const sp_u64 a = lane < n ? L.list[lane] : 0, b = lane + 64 < n ? L.list[lane + 64] : 0;
        int at_a = 0, at_b = 0;
        if (n <= 64) {
#pragma unroll 8
            for (int i = 0; i < n; i++) at_a += L.list[i] > a;
        } else
#pragma unroll 8
            for (int i = 0; i < n; i++) { const sp_u64 o = L.list[i]; at_a += o > a; at_b += o > b; }
        if (lane < n) L.chance[at_a] = a;
        if (lane + 64 < n) L.chance[at_b] = b;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    R.known(L.chance[0]);
    sp_u64 r[2], e[2] = { 0, 0 }, before = 0, edge_sum = 0;
    double w[2], c[2] = { 0.0, 0.0 };
    bool stays[2];
    int id[2], kept = 0;
    const int sets = k <= 64 ? 1 : 2;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        stays[i] = i < sets && lane + 64 * i < k;
        r[i] = stays[i] ? L.chance[lane + 64 * i] : 0; id[i] = sp_id(r[i]); w[i] = 0.0;
        if (i < sets) w[i] = stays[i] ? R.weight(sp_value(r[i])) : 0.0;
    }
    if (R.nucleus()) {
        sp_u64 s[2], run[2];
        for (int i = 0; i < sets; i++) { s[i] = stays[i] ? sp_steps(w[i]) : 0; run[i] = pi_wave_scan(s[i]); edge_sum += sp_lane(run[i], 63); }
        const double edge = (double) R.top_p * (double) edge_sum;
        for (int i = 0; i < sets; i++) { stays[i] = stays[i] && (lane + i == 0 || (double) (before + run[i] - s[i]) < edge); before += sp_lane(run[i], 63); }
    }
    sp_u64 sum = 0;
    for (int i = 0; i < sets; i++) {
        stays[i] = stays[i] && (lane + i == 0 || R.enough(w[i]));
        kept += __popcll(__ballot(stays[i]));
        if (R.greedy) c[i] = stays[i] && lane + i == 0 ? 1.0 : 0.0;
        else c[i] = stays[i] ? R.cooled == 1.0 ? w[i] : R.chance(sp_value(r[i])) : 0.0;
        e[i] = stays[i] ? sp_steps(c[i]) : 0;
        sum += e[i];
    }
    sum = sp_wave_sum(sum);
    const sp_u64 t = sp_drawn(A.u[row], sum);
    sp_u64 upto[2] = { 0, 0 };                               // what the ids up to its own add up to (what stays is ahead in the order)
    for (int l = 0; l < min(kept, 64); l++) {
        const int p = sp_lane(id[0], l);
        const sp_u64 x = sp_lane(e[0], l);
        upto[0] += p <= id[0] ? x : 0;
        if (kept > 64) upto[1] += p <= id[1] ? x : 0;
    }
    for (int l = 0; l < kept - 64; l++) {
        const int p = sp_lane(id[1], l);
        const sp_u64 x = sp_lane(e[1], l);
        upto[0] += p <= id[0] ? x : 0; upto[1] += p <= id[1] ? x : 0;
    }
    // the first id whose sum exceeds t: the one with a - e <= t < a
    const bool h0 = e[0] > 0 && upto[0] > t && upto[0] - e[0] <= t, h1 = e[1] > 0 && upto[1] > t && upto[1] - e[1] <= t;
    if (h0 || h1) sp_leave(A, row, h0 ? id[0] : id[1], (float) ((h0 ? c[0] : c[1]) * SP_ONE / (double) sum), kept);
}

// The same with more of them (k <= SP_BEST) by the workgroup
static __device__ __forceinline__ void sp_of_best(const sp_args & A, sp_row & R, sp_shared & L, int row, int n) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int k = min(R.k, n);
    if (n <= SP_RANKED / 2) {
        const sp_u64 r = tid < n ? L.list[tid] : 0;
        int at = 0;
        if (tid < n)
#pragma unroll 8
            for (int i = 0; i < n; i++) at += L.list[i] > r;
        __syncthreads();
        if (tid < n) L.list[at] = r;
        __syncthreads();
    } else sp_sort(L.list, n);
    R.known(L.list[0]);
    const sp_u64 r = tid < k ? L.list[tid] : 0;
    const double w = tid < k ? R.weight(sp_value(r)) : 0.0;
    bool stays = tid < k;
    if (R.nucleus()) {
        sp_u64 all;
        const sp_u64 before = sp_before(sp_steps(w), L, lane, wave, all);
        stays = stays && (tid == 0 || (double) before < (double) R.top_p * (double) all);
    }
    stays = stays && (tid == 0 || R.enough(w));
    const int kept = __syncthreads_count(stays);              // (what stays is ahead in the order)
    const float v = sp_value(r);
    const double c = !stays ? 0.0 : R.greedy ? (tid == 0 ? 1.0 : 0.0) : R.chance(v);
    const sp_u64 e = sp_steps(c), sum = sp_all_sum(e, L, lane, wave), t = sp_drawn(A.u[row], sum);
    const int id = sp_id(r);
    sp_u64 upto = 0;                                         // what the ids up to its own add up to
    if (kept <= 2 * 64) {
        if (tid < kept) { L.chance[tid] = e; L.weight[tid] = (sp_u64) id; }
        __syncthreads();
        if (tid < kept)
#pragma unroll 8
            for (int i = 0; i < kept; i++) upto += (int) L.weight[i] <= id ? L.chance[i] : 0;
        if (tid < kept && e > 0 && upto > t && upto - e <= t) sp_leave(A, row, id, R.part(v, sum), kept);
        return;
    }
    // (in the order of the ids, each with its place in the list)
    __syncthreads();
    if (tid < kept) { L.chance[tid] = e; L.list[tid] = (sp_u64) (uint32_t) ~id << 32 | (uint32_t) tid; }
    __syncthreads();
    sp_sort(L.list, kept);
    const int from = tid < kept ? (int) (uint32_t) L.list[tid] : 0;
    const sp_u64 mine = tid < kept ? L.chance[from] : 0;
    sp_u64 all;
    upto = sp_before(mine, L, lane, wave, all) + mine;
    if (mine > 0 && upto > t && upto - mine <= t) {
        const int i = (int) ~(uint32_t) (L.list[tid] >> 32);
        sp_leave(A, row, i, R.part(R.x[i], sum), kept);
    }
}

// A row by one workgroup.  VPT > 0: up to 1024 VPT values stay in registers.  A wave has a run of `chunk` ids, 256 of them a step: four to a lane side by side where rows lie on 16 bytes and end there (WIDE)
template <int VPT, bool WIDE> struct sp_values {
    const float * x; int V, steps, chunk, first, end, lane;
    float own[VPT > 0 ? VPT : 1];
    __device__ __forceinline__ int id(int j, int e) const { return first + 256 * j + (WIDE ? 4 * lane + e : 64 * e + lane); }
    // (without a branch, so that many are on their way at once)
    __device__ __forceinline__ void load(int j, float * to, int at) const {
        if constexpr (WIDE) {
            const float4 v = *(const float4 *) (x + min(id(j, 0), V - 4));
            const bool is = j < steps && id(j, 0) < end;
            to[at] = is ? v.x : -INFINITY; to[at + 1] = is ? v.y : -INFINITY; to[at + 2] = is ? v.z : -INFINITY; to[at + 3] = is ? v.w : -INFINITY;
        } else
#pragma unroll
            for (int e = 0; e < 4; e++) { const float v = x[min(id(j, e), V - 1)]; to[at + e] = j < steps && id(j, e) < end ? v : -INFINITY; }
    }
    __device__ __forceinline__ sp_values(const float * row, int n) : x(row), V(n) {
        lane = threadIdx.x & 63; chunk = (V + 4 * SP_WAVES - 1) / (4 * SP_WAVES) * 4; steps = (chunk + 255) / 256; first = (int) (threadIdx.x >> 6) * chunk; end = min(first + chunk, V);
        if constexpr (VPT > 0)
#pragma unroll
            for (int j = 0; j < VPT / 4; j++) load(j, own, 4 * j);
    }
    // in(value, id) of the thread's values as bits (minus infinity for what is not there or another wave's), 32 at a time: done(bits, the first one's step); whole waves call
    template <class F, class G> __device__ __forceinline__ void marked(F && in, G && done) const {
        if constexpr (VPT > 0) {
            uint32_t bits = 0;
#pragma unroll
            for (int i = 0; i < VPT; i++) bits |= (own[i] > -INFINITY && in(own[i], id(i / 4, i % 4)) ? 1u : 0u) << i;
            done(bits, 0);
        } else
            for (int j0 = 0; j0 < steps; j0 += 8) {
                float v[32];
#pragma unroll
                for (int j = 0; j < 8; j++) load(j0 + j, v, 4 * j);
                uint32_t bits = 0;
#pragma unroll
                for (int i = 0; i < 32; i++) bits |= (v[i] > -INFINITY && in(v[i], id(j0 + i / 4, i % 4)) ? 1u : 0u) << i;
                done(bits, j0);
            }
    }
    // f(value, id) of the thread's values that are there
    template <class F> __device__ __forceinline__ void each(F && f) const {
        if constexpr (VPT > 0) {
#pragma unroll
            for (int j = 0; j < VPT / 4; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) { const float v = own[4 * j + e]; if (v > -INFINITY) f(v, id(j, e)); }
        } else
            for (int j0 = 0; j0 < steps; j0 += 8) {          // (eight loads on their way at a time: one by one a pass over 131072 values waits 32 times)
                float v[32];
#pragma unroll
                for (int j = 0; j < 8; j++) load(j0 + j, v, 4 * j);
#pragma unroll
                for (int j = 0; j < 8; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++) { const float w = v[4 * j + e]; if (w > -INFINITY) f(w, id(j0 + j, e)); }
            }
    }
};
// The ranks of the values with a bit into `list`, in any order, while there is room; `count` goes up by how many there are.  A few of a row: what is listed is read once more, and the code is short (with a ballot and the store for each of
// a thread's 32 values, all of it code that runs once, the list of 40 of 32000 took 8000 clocks and takes 4800)
template <class F> static __device__ __forceinline__ void sp_list_few(uint32_t bits, int * count, int room, sp_u64 * list, const float * x, F && id_of) {
    const int lane = threadIdx.x & 63, n = __popc(bits), upto = (int) pi_wave_scan((uint32_t) n), all = __builtin_amdgcn_readlane(upto, 63);
    if (all == 0) return;
    int at = 0;
    if (lane == 0) at = atomicAdd(count, all);
    at = __builtin_amdgcn_readfirstlane(at) + upto - n;
#pragma unroll 1
    for (; bits; bits &= bits - 1, at++) {
        const int id = id_of(__builtin_ctz(bits));
        if (at < room) list[at] = sp_rank(x[id], id);
    }
}
// the ranks of what `in` says into L.list, in any order; how many there are (more than the list holds: the list is of no use)
template <class S, class F> static __device__ __forceinline__ int sp_gather(const S & X, sp_shared & L, F && in) {
    __syncthreads();
    if (threadIdx.x == 0) L.n = 0;
    __syncthreads();
    X.marked(in, [&](uint32_t bits, int j0) __attribute__((always_inline)) { sp_list_few(bits, &L.n, SP_LIST, L.list, X.x, [&](int i) __attribute__((always_inline)) { return X.id(j0 + i / 4, i % 4); }); });
    __syncthreads();
    return L.n;
}

template <class S> static __device__ __forceinline__ void sp_any_number(const sp_args & A, sp_row & R, sp_shared & L, const S & X, int row) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int k = R.k;
    if (k > 0) {                                             // (no more than there are: no border)
        sp_u64 present = 0;
        X.each([&](float, int) __attribute__((always_inline)) { present++; });
        if ((sp_u64) k >= sp_all_sum(present, L, lane, wave)) k = 0;
    }
    // the last of the order that stays: measure 1 or weights, so much of it reached
    if (k > 0 || R.nucleus()) {
        __syncthreads();
        for (int i = tid; i < SP_BINS; i += SP_THREADS) { L.weight[i] = 0; L.count[i] = 0; }
        __syncthreads();
        X.each([&](float v, int) __attribute__((always_inline)) {
            const int b = R.bin(v);
            if (k > 0) atomicAdd(&L.count[b], 1u);
            if (R.nucleus()) atomicAdd(&L.weight[b], sp_steps(R.weight(v)));
        });
        __syncthreads();
        // (the weights of a list's entries take the place of the bins' where those have been read)
        sp_u64 held[4] = { 0, 0, 0, 0 };
        if (R.nucleus())
#pragma unroll
            for (int e = 0; e < 4; e++) held[e] = L.weight[4 * tid + e];
        if (k > 0) {
            sp_u64 ahead;
            const int edge = sp_reach(L, (sp_u64) k, [&](int i) __attribute__((always_inline)) { return (sp_u64) L.count[i]; }, ahead);
            const int n = sp_gather(X, L, [&](float v, int) __attribute__((always_inline)) { return R.bin(v) == edge; });
            const bool listed = n <= SP_RANKED;
            if (listed) {
                if (tid < n) L.weight[tid] = 1;
                R.last = sp_ranked(R, L, n, (sp_u64) k - ahead);
            } else R.last = sp_digits(R, L, (sp_u64) k, [](float) __attribute__((always_inline)) { return (sp_u64) 1; });
            if (R.nucleus()) {                               // of the bin at the edge only what stayed
                sp_u64 part = 0;
                if (listed) { if (tid < n && L.list[tid] >= R.last) part = sp_steps(R.weight(sp_value(L.list[tid]))); }
                else for (int i = tid; i < R.V; i += SP_THREADS) { const float v = R.x[i]; if (v > -INFINITY && R.bin(v) == edge && sp_rank(v, i) >= R.last) part += sp_steps(R.weight(v)); }
                part = sp_all_sum(part, L, lane, wave);
#pragma unroll
                for (int e = 0; e < 4; e++) held[e] = 4 * tid + e < edge ? held[e] : 4 * tid + e == edge ? part : 0;
            }
        }
        if (R.nucleus()) {
            sp_u64 s = 0, ahead;
#pragma unroll
            for (int e = 0; e < 4; e++) s += held[e];
            const sp_u64 total = sp_all_sum(s, L, lane, wave);
            // the first whose sum, itself included, is not less than top_p * total
            const double want = (double) R.top_p * (double) total;
            const sp_u64 target = min(want >= 1.0 ? (sp_u64) __builtin_ceil(want) : 1, total);
            const int bin = sp_reach(L, target, [&](int i) __attribute__((always_inline)) { return held[i & 3]; }, ahead);
            const int n = sp_gather(X, L, [&](float v, int id) __attribute__((always_inline)) { return R.bin(v) == bin && sp_rank(v, id) >= R.last; });
            if (n <= SP_RANKED) {
                if (tid < n) L.weight[tid] = sp_steps(R.weight(sp_value(L.list[tid])));
                R.last = sp_ranked(R, L, n, target - ahead);
            } else R.last = sp_digits(R, L, target, [&](float v) __attribute__((always_inline)) { return sp_steps(R.weight(v)); });
        }
    }
    sp_u64 kept = 0, e = 0;
    X.each([&](float v, int id) __attribute__((always_inline)) { if (R.stays(v, id)) { kept++; e += R.share(v, id); } });
    kept = sp_all_sum(kept, L, lane, wave);
    e = sp_wave_sum(e);
    __syncthreads();
    if (lane == 0) L.waves[wave] = e;
    __syncthreads();
    sp_u64 sum = 0;
#pragma unroll
    for (int i = 0; i < SP_WAVES; i++) sum += L.waves[i];
    sp_u64 t = sp_drawn(A.u[row], sum);
    int seg = 0;
    while (seg < SP_WAVES - 1 && t >= L.waves[seg]) t -= L.waves[seg++];
    sp_pick_run(A, R, L, row, min(seg * X.chunk, R.V), min((seg + 1) * X.chunk, R.V), t, sum, (int) kept);
}

template <int VPT, bool WIDE> __global__ void __launch_bounds__(SP_THREADS) k_sample(const sp_args A, const int32_t * __restrict__ abort_w) {
    const int gone = pi_abort_peek(abort_w);
    __shared__ sp_shared L;
    __shared__ uint32_t bounds[2 * SP_WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = blockIdx.x;
    sp_row R(A, row, L.table);
    const sp_values<VPT, WIDE> X(R.x, R.V);
    sp_table(L.table);
    if (pi_aborted_together(gone, abort_w)) return;
    // the largest value, a thread's and everybody's, and a bound that at least k of them reach
    float mine = -INFINITY; int mine_id = 0;
    X.each([&](float v, int id) __attribute__((always_inline)) { if (v > mine) { mine = v; mine_id = id; } });       // (a thread's ids ascend: the first of equals)
    const bool few = R.k > 0 && R.k <= 128;
    sp_u64 top = 0;
    if (few) {                                               // (the largest comes with the list)
        const float least = sp_at_least(sp_wave_bound<SP_WAVES>(bounds, mine, R.k));
        const int n = sp_gather(X, L, [&](float v, int) __attribute__((always_inline)) { return v >= least; });
        if (n == 0) {
            if (tid == 0) sp_leave(A, row, -1, 0.0f, 0);
            return;
        }
        if (n <= 128) {
            if (wave == 0) sp_of_few(A, R, L, row, n);
            return;
        }
        if (n <= SP_LIST) { sp_of_best(A, R, L, row, n); return; }
    }
    top = sp_wave_top(mine > -INFINITY ? sp_rank(mine, mine_id) : 0);
    if (lane == 0) L.waves[wave] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < SP_WAVES; i++) top = max(top, L.waves[i]);
    if (top == 0) {
        if (tid == 0) sp_leave(A, row, -1, 0.0f, 0);
        return;
    }
    R.known(top);
    sp_any_number(A, R, L, X, row);
}

// ---- rows in slices -----------------------------------------------------------------------------------------------------------------------------------------------------------------
// a slice's values, a run of them to a wave, 256 a step
template <bool WIDE> static __device__ __forceinline__ int sp_slice_id(int base, int j, int e) { const int lane = threadIdx.x & 63; return base + 256 * j + (WIDE ? 4 * lane + e : 64 * e + lane); }
template <bool WIDE, int STEPS> static __device__ __forceinline__ void sp_slice_load(const sp_row & R, int base, float (&x)[4 * STEPS]) {
#pragma unroll
    for (int j = 0; j < STEPS; j++) {
        const int i = sp_slice_id<WIDE>(base, j, 0);
        if constexpr (WIDE) {
            const float4 v = *(const float4 *) (R.x + min(i, R.V - 4));
            x[4 * j] = i < R.V ? v.x : -INFINITY; x[4 * j + 1] = i < R.V ? v.y : -INFINITY; x[4 * j + 2] = i < R.V ? v.z : -INFINITY; x[4 * j + 3] = i < R.V ? v.w : -INFINITY;
        } else
#pragma unroll
            for (int e = 0; e < 4; e++) { const float v = R.x[min(i + 64 * e, R.V - 1)]; x[4 * j + e] = i + 64 * e < R.V ? v : -INFINITY; }
    }
}

// Bound by the logits (256 rows of 131072: 30 us, 4.4 TB/s; 64 rows 16 us, the bins' atomics behind the only round of loads; 33 rows of 65024, lists alone, 6.5)
template <bool WIDE> __global__ void __launch_bounds__(256) k_sample_slice(const sp_args A, const sp_scratch S, int slices, const int32_t * __restrict__ abort_w) {
    const int gone = pi_abort_peek(abort_w), row = blockIdx.x / slices, slice = blockIdx.x % slices;
    __shared__ uint32_t bins[SP_COARSE], bounds[8];
    __shared__ sp_u64 tops[4];
    __shared__ float firsts[4], lows[4];
    __shared__ double overs[4];
    __shared__ int listed;
    __shared__ double table[SP_TABLE];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    sp_row R(A, row, table);
    // (the row's last values for the last slice, so that its waves are as full as the others': the fewer lanes, the lower a bound.  What stands in the slice before is taken out once the bound is known)
    const int begin = slice * SP_SLICE, from = min(begin, R.V - SP_SLICE), base = from + wave * (SP_SLICE / 4);
    float x[32], first = -INFINITY, low = INFINITY;
    sp_slice_load<WIDE, 8>(R, base, x);
    const bool few = R.k > 0 && R.k <= 128, border = !few && (R.k > 0 || R.nucleus());
    if (border)
#pragma unroll
        for (int e = 0; e < 4; e++) { const float v = R.x[256 * e + tid]; first = fmaxf(first, v); low = fminf(low, v > -INFINITY ? v : INFINITY); }         // (rows are longer)
    if (tid == 0) listed = 0;
    if (pi_aborted_together(gone, abort_w)) return;
    sp_slice * mine_of = S.slices + (int64_t) row * slices + slice;
    float mine = -INFINITY; int mine_id = 0;
#pragma unroll
    for (int e = 0; e < 32; e++) if (x[e] > mine) { mine = x[e]; mine_id = sp_slice_id<WIDE>(base, e / 4, e % 4); }
    auto own_ones = [&]() __attribute__((always_inline)) {
        if (from == begin) return;
#pragma unroll
        for (int e = 0; e < 32; e++) if (sp_slice_id<WIDE>(base, e / 4, e % 4) < begin) x[e] = -INFINITY;
    };
    if (few) {
        const float least = sp_at_least(sp_wave_bound<4>(bounds, mine, R.k));
        own_ones();
        sp_u64 * list = S.lists + ((int64_t) row * slices + slice) * SP_SLICE_LIST;
        uint32_t bits = 0;
#pragma unroll
        for (int e = 0; e < 32; e++) bits |= (x[e] >= least && x[e] > -INFINITY ? 1u : 0u) << e;
        sp_list_few(bits, &listed, SP_SLICE_LIST, list, R.x, [&](int e) __attribute__((always_inline)) { return sp_slice_id<WIDE>(base, e / 4, e % 4); });
        __syncthreads();
        if (tid == 0) mine_of->listed = (sp_u64) listed;
        return;
    }
    own_ones();
    sp_u64 top = sp_wave_top(mine > -INFINITY ? sp_rank(mine, mine_id) : 0);
    first = pi_wave_max(first); low = -pi_wave_max(-low);
    if (lane == 0) { tops[wave] = top; firsts[wave] = first; lows[wave] = low; }
    if (border) sp_table(table);
    if (border)
#pragma unroll
        for (int i = 0; i < SP_COARSE / 256; i++) bins[i * 256 + tid] = 0;
    __syncthreads();
    if (tid == 0) mine_of->best = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
    if (!border) return;
    first = fmaxf(fmaxf(firsts[0], firsts[1]), fmaxf(firsts[2], firsts[3]));
    low = fminf(fminf(lows[0], lows[1]), fminf(lows[2], lows[3]));
    R.unit = sp_unit(first - low);
    R.zero = (first > -INFINITY && first < INFINITY ? first : 0.0f) + SP_AHEAD / R.unit;
    const bool counts = R.k > 0;
    const float step = 1.0f / R.unit;
    double over = 0.0;                                       // the weights of what lies above the bins
#pragma unroll
    for (int e = 0; e < 32; e++) {
        if (!counts && __any(x[e] > R.zero)) { if (x[e] > R.zero) { over += sp_exp((double) x[e] - (double) R.zero, table); continue; } }
        float rest;
        const int b = R.coarse(x[e], rest);
        const float r = rest * step;
        // (of e^-r 16 bits, r <= 1/64: 8192 of them fit a bin; the series up to r^3 / 6, the next term: 2^-29)
        const uint32_t w = counts ? 1u : (uint32_t) fmaf(65536.0f, 1.0f - r * fmaf(-r, fmaf(r, -1.0f / 6.0f, 0.5f), 1.0f), 0.5f);
        if (x[e] > -INFINITY) atomicAdd(&bins[b], w);
    }
    if (!counts && __any(over != 0.0)) { over = pi_wave_sum_f64(over); if (lane == 0) overs[wave] = over; } else if (lane == 0) overs[wave] = 0.0;
    __syncthreads();
    if (tid == 0) mine_of->over = (overs[0] + overs[1]) + (overs[2] + overs[3]);
    uint32_t * to = S.bins + ((int64_t) row * slices + slice) * SP_COARSE;
#pragma unroll
    for (int i = 0; i < SP_COARSE / 1024; i++) *(uint4 *) (to + 1024 * i + 4 * tid) = *(const uint4 *) (bins + 1024 * i + 4 * tid);
    if (slice == 0 && tid == 0) { S.rest[row].zero = R.zero; S.rest[row].unit = R.unit; }
}

// Bound by its steps one after the other (64 rows of 131072 8 us, 33 rows of 65024 with their lists 11)
__global__ void __launch_bounds__(SP_THREADS) k_sample_border(const sp_args A, const sp_scratch S, int slices, const int32_t * __restrict__ abort_w) {
    const int gone = pi_abort_peek(abort_w), row = blockIdx.x;
    __shared__ sp_shared L;
    __shared__ sp_u64 pool[SP_POOL];
    __shared__ uint32_t bounds[SP_WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    sp_row R(A, row, L.table);
    const sp_slice * of = S.slices + (int64_t) row * slices;
    sp_rest * rest = S.rest + row;
    if (tid == 0) L.n = 0;
    sp_table(L.table);
    if (pi_aborted_together(gone, abort_w)) return;
    if (R.k > 0 && R.k <= 128) {
        // the slices' lists one after the other, what their threads' largest bound from them
        const int listed = lane < slices ? (int) of[lane].listed : 0;
        const int behind = (int) pi_wave_scan((uint32_t) listed);
        const int all = __builtin_amdgcn_readlane(behind, 63);
        const bool fits = !__any(listed > SP_SLICE_LIST) && all <= SP_POOL;
        if (tid == 0) *rest = sp_rest{ 0, 0.0f, 0.0f, 0.0f, fits ? 0 : 1, 0, 0 };
        if (!fits) return;
        if (all == 0) {
            if (tid == 0) sp_leave(A, row, -1, 0.0f, 0);
            return;
        }
        const sp_u64 * lists = S.lists + (int64_t) row * slices * SP_SLICE_LIST;
        for (int i = wave; i < slices; i += SP_WAVES) {
            const int end = __builtin_amdgcn_readlane(behind, i), c = __builtin_amdgcn_readlane(listed, i);
            for (int l = lane; l < c; l += 64) pool[end - c + l] = lists[i * SP_SLICE_LIST + l];
        }
        __syncthreads();
        sp_u64 mine = 0;
        for (int i = tid; i < all; i += SP_THREADS) mine = max(mine, pool[i]);
        // (of the waves whose lanes all have something, each its share of k)
        const int whole = min(SP_WAVES, all / 64), share = whole == 0 ? R.k : (R.k + whole - 1) / whole;
        const uint32_t b = sp_bound((uint32_t) (mine >> 32), share);
        if (lane == 0) bounds[wave] = b;
        __syncthreads();
        uint32_t bound = ~0u;
        for (int i = 0; i < max(whole, 1); i++) bound = min(bound, bounds[i]);
        for (int i = tid; i < all; i += SP_THREADS)
            if ((uint32_t) (pool[i] >> 32) >= bound) { const int at = atomicAdd(&L.n, 1); if (at < SP_LIST) L.list[at] = pool[i]; }
        __syncthreads();
        const int n = L.n;
        if (n <= 128) {
            if (wave == 0) sp_of_few(A, R, L, row, n);
            return;
        }
        if (n <= SP_LIST) sp_of_best(A, R, L, row, n);
        else if (tid == 0) rest->open = 1;
        return;
    }
    const sp_u64 best = sp_wave_top(lane < slices ? of[lane].best : 0);
    if (best == 0) {
        if (tid == 0) { sp_leave(A, row, -1, 0.0f, 0); rest->open = 0; }
        return;
    }
    R.known(best);
    if (R.k == 0 && !R.nucleus()) {                          // everything lies above
        if (tid == 0) *rest = sp_rest{ best, R.top, -INFINITY, -INFINITY, 1, R.top < INFINITY, 0 };
        return;
    }
    const float zero = rest->zero, unit = rest->unit;
    // two bins to a thread, over the slices
    const uint32_t * from = S.bins + (int64_t) row * slices * SP_COARSE + 2 * tid;
    sp_u64 a = 0, b = 0;
#pragma unroll 8
    for (int i = 0; i < slices; i++) { const uint2 v = *(const uint2 *) (from + i * SP_COARSE); a += v.x; b += v.y; }
    int lo, hi;
    if (R.k > 0) {
        sp_u64 all;
        const sp_u64 before = sp_before(a + b, L, lane, wave, all), k = min((sp_u64) R.k, all);
        if (before < k && before + a + b >= k) L.hit = 2 * tid + (before + a < k);
        __syncthreads();
        lo = 0; hi = R.k <= SP_BEST ? L.hit : -1;
    } else {
        const float each = 1.44269504f / unit, far = fmaxf((R.top - zero) * 1.44269504f, 0.0f);            // (relative to what is largest)
        double over = 0.0;
        if (tid == 0 && far > 0.0f) for (int i = 0; i < slices; i++) over += of[i].over;
        const double wa = (double) a * (double) __builtin_amdgcn_exp2f(-each * (float) (2 * tid) - far) + over * 65536.0 * (double) __builtin_amdgcn_exp2f(-far);
        const double wb = (double) b * (double) __builtin_amdgcn_exp2f(-each * (float) (2 * tid + 1) - far);
        const sp_u64 sa = (sp_u64) (wa * 268435456.0 + 0.5), sb = (sp_u64) (wb * 268435456.0 + 0.5);         // (steps of 2^-44 of the bins' beginning: the sums' 16 bits)
        sp_u64 all;
        const sp_u64 before = sp_before(sa + sb, L, lane, wave, all);
        if (tid == 0) { L.answer = SP_COARSE; L.before = 0; }
        __syncthreads();
        // (sums off by a few 2^-18 of themselves: the bins in which the border lies if it is that far to either side)
        const double want = fmax((double) R.top_p, 0.0) * (double) all, off = (double) all * 0x1p-17;
        const sp_u64 least = want - off >= 1.0 ? (sp_u64) (want - off) : 1, most = min((sp_u64) (want + off) + 1, all);
        if (before < least && before + sa + sb >= least) L.answer = 2 * tid + (before + sa < least);
        if (before < most && before + sa + sb >= most) L.before = 2 * tid + (before + sa < most);
        __syncthreads();
        lo = (int) L.answer; hi = (int) L.before;
    }
    // (far below an infinity, or bins that end too high: no)
    const bool joined = R.top - zero <= 100.0f && hi >= 0 && hi < SP_COARSE - 1 && fabsf(zero) * unit < 32768.0f * SP_COARSE_UNIT;
    // (half a bin further down: every value of bin hi is listed, whichever way its difference was rounded)
    if (tid == 0) *rest = sp_rest{ best, zero, lo == 0 ? INFINITY : zero - (float) lo / unit, zero - ((float) hi + 1.5f) / unit, 1, joined, unit };
}

// Sums of a run in fp64, in an order that is always the same, then in steps; of the chances without those that are no step by themselves, so that no run of nothing but such ones is drawn.  Bound by its instructions, the fp64 ones for the most part: 24 a value, 18 of them the two exponentials' (64 rows of 131072: with each value in steps 29, so 22 us;
// exponentials by two and three workgroups on a compute unit 21.5, four with spilled registers 28)
template <bool WIDE> __global__ void __launch_bounds__(512) k_sample_exact(const sp_args A, const sp_scratch S, int slices, const int32_t * __restrict__ abort_w) {
    const int gone = pi_abort_peek(abort_w), row = blockIdx.x / slices, slice = blockIdx.x % slices;
    const sp_rest rest = S.rest[row];
    if (rest.open == 0 || rest.joined == 0 || pi_aborted_together(gone, abort_w)) return;
    __shared__ int listed;
    __shared__ double table[SP_TABLE];
    __shared__ sp_u64 sums[8][3];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, base = slice * SP_SLICE + wave * (SP_SLICE / 8);
    sp_row R(A, row, table);
    R.known(rest.best);
    float x[16];
    sp_slice_load<WIDE, 4>(R, base, x);
    if (tid == 0) listed = 0;
    sp_table(table);
    __syncthreads();
    sp_slice * mine = S.slices + (int64_t) row * slices + slice;
    sp_u64 * list = S.lists + ((int64_t) row * slices + slice) * SP_SLICE_LIST;
    uint32_t bits = 0;
#pragma unroll
    for (int e = 0; e < 16; e++) bits |= (x[e] > rest.listed && !(x[e] > rest.above) ? 1u : 0u) << e;
    sp_list_few(bits, &listed, SP_SLICE_LIST, list, R.x, [&](int e) __attribute__((always_inline)) { return sp_slice_id<WIDE>(base, e / 4, e % 4); });
    if (R.k == 0) {                                          // (top-k: the list is all that is asked for)
        const bool once = R.cooled == 1.0, few_stay = R.min_p > 0.0f;
        const double top = (double) R.top;
        double all = 0.0, above = 0.0, chance = 0.0;
        int kept = 0;
#pragma unroll 1
        for (int run = 0; run < 2; run++) {
#pragma unroll
            for (int half = 0; half < 2; half++) {
                double below[4], d[4], w[4];
                bool stays[4];
#pragma unroll
                for (int e = 0; e < 4; e++) { const float v = run ? x[8 + 4 * half + e] : x[4 * half + e]; below[e] = (double) v - top; d[e] = fmax(below[e], -600.0); stays[e] = v > rest.above; }
                sp_exp4(d, w, table);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    all += w[e]; above += stays[e] ? w[e] : 0.0;
                    stays[e] = stays[e] && (!few_stay || w[e] >= (double) R.min_p);
                    kept += __popcll(__ballot(stays[e]));
                }
                if (!once && !R.greedy) {
#pragma unroll
                    for (int e = 0; e < 4; e++) d[e] = fmax(below[e] * R.cooled, -600.0);          // (of what is far below the largest a high temperature leaves something)
                    sp_exp4(d, w, table);
                }
#pragma unroll
                for (int e = 0; e < 4; e++) chance += stays[e] && w[e] > SP_HALF ? w[e] : 0.0;
            }
            const sp_u64 c = sp_sum_steps(pi_wave_sum_f64(chance));
            if (lane == 0) mine->chances[2 * wave + run] = c;
            chance = 0.0;
        }
        const sp_u64 a = sp_sum_steps(pi_wave_sum_f64(all)), b = sp_sum_steps(pi_wave_sum_f64(above));
        if (lane == 0) { sums[wave][0] = a; sums[wave][1] = b; sums[wave][2] = (sp_u64) kept; }
    }
    __syncthreads();
    if (wave == 0) {
        sp_u64 a = 0, b = 0, c = 0;
        if (R.k == 0 && lane < 8) { a = sums[lane][0]; b = sums[lane][1]; c = sums[lane][2]; }
        a = sp_wave_sum(a); b = sp_wave_sum(b); c = sp_wave_sum(c);
        if (lane == 0) { mine->weights = a; mine->above = b; mine->kept = c; mine->listed = (sp_u64) listed; }
    }
}

// the slices of a row; false: they do not say enough
static __device__ __forceinline__ bool sp_join(const sp_args & A, sp_row & R, sp_shared & L, int row, const sp_slice * mine, const sp_u64 * lists, int slices, bool border, float above_v, float least) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // (every wave for itself: a lane has a slice)
    static_assert(SP_MAX_VOCAB / SP_SLICE <= 64, "");
    sp_u64 weights = 0, above = 0, kept = 0, listed = 0;
    if (lane < slices) { weights = mine[lane].weights; above = mine[lane].above; kept = mine[lane].kept; listed = mine[lane].listed; }
    if (__any(listed > SP_SLICE_LIST)) return false;
    const int behind = (int) pi_wave_scan((uint32_t) listed);
    const int n = __builtin_amdgcn_readlane(behind, 63);
    if (n > SP_LIST) return false;
    for (int i = wave; i < slices; i += SP_WAVES) { const int end = __builtin_amdgcn_readlane(behind, i), c = __builtin_amdgcn_readlane((int) listed, i); for (int l = lane; l < c; l += 64) L.list[end - c + l] = lists[i * SP_SLICE_LIST + l]; }
    weights = sp_wave_sum(weights); above = sp_wave_sum(above); kept = sp_wave_sum(kept);
    if (tid == 0) L.answer = ~0ull;
    __syncthreads();
    if (R.k > 0) {
        if (n <= 128) { if (wave == 0) sp_of_few(A, R, L, row, n); }
        else sp_of_best(A, R, L, row, n);
        return true;
    }
    if (border) {
        // the border's rank: the list's weights in 512 bins of their own, and the ranks inside the one that the border is in
        const double want = (double) R.top_p * (double) weights;
        const sp_u64 target = min(want >= 1.0 ? (sp_u64) __builtin_ceil(want) : 1, weights);
        if (above >= target) return false;
        const float from = fminf(above_v, R.top), scale = 512.0f / fmaxf(from - least, 1e-30f);
        auto bin = [&](float v) __attribute__((always_inline)) { return (int) __builtin_amdgcn_fmed3f((from - v) * scale, 0.0f, 511.0f); };
        if (tid < 512) L.weight[tid] = 0;
        if (tid == 0) { L.n = 0; L.hit = -1; }
        __syncthreads();
        for (int i = tid; i < n; i += SP_THREADS) { const float v = sp_value(L.list[i]); atomicAdd(&L.weight[bin(v)], sp_steps(R.weight(v))); }
        __syncthreads();
        sp_u64 all;
        const sp_u64 mine_w = tid < 512 ? L.weight[tid] : 0, ahead = above + sp_before(mine_w, L, lane, wave, all);
        if (tid < 512 && ahead < target && ahead + mine_w >= target) { L.hit = tid; L.before = ahead; }
        __syncthreads();
        if (L.hit < 0) return false;
        const int hit = L.hit;
        const sp_u64 base = L.before;
        for (int i = tid; i < n; i += SP_THREADS) {
            const sp_u64 r = L.list[i];
            if (bin(sp_value(r)) == hit) { const int at = atomicAdd(&L.n, 1); L.weight[2 * at] = r; L.weight[2 * at + 1] = sp_steps(R.weight(sp_value(r))); }
        }
        __syncthreads();
        const int m = L.n;
        for (int i = tid; i < m; i += SP_THREADS) {
            const sp_u64 r = L.weight[2 * i];
            sp_u64 sum = base;
#pragma unroll 4
            for (int o = 0; o < m; o++) { const ulonglong2 x = *(const ulonglong2 *) &L.weight[2 * o]; sum += x.x > r ? x.y : 0; }
            if (sum < target) atomicMin(&L.answer, r);
        }
        __syncthreads();
        R.last = L.answer;
    }
    if (R.greedy) {                                          // (the first; how many stay is all there is to say)
        sp_u64 more = 0;
        for (int i = tid; i < n; i += SP_THREADS) more += R.stays(sp_value(L.list[i]), sp_id(L.list[i]));
        kept += sp_all_sum(more, L, lane, wave);
        if (tid == 0) sp_leave(A, row, sp_id(R.best), 1.0f, (int) kept);
        return true;
    }
    // the runs' chances with what stays of the list: a thread has a run
    static_assert(SP_MAX_VOCAB / SP_RUN <= SP_THREADS && SP_THREADS <= SP_BINS, "");
    const int runs = slices * SP_RUNS;
    __syncthreads();
    if (tid < runs) L.weight[tid] = mine[tid / SP_RUNS].chances[tid % SP_RUNS];
    __syncthreads();
    sp_u64 more = 0;
    for (int i = tid; i < n; i += SP_THREADS) {
        const sp_u64 r = L.list[i];
        const float v = sp_value(r);
        if (R.stays(v, sp_id(r))) { more++; atomicAdd(&L.weight[sp_id(r) / SP_RUN], R.share(v, sp_id(r))); }
    }
    kept += sp_all_sum(more, L, lane, wave);
    const sp_u64 e = tid < runs ? L.weight[tid] : 0;
    sp_u64 sum;
    const sp_u64 before = sp_before(e, L, lane, wave, sum), t = sp_drawn(A.u[row], sum);
    if (before <= t && before + e > t) { L.hit = tid; L.before = t - before; }
    __syncthreads();
    const int at = L.hit * SP_RUN;
    sp_pick_run(A, R, L, row, at, min(at + SP_RUN, R.V), L.before, sum, (int) kept);
    return true;
}

// (64 rows of 131072: 11 us, of steps one after the other)
template <bool WIDE> __global__ void __launch_bounds__(SP_THREADS) k_sample_join(const sp_args A, const sp_scratch S, int slices, const int32_t * __restrict__ abort_w) {
    const int gone = pi_abort_peek(abort_w), row = blockIdx.x;
    const sp_rest rest = S.rest[row];
    if (rest.open == 0 || pi_aborted_together(gone, abort_w)) return;
    __shared__ sp_shared L;
    sp_row R(A, row, L.table);
    if (rest.joined != 0) R.known(rest.best);
    sp_table(L.table);
    if (rest.joined != 0 && sp_join(A, R, L, row, S.slices + (int64_t) row * slices, S.lists + (int64_t) row * slices * SP_SLICE_LIST, slices, R.nucleus(), rest.above, rest.listed)) return;
    __syncthreads();
    const sp_values<0, WIDE> X(R.x, R.V);
    sp_u64 best = 0;
    X.each([&](float v, int id) __attribute__((always_inline)) { best = max(best, sp_rank(v, id)); });
    best = sp_wave_top(best);
    if ((threadIdx.x & 63) == 0) L.waves[threadIdx.x >> 6] = best;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < SP_WAVES; i++) best = max(best, L.waves[i]);
    R.known(best);
    R.last = 0;
    sp_any_number(A, R, L, X, row);
}

extern "C" size_t pi_op_sample_scratch_bytes(int n_vocab, int rows) {
    if (n_vocab <= SP_REGISTERS || n_vocab > SP_MAX_VOCAB || rows < 1) return 0;
    const size_t n = (size_t) rows * sp_slices(n_vocab);
    return n * (SP_COARSE * sizeof(uint32_t) + SP_SLICE_LIST * sizeof(sp_u64) + sizeof(sp_slice)) + rows * sizeof(sp_rest);
}

extern "C" int pi_op_sample(const float * logits, int64_t stride, int n_vocab, int rows, const float * temp, const int32_t * top_k, const float * top_p, const float * min_p, const float * u, void * scratch, size_t scratch_bytes,
                            int32_t * id, float * prob, int32_t * kept, void * stream) {
    if (rows < 0 || n_vocab < 1 || n_vocab > SP_MAX_VOCAB || stride < n_vocab) { pi_set_error("pi_op_sample: %d rows of %d logits (1 .. 524288), %lld apart", rows, n_vocab, (long long) stride); return -1; }
    if (rows == 0) return 0;
    if (!logits || !u || !id) { pi_set_error("pi_op_sample: logits, random numbers or ids are NULL"); return -1; }
    const size_t need = pi_op_sample_scratch_bytes(n_vocab, rows);
    if (need > 0 && (!scratch || ((uintptr_t) scratch & 15) || scratch_bytes < need)) { pi_set_error("pi_op_sample: %zu bytes of scratch, on 16, for %zu (pi_op_sample_scratch_bytes)", scratch ? scratch_bytes : 0, need); return -1; }
    const sp_args A{ logits, stride, n_vocab, temp, top_k, top_p, min_p, u, id, prob, kept };
    const bool wide = n_vocab % 4 == 0 && stride % 4 == 0 && ((uintptr_t) logits & 15) == 0;
    const int slices = sp_slices(n_vocab), nt = std::min(rows, PI_KT_MAXNT - 1);
    const hipStream_t s = (hipStream_t) stream;
    if (need == 0) {
#define SP_GO(V, W) PI_KT_LAUNCH(PI_KT_OTHER, 0, nt, 4.0 * rows * n_vocab, (k_sample<V, W>), dim3((unsigned) rows), dim3(SP_THREADS), 0, s, A, pi_abort_word())
        if (n_vocab <= SP_REGISTERS / 4) { if (wide) SP_GO(8, true); else SP_GO(8, false); }
        else if (wide) SP_GO(32, true);
        else SP_GO(32, false);
#undef SP_GO
        PI_CHECK_LAUNCH();
        return 0;
    }
    if ((int64_t) rows * slices > 0x7fffffff) { pi_set_error("pi_op_sample: %d rows of %d logits in one call", rows, n_vocab); return -1; }
    sp_scratch S{};
    S.bins = (uint32_t *) scratch;
    S.lists = (sp_u64 *) (S.bins + (size_t) rows * slices * SP_COARSE);
    S.slices = (sp_slice *) (S.lists + (size_t) rows * slices * SP_SLICE_LIST);
    S.rest = (sp_rest *) (S.slices + (size_t) rows * slices);
    const dim3 all((unsigned) (rows * slices)), each((unsigned) rows);
#define SP_GO(W) do { \
        PI_KT_LAUNCH(PI_KT_OTHER, 0, nt, 4.0 * rows * n_vocab, k_sample_slice<W>, all, dim3(256), 0, s, A, S, slices, pi_abort_word()); \
        PI_KT_LAUNCH(PI_KT_OTHER, 0, nt, 0.0, k_sample_border, each, dim3(SP_THREADS), 0, s, A, S, slices, pi_abort_word()); \
        PI_KT_LAUNCH(PI_KT_OTHER, 0, nt, 4.0 * rows * n_vocab, k_sample_exact<W>, all, dim3(512), 0, s, A, S, slices, pi_abort_word()); \
        PI_KT_LAUNCH(PI_KT_OTHER, 0, nt, 0.0, k_sample_join<W>, each, dim3(SP_THREADS), 0, s, A, S, slices, pi_abort_word()); \
    } while (0)
    if (wide) SP_GO(true); else SP_GO(false);
#undef SP_GO
    PI_CHECK_LAUNCH();
    return 0;
}
