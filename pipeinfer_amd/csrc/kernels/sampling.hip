// A token for every row of logits, from a given random number.
//
//   order: larger logits first, the lower id on a tie; minus infinity and what is no number are not there
//   top-k: the first top_k (0 or less: all)                                          w = exp(x - max)
//   top-p: of those, the ones whose weights ahead of them add up to less than top_p * (the weights of all of them), and the first       (1 or more: all)
//   min-p: of those, the ones with w >= min_p, and the first
//   e = exp((x - max) / temperature) of what stays (temperature 0 or less: of the first alone);  the token: in the order of the ids the first whose running sum of e exceeds u * (the sum of all), its probability e / sum
//
// Sums are whole numbers, weights in steps of 2^-44 (a row of 2^19 of the largest weight fits 64 bits): the order of additions, and with it of atomics, is without effect, and a sum is off by less than the number of its terms x 2^-45
// of a total of at least 1.  Exponentials are fp64, within 1e-13: with fp32's the borders of thousands of candidates would move by whole tokens.
// A workgroup per row.  Few of the best (top_k up to 128): every thread's largest value bounds the top_k-th from below, what reaches the bound - little more than top_k values - is ranked in LDS and the rest is never looked at again.
// Otherwise the weights of all values are added up in bins of equal width below the maximum, the bin that holds the border is listed and ranked; a list that does not fit gives way to the digits of (value, id), eight bits a pass.
#include "ops_common.h"
#include "kernel_timing.h"

#include <algorithm>

#define SP_THREADS 1024
#define SP_WAVES (SP_THREADS / 64)
#define SP_BINS 4096
#define SP_PER_UNIT 128.0f   /* bins to a unit of logits: 32 below the maximum; 330 values in the fullest where 2^18 are spread by 2.5 */
#define SP_LIST 512
#define SP_FEW 128
#define SP_ONE 17592186044416.0    /* 2^44 */
#define SP_MAX_VOCAB (1 << 19)

typedef unsigned long long sp_u64;

// e^x, x <= 0: x = n ln 2 + r, |r| <= 0.35, by the series of e^r up to r^12 / 12! (the next term: 2e-16)
static __device__ __forceinline__ double sp_exp(double x) {
    if (!(x > -700.0)) return 0.0;
    const double n = __builtin_rint(x * 1.4426950408889634), r = fma(n, -1.9082149292705877e-10, fma(n, -0.693147180369123816490, x));
    double s = 1.0 / 479001600.0;
    s = fma(s, r, 1.0 / 39916800.0); s = fma(s, r, 1.0 / 3628800.0); s = fma(s, r, 1.0 / 362880.0); s = fma(s, r, 1.0 / 40320.0); s = fma(s, r, 1.0 / 5040.0); s = fma(s, r, 1.0 / 720.0);
    s = fma(s, r, 1.0 / 120.0); s = fma(s, r, 1.0 / 24.0); s = fma(s, r, 1.0 / 6.0); s = fma(s, r, 0.5); s = fma(s, r, 1.0); s = fma(s, r, 1.0);
    return ldexp(s, (int) n);
}
static __device__ __forceinline__ sp_u64 sp_steps(double w) { return (sp_u64) (w * SP_ONE + 0.5); }

// larger value first, then the lower id; 0: not there
static __device__ __forceinline__ sp_u64 sp_rank(float x, int id) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return (sp_u64) (b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (uint32_t) ~id;
}
static __device__ __forceinline__ float sp_value(sp_u64 r) { const uint32_t k = (uint32_t) (r >> 32); return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
static __device__ __forceinline__ int sp_id(sp_u64 r) { return (int) ~(uint32_t) r; }

static __device__ __forceinline__ sp_u64 sp_wave_sum(sp_u64 v) { pi_butterfly<32>([&](auto o) { v += pi_partner<decltype(o)::value>(v); }); return v; }
static __device__ __forceinline__ sp_u64 sp_wave_top(sp_u64 v) { pi_butterfly<32>([&](auto o) { const sp_u64 x = pi_partner<decltype(o)::value>(v); v = x > v ? x : v; }); return v; }

struct sp_args {
    const float * logits; int64_t stride; int vocab;
    const float * temp; const int32_t * top_k; const float * top_p, * min_p, * u;
    int32_t * id; float * prob; int32_t * kept;
};

struct sp_shared {
    sp_u64 weight[SP_BINS]; uint32_t count[SP_BINS];         // bins; digits
    sp_u64 list[SP_LIST], sorted[SP_FEW], waves[SP_WAVES]; double w[SP_FEW]; int n, hit; sp_u64 before, answer;
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
    sp_u64 x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) { const sp_u64 y = __shfl_up(x, o, 64); if (lane >= o) x += y; }
    __syncthreads();
    if (lane == 63) L.waves[wave] = x;
    __syncthreads();
    sp_u64 base = 0; all = 0;
#pragma unroll
    for (int i = 0; i < SP_WAVES; i++) { const sp_u64 w = L.waves[i]; if (i < wave) base += w; all += w; }
    return base + x - v;
}

// VPT > 0: up to 1024 VPT values stay in registers.  A wave has a run of `chunk` ids, 256 of them a step: four to a lane side by side where rows lie on 16 bytes
template <int VPT, bool WIDE> __global__ void __launch_bounds__(SP_THREADS) k_sample(const sp_args A, const int32_t * __restrict__ abort_w) {
    if (pi_aborted(abort_w)) return;
    __shared__ sp_shared L;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = blockIdx.x, V = A.vocab, steps = (V + 256 * SP_WAVES - 1) / (256 * SP_WAVES), chunk = 256 * steps;
    const float * x = A.logits + (int64_t) row * A.stride;
    const float temp = A.temp ? A.temp[row] : 1.0f, top_p = A.top_p ? A.top_p[row] : 1.0f, min_p = A.min_p ? A.min_p[row] : 0.0f;
    const int first = wave * chunk;
    float own[VPT > 0 ? VPT : 4];
    auto id_of = [&](int j, int e) __attribute__((always_inline)) { return first + 256 * j + (WIDE ? 4 * lane + e : 64 * e + lane); };
    auto load = [&](int j, float * to) __attribute__((always_inline)) {
        if (WIDE && id_of(j, 3) < V) { const float4 v = *(const float4 *) (x + id_of(j, 0)); to[0] = v.x; to[1] = v.y; to[2] = v.z; to[3] = v.w; }
        else
#pragma unroll
            for (int e = 0; e < 4; e++) to[e] = id_of(j, e) < V ? x[id_of(j, e)] : -INFINITY;
#pragma unroll
        for (int e = 0; e < 4; e++) to[e] = to[e] > -INFINITY ? to[e] : -INFINITY;          // (and what is no number)
    };
    if constexpr (VPT > 0) {
#pragma unroll
        for (int j = 0; j < VPT / 4; j++) {
            if (j < steps) load(j, own + 4 * j);
            else
#pragma unroll
                for (int e = 0; e < 4; e++) own[4 * j + e] = -INFINITY;
        }
    }
    auto each = [&](auto && f) __attribute__((always_inline)) {
        if constexpr (VPT > 0) {
#pragma unroll
            for (int j = 0; j < VPT / 4; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) f(own[4 * j + e], id_of(j, e));
        } else
            for (int j = 0; j < steps; j++) {
                float v[4];
                load(j, v);
#pragma unroll
                for (int e = 0; e < 4; e++) f(v[e], id_of(j, e));
            }
    };

    auto each_again = [&](auto && f) __attribute__((always_inline)) {    // (where it is rarely needed: from memory)
        for (int i = tid; i < V; i += SP_THREADS) { const float v = x[i]; if (v > -INFINITY) f(v, i); }
    };

    // the first of the order, how many there are
    sp_u64 best = 0, present = 0;
    float mine = -INFINITY; int mine_id = 0;
    each([&](float v, int id) __attribute__((always_inline)) { if (v > mine) { mine = v; mine_id = id; } present += v > -INFINITY; });
    if (mine > -INFINITY) best = sp_rank(mine, mine_id);      // (a thread's ids ascend: the first of equals)
    const sp_u64 thread_best = best;
    best = sp_wave_top(best);
    if (lane == 0) L.waves[wave] = best;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < SP_WAVES; i++) best = L.waves[i] > best ? L.waves[i] : best;
    present = sp_all_sum(present, L, lane, wave);
    if (best == 0) {
        if (tid == 0) { A.id[row] = -1; if (A.prob) A.prob[row] = 0.0f; if (A.kept) A.kept[row] = 0; }
        return;
    }
    const float top = sp_value(best);
    int k = A.top_k ? A.top_k[row] : 0;
    if (k <= 0 || (sp_u64) k >= present) k = 0;
    auto below = [&](float v) __attribute__((always_inline)) { return v == top ? 0.0 : (double) v - (double) top; };        // (an infinite maximum: 0 of itself)
    auto weight = [&](float v) __attribute__((always_inline)) { return sp_exp(below(v)); };
    const double cooled = temp > 0.0f ? 1.0 / (double) temp : 1.0;
    auto chance = [&](float v) __attribute__((always_inline)) { return sp_exp(below(v) * cooled); };
    auto enough = [&](double w) __attribute__((always_inline)) { return !(min_p > 0.0f) || w >= (double) min_p; };
    auto bin_of = [&](float v) __attribute__((always_inline)) { return (int) fminf((v == top ? 0.0f : top - v) * SP_PER_UNIT, (float) (SP_BINS - 1)); };
    // bins from the top down, four to a thread: the bin in which a sum of `target` is reached, and what the bins ahead of it hold
    auto reach = [&](sp_u64 target, auto && bin, sp_u64 & ahead) __attribute__((always_inline)) {
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
    };
    auto gather = [&](auto && in) __attribute__((always_inline)) {       // the ranks of what `in` says, in any order; how many there are (more than the list holds: the list is of no use)
        __syncthreads();
        if (tid == 0) L.n = 0;
        __syncthreads();
        each([&](float v, int id) __attribute__((always_inline)) {
            if (v > -INFINITY && in(v, id)) { const int at = atomicAdd(&L.n, 1); if (at < SP_LIST) L.list[at] = sp_rank(v, id); }
        });
        __syncthreads();
        return L.n;
    };

    if (k > 0 && k <= SP_FEW) {
        // a bound that at least k threads' largest values reach
        for (int i = tid; i < SP_BINS; i += SP_THREADS) L.count[i] = 0;
        __syncthreads();
        if (thread_best != 0) atomicAdd(&L.count[bin_of(mine)], 1u);
        sp_u64 ahead;
        __syncthreads();
        const int bound = reach((sp_u64) k, [&](int i) __attribute__((always_inline)) { return (sp_u64) L.count[i]; }, ahead);
        const int n = bound == SP_BINS - 1 ? SP_LIST + 1 : gather([&](float v, int) __attribute__((always_inline)) { return bin_of(v) <= bound; });
        if (n >= k && n <= SP_LIST) {
            if (tid < n) {
                const sp_u64 r = L.list[tid];
                int at = 0;
                for (int i = 0; i < n; i++) at += L.list[i] > r;
                if (at < k) L.sorted[at] = r;
            }
            __syncthreads();
            if (wave == 0) {
                // two to a lane, in order: 2 lane, 2 lane + 1
                const bool is0 = 2 * lane < k, is1 = 2 * lane + 1 < k;
                const sp_u64 r0 = is0 ? L.sorted[2 * lane] : 0, r1 = is1 ? L.sorted[2 * lane + 1] : 0;
                const double w0 = is0 ? weight(sp_value(r0)) : 0.0, w1 = is1 ? weight(sp_value(r1)) : 0.0;
                const sp_u64 s0 = sp_steps(w0), s1 = sp_steps(w1);
                sp_u64 run = s0 + s1;
#pragma unroll
                for (int o = 1; o < 64; o <<= 1) { const sp_u64 y = __shfl_up(run, o, 64); if (lane >= o) run += y; }
                const sp_u64 all = __shfl(run, 63, 64), b0 = run - s0 - s1, b1 = b0 + s0;
                const double edge = (double) top_p * (double) all;
                const bool nucleus = top_p < 1.0f;
                const bool k0 = is0 && (lane == 0 || ((!nucleus || (double) b0 < edge) && enough(w0))), k1 = is1 && (!nucleus || (double) b1 < edge) && enough(w1);
                const int kept = __popcll(__ballot(k0)) + __popcll(__ballot(k1));
                const bool greedy = !(temp > 0.0f);
                const double c0 = !k0 ? 0.0 : greedy ? (lane == 0 ? 1.0 : 0.0) : chance(sp_value(r0)), c1 = !k1 || greedy ? 0.0 : chance(sp_value(r1));
                const sp_u64 e0 = sp_steps(c0), e1 = sp_steps(c1), sum = sp_wave_sum(e0 + e1);
                const int i0 = sp_id(r0), i1 = sp_id(r1);
                sp_u64 a0 = 0, a1 = 0;                       // what the ids up to its own add up to
                for (int l = 0; l < (kept + 1) / 2; l++) {   // (what stays is ahead in the order)
                    const int p = __shfl(i0, l, 64), q = __shfl(i1, l, 64);
                    const sp_u64 x0 = __shfl(e0, l, 64), x1 = __shfl(e1, l, 64);
                    a0 += (p <= i0 ? x0 : 0) + (q <= i0 ? x1 : 0); a1 += (p <= i1 ? x0 : 0) + (q <= i1 ? x1 : 0);
                }
                const double want = (double) A.u[row] * (double) sum;
                const sp_u64 t = want >= (double) sum ? sum - 1 : want > 0.0 ? min((sp_u64) want, sum - 1) : 0;
                // the first id whose sum exceeds t: the one with a - e <= t < a
                const bool h0 = e0 > 0 && a0 > t && a0 - e0 <= t, h1 = e1 > 0 && a1 > t && a1 - e1 <= t;
                if (h0 || h1) { A.id[row] = h0 ? i0 : i1; if (A.prob) A.prob[row] = (float) ((h0 ? c0 : c1) * SP_ONE / (double) sum); }
                if (lane == 0 && A.kept) A.kept[row] = kept;
            }
            return;
        }
    }

    // the last of the order that stays: measure 1 or weights, `target` of it reached.  Bins first, then the list of the bin, or where that is too long the digits of the rank
    sp_u64 last = 0;                                         // nothing below this rank stays
    auto digits = [&](sp_u64 target, auto && measure) __attribute__((always_inline)) -> sp_u64 {
        sp_u64 prefix = 0;
        for (int p = 7; p >= 0; p--) {
            __syncthreads();
            for (int i = tid; i < 256; i += SP_THREADS) L.weight[i] = 0;
            __syncthreads();
            each_again([&](float v, int id) __attribute__((always_inline)) {
                const sp_u64 r = sp_rank(v, id);
                if (r >= last && (p == 7 || r >> (8 * p + 8) == prefix)) atomicAdd(&L.weight[r >> (8 * p) & 255], measure(v));
            });
            __syncthreads();
            if (tid == 0) {
                int d = 255;
                sp_u64 left = target;
                for (; d > 0 && L.weight[d] < left; d--) left -= L.weight[d];
                L.hit = d; L.before = target - left;
            }
            __syncthreads();
            prefix = prefix << 8 | (sp_u64) L.hit; target -= L.before;
        }
        return prefix;
    };
    auto ranked = [&](int n, sp_u64 target) __attribute__((always_inline)) -> sp_u64 {    // the same from a list of n whose measures stand in L.weight
        __syncthreads();
        if (tid == 0) L.answer = ~0ull;
        __syncthreads();
        if (tid < n) {
            const sp_u64 r = L.list[tid];
            sp_u64 ahead = 0;
            for (int i = 0; i < n; i++) { const sp_u64 o = L.list[i]; if (o > r && o >= last) ahead += L.weight[i]; }
            if (r >= last && ahead < target) atomicMin(&L.answer, r);        // (the last that is not behind the target)
        }
        __syncthreads();
        return L.answer;
    };
    const bool nucleus = top_p < 1.0f;
    if (k > 0 || nucleus) {
        for (int i = tid; i < SP_BINS; i += SP_THREADS) { L.weight[i] = 0; L.count[i] = 0; }
        __syncthreads();
        each([&](float v, int) __attribute__((always_inline)) {
            if (!(v > -INFINITY)) return;
            const int b = bin_of(v);
            if (k > 0) atomicAdd(&L.count[b], 1u);
            if (nucleus) atomicAdd(&L.weight[b], sp_steps(weight(v)));
        });
        __syncthreads();
        sp_u64 total = 0, ahead = 0;
        int edge = SP_BINS - 1;
        bool listed = true;
        // (the weights of a list's entries take the place of the bins' where those have been read)
        sp_u64 held[4] = { 0, 0, 0, 0 };
        if (nucleus)
#pragma unroll
            for (int e = 0; e < 4; e++) held[e] = L.weight[4 * tid + e];
        if (k > 0) {
            sp_u64 ahead_k;
            edge = reach((sp_u64) k, [&](int i) __attribute__((always_inline)) { return (sp_u64) L.count[i]; }, ahead_k);
            const int n = gather([&](float v, int) __attribute__((always_inline)) { return bin_of(v) == edge; });
            listed = n <= SP_LIST;
            if (listed) {
                if (tid < n) L.weight[tid] = 1;
                last = ranked(n, (sp_u64) k - ahead_k);
            } else last = digits((sp_u64) k, [](float) { return (sp_u64) 1; });
            if (nucleus) {                                   // of the bin at the edge only what stayed
                sp_u64 part = 0;
                if (listed) { if (tid < n && L.list[tid] >= last) part = sp_steps(weight(sp_value(L.list[tid]))); }
                else each_again([&](float v, int id) __attribute__((always_inline)) { if (bin_of(v) == edge && sp_rank(v, id) >= last) part += sp_steps(weight(v)); });
                part = sp_all_sum(part, L, lane, wave);
#pragma unroll
                for (int e = 0; e < 4; e++) held[e] = 4 * tid + e < edge ? held[e] : 4 * tid + e == edge ? part : 0;
            }
        }
        if (nucleus) {
            sp_u64 s = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) s += held[e];
            total = sp_all_sum(s, L, lane, wave);
            // the first whose sum, itself included, is not less than top_p * total
            const double want = (double) top_p * (double) total;
            sp_u64 target = want >= 1.0 ? (sp_u64) __builtin_ceil(want) : 1;
            target = min(target, total);
            const int bin = reach(target, [&](int i) __attribute__((always_inline)) { return held[i & 3]; }, ahead);
            const int n = gather([&](float v, int id) __attribute__((always_inline)) { return bin_of(v) == bin && sp_rank(v, id) >= last; });
            if (n <= SP_LIST) {
                if (tid < n) L.weight[tid] = sp_steps(weight(sp_value(L.list[tid])));
                last = ranked(n, target - ahead);
            } else last = digits(target, [&](float v) { return sp_steps(weight(v)); });
        }
    }
    const bool greedy = !(temp > 0.0f);
    auto stays = [&](float v, int id) __attribute__((always_inline)) {
        if (!(v > -INFINITY)) return false;
        const sp_u64 r = sp_rank(v, id);
        return r >= last && (r == best || !(min_p > 0.0f) || enough(weight(v)));
    };
    auto share = [&](float v, int id) __attribute__((always_inline)) { return greedy ? (sp_rank(v, id) == best ? sp_steps(1.0) : 0) : sp_steps(chance(v)); };
    sp_u64 kept = 0, e = 0;
    each([&](float v, int id) __attribute__((always_inline)) { if (stays(v, id)) { kept++; e += share(v, id); } });
    kept = sp_all_sum(kept, L, lane, wave);
    e = sp_wave_sum(e);
    __syncthreads();
    if (lane == 0) L.waves[wave] = e;
    __syncthreads();
    sp_u64 sum = 0;
#pragma unroll
    for (int i = 0; i < SP_WAVES; i++) sum += L.waves[i];
    const double want = (double) A.u[row] * (double) sum;
    sp_u64 t = want >= (double) sum ? sum - 1 : want > 0.0 ? min((sp_u64) want, sum - 1) : 0;
    // the wave's run that the sum t falls into, then a sixteenth of that, then its values one by one
    int seg = 0;
    while (seg < SP_WAVES - 1 && t >= L.waves[seg]) t -= L.waves[seg++];
    const int part = 64 * ((chunk / 64 + SP_WAVES - 1) / SP_WAVES), from = seg * chunk + wave * part, to = min(min(from + part, (seg + 1) * chunk), V);
    e = 0;
    for (int i = from + lane; i < to; i += 64) { const float v = x[i]; if (stays(v, i)) e += share(v, i); }
    e = sp_wave_sum(e);
    __syncthreads();
    if (lane == 0) L.waves[wave] = e;
    __syncthreads();
    int sub = 0;
    while (sub < SP_WAVES - 1 && t >= L.waves[sub]) t -= L.waves[sub++];
    if (wave != sub) return;
    for (int i0 = from; i0 < to; i0 += 64) {
        const int i = i0 + lane;
        const float v = i < to ? x[i] : -INFINITY;
        const sp_u64 mine_e = i < to && stays(v, i) ? share(v, i) : 0;
        sp_u64 run = mine_e;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) { const sp_u64 y = __shfl_up(run, o, 64); if (lane >= o) run += y; }
        const sp_u64 all = __shfl(run, 63, 64);
        if (t < all) {
            if (run > t && run - mine_e <= t) {
                A.id[row] = i;
                if (A.prob) A.prob[row] = (float) ((greedy ? 1.0 : chance(v)) * SP_ONE / (double) sum);
                if (A.kept) A.kept[row] = (int32_t) kept;
            }
            return;
        }
        t -= all;
    }
}

extern "C" size_t pi_op_sample_scratch_bytes(int n_vocab, int rows) { (void) n_vocab; (void) rows; return 0; }

extern "C" int pi_op_sample(const float * logits, int64_t stride, int n_vocab, int rows, const float * temp, const int32_t * top_k, const float * top_p, const float * min_p, const float * u, void * scratch, size_t scratch_bytes,
                            int32_t * id, float * prob, int32_t * kept, void * stream) {
    if (rows < 0 || n_vocab < 1 || n_vocab > SP_MAX_VOCAB || stride < n_vocab) { pi_set_error("pi_op_sample: %d rows of %d logits (1 .. 524288), %lld apart", rows, n_vocab, (long long) stride); return -1; }
    if (rows == 0) return 0;
    if (!logits || !u || !id) { pi_set_error("pi_op_sample: logits, random numbers or ids are NULL"); return -1; }
    const size_t need = pi_op_sample_scratch_bytes(n_vocab, rows);
    if (need > 0 && (!scratch || ((uintptr_t) scratch & 15) || scratch_bytes < need)) { pi_set_error("pi_op_sample: %zu bytes of scratch, on 16, for %zu (pi_op_sample_scratch_bytes)", scratch ? scratch_bytes : 0, need); return -1; }
    const sp_args A{ logits, stride, n_vocab, temp, top_k, top_p, min_p, u, id, prob, kept };
    const bool wide = stride % 4 == 0 && ((uintptr_t) logits & 15) == 0;
#define SP_GO(V, W) PI_KT_LAUNCH(PI_KT_OTHER, 0, std::min(rows, PI_KT_MAXNT - 1), 4.0 * rows * n_vocab, (k_sample<V, W>), dim3((unsigned) rows), dim3(SP_THREADS), 0, (hipStream_t) stream, A, pi_abort_word())
#define SP_BY(V) do { if (wide) SP_GO(V, true); else SP_GO(V, false); } while (0)
    if (n_vocab <= 8192) SP_BY(8); else if (n_vocab <= 32768) SP_BY(32); else SP_BY(0);
#undef SP_BY
#undef SP_GO
    PI_CHECK_LAUNCH();
    return 0;
}
